"""Plain 64-bit implementations for the tests of the 4-bit K/V cache: the
quantiser, the byte layout of a page read code by code, block tables in
loops, attention row by row."""
import math

import numpy as np
import torch

PAGE = 16


def quantise(x):
    """(scale, zero, codes) in float64 of rows x [..., d] (fp16 / bf16 values)."""
    x = x.double()
    nan = torch.isnan(x).any(-1, keepdim=True)
    x = torch.where(nan, torch.zeros_like(x), x)
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    scale = ((hi - lo) / 15).to(torch.float16).double().clamp(2.0 ** -24, 65504.0)
    zero = torch.round(-lo / scale).clamp(0, 15)
    codes = (torch.round(x / scale) + zero).clamp(0, 15)
    scale = torch.where(nan, torch.full_like(scale, math.nan), scale)
    zero, codes = torch.where(nan, torch.zeros_like(zero), zero), torch.where(nan, torch.zeros_like(codes), codes)
    return scale, zero, codes


def dequantise(x):
    s, z, u = quantise(x)
    return s * (u - z)


def page_values(pages, d):
    """K and V float64 [num_pages, kv_heads, 16, d] of a page buffer, byte by byte
    from the description in include/fused3s.h."""
    raw = pages.cpu().numpy()
    n, h = raw.shape[:2]
    flat = raw.reshape(n * h, -1)
    words = flat[:, :8 * d].copy().view("<u4").reshape(n * h, PAGE, d // 8)
    halves = flat[:, 8 * d:16 * d].copy().view("<u2").reshape(n * h, 2, 8, 4, d // 32, 2)
    scales = flat[:, 16 * d:].copy().view("<f2").reshape(n * h, 8, 2, 2, 2).astype(np.float64)
    k = np.zeros((n * h, PAGE, d))
    v = np.zeros((n * h, PAGE, d))
    for token in range(PAGE):
        sk, zk = scales[:, token % 8, token // 8, 0].T
        sv, zv = scales[:, token % 8, token // 8, 1].T
        for c in range(d):
            code = (words[:, token, c // 8] >> (4 * (c % 8 // 2) + 16 * (c % 2))) & 15
            k[:, token, c] = sk * (code.astype(np.float64) - zk)
            g, w, i = c // (d // 8), c % (d // 8) // 4, c % 4
            code = (halves[:, token // 8, g, token % 8 // 2, w, token % 2] >> (4 * i)) & 15
            v[:, token, c] = sv * (code.astype(np.float64) - zv)
    return torch.from_numpy(k).reshape(n, h, PAGE, d), torch.from_numpy(v).reshape(n, h, PAGE, d)


def block_tables(context, new, tables, free, begin, num_tokens):
    """(query_offsets, positions, slots, tables, free_begin), in loops; lengths that fit."""
    tables = [list(row) for row in tables]
    offsets, positions, slots = [0], [], []
    for i, (c, n) in enumerate(zip(context, new)):
        for k in range(-(-c // PAGE), -(-(c + n) // PAGE)):
            if begin < len(free):
                tables[i][k] = free[begin]
                begin += 1
            else:
                tables[i][k] = -1
        for p in range(c, c + n):
            page = tables[i][p // PAGE]
            positions.append(p)
            slots.append(-1 if page < 0 else page * PAGE + p % PAGE)
        offsets.append(offsets[-1] + n)
    pad = num_tokens - len(slots)
    return offsets, positions + [0] * pad, slots + [-1] * pad, tables, begin


def attention(q, k, v, scale, visible):
    """One head: q [n, d], k / v [t, d] float64, visible bool [n, t].  Rows that see
    nothing are 0."""
    s = (q @ k.T) * scale
    s = torch.where(visible, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    p = torch.where(visible, torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(s))
    total = p.sum(-1, keepdim=True)
    v = torch.where(visible.any(0)[:, None], v, torch.zeros_like(v))  # what nobody sees may be NaN
    return torch.where(total > 0, (p @ v) / total, torch.zeros_like(total))


def tolerance(q, k, v, scale, out, out_dtype):
    """How far a result may be from float64, per element of out.

    q and the codes are exact in the products.  The score's fp32 sum of d + 1
    terms adds 16 products a step and truncates: d / 16 + 4 steps of 2^-22 of the sum A
    of the magnitudes (codes and zeros apart: |s| (u + z) <= 3 max|k| where
    zero lies inside the row's range, so 3 |q| . max|k|); times scale; a weight is
    off by that, twice (numerator and denominator).  Weights, reciprocals and sums in
    fp32 add at most 64 steps of 2^-23 for the lengths tested.  Every error acts on
    values of at most V = max|v| (codes and zeros apart: 3 V).  bf16 results round the
    weights to fp16: 2^-11 of them, twice.  The result is rounded once."""
    d = q.shape[-1]
    a = 3.0 * abs(scale) * float(q.abs().sum(-1).max()) * float(k.abs().max())
    big = 3.0 * float(v.abs().max())
    rel = 2 * a * (d / 16 + 4) * 2.0 ** -22 + 64 * 2.0 ** -23
    if out_dtype == torch.bfloat16:
        rel += 2 * 2.0 ** -11
    step = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[out_dtype]
    return big * rel + step * out.abs()


def assert_close(got, want, tol, what=""):
    got = got.double().cpu()
    off = (got - want).abs() - tol
    assert torch.isfinite(got).all(), what
    assert float(off.max()) <= 0, f"{what}: off by {float((got - want).abs().max()):.3e}, {float(off.max()):.3e} too far"
