"""Attention over K / V in 4 bits where a row's numbers are far apart: weights
that round alike, one token above all others, query rows of very different
sizes in one tile; and the masks of the 8-, 16- and 128-row tiles, each with
its height asserted."""
import math

import numpy as np
import pytest
import torch

import fused3s_b200 as F
import kv4_ref as R
import test_kv4 as T
from fused3s_b200 import _lib

gpu = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def tile_rows(bt):
    """The height of the tiles of a plan (its header, behind the 64 words of the status)."""
    return int(bt.buffer[67])


def paged(lengths, heads, kv_heads, d, seed, tokens=None):
    """(cache, block tables, table rows) of requests, their pages in any order."""
    tables, free, begin, num_pages = T.make_tables(lengths, seed)
    cache = F.empty_kv4_cache(num_pages, kv_heads, d)
    bt = T.build(lengths, tables, free, begin, tokens or sum(n for _, n in lengths), heads=heads, kv_heads=kv_heads)
    return cache, bt, bt.tables.tolist()


def slots_of(row, n):
    return T.i32([row[p // 16] * 16 + p % 16 for p in range(n)])


def values(cache, row, n, kv_head=0):
    """K and V float64 [n, d] of a request, from the cache's bytes."""
    pk, pv = R.page_values(cache.pages[row[:-(-n // 16)], kv_head:kv_head + 1], cache.head_dim)
    return (x[:, 0].reshape(-1, cache.head_dim)[:n] for x in (pk, pv))


def star(n):
    """A graph whose first window sees every block column; the others see the first."""
    row_ptr = np.concatenate([[0], np.full(n, n, dtype=np.int64) + np.arange(n)]).astype(np.int32)
    return F.convert_csr_to_block_sparse(n, row_ptr, np.concatenate([np.arange(n), np.zeros(n - 1)]).astype(np.int32))


# ------------------------------------------------- weights that round alike --

def alike(n, kv_heads, d, seed):
    """K and V of n tokens: every sixteenth token scores L above the others, L
    such that the others' weight lies 0.49 of an fp16 step above an fp16 number;
    V of +1 and -1, so that every row has the same scale.  And q's value, the
    scale that makes L, L."""
    level = 1 - math.log2(1.5 + 0.49 * 2.0 ** -10)
    k = torch.zeros(n, kv_heads, d)
    k[::16] = 1.0
    v = torch.where(T.randn((n, kv_heads, d), seed) > 0, 1.0, -1.0)
    one = 15 * float(torch.tensor(1 / 15).half())  # what a row of ones stands for
    return k.half().cuda(), v.half().cuda(), 0.125, level * math.log(2) / (d * 0.125 * one), level


def check_alike(got, k, v, visible, level, out_dtype):
    """got [rows, d] against 64 bits.

    Rounding the weights to fp16 (off by e <= 2^-11 of them, the same for tokens of
    the same score) moves the result by at most 2 e p (1 - p) |A - B|, with p the
    share of the high tokens and A, B the means of V over the high and the other
    tokens -- if the same weights are used in every sum.  The sums of codes times
    scales reach 2 (codes 0 ... 15 of a span of 2) and are off by 64 steps of
    2^-23 and one per product of 16 tokens.  The result is rounded once."""
    high = torch.arange(k.shape[0]) % 16 == 0
    weight = torch.where(high, 2.0 ** level, 1.0).double() * visible
    share = weight / weight.sum(-1, keepdim=True)
    want = share @ v
    p = (share * high).sum(-1, keepdim=True)
    a, b = (share * high) @ v / p, (share * ~high) @ v / (1 - p)
    tol = 2 * 2.0 ** -11 * p * (1 - p) * (a - b).abs() if out_dtype == torch.bfloat16 else 0.0
    tol = tol + 2 * (64 + k.shape[0] / 16) * 2.0 ** -23 + HALF_STEP[out_dtype] * want.abs()
    R.assert_close(got, want, tol)


@gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,new,height", [(2, 1, 8), (2, 30, 16), (2, 150, 128)])
def test_attention_weights_that_round_alike(lib, heads, new, height, d, out_dtype):
    n = 3000 + new
    cache, bt, rows = paged([(3000, new)], heads, 1, d, 5)
    assert tile_rows(bt) == height
    k, v, q, scale, level = alike(n, 1, d, 7)
    F.store_kv4(k, v, slots_of(rows[0], n), cache, check_status=True)
    Q = torch.full((new, heads, d), q, dtype=torch.bfloat16, device="cuda")
    o = F.attention_kv4(Q, cache, bt, scale=scale, out_dtype=out_dtype, check_status=True)
    k, v = values(cache, rows[0], n)
    visible = torch.arange(n)[None, :] <= (3000 + torch.arange(new))[:, None]
    for h in range(heads):
        check_alike(o[:, h], k, v, visible, level, out_dtype)


@gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,d", [(1, 64), (2, 64), (4, 64), (4, 128)])
def test_graph_weights_that_round_alike(lib, heads, d, out_dtype):
    n = 3008
    fmt = star(n)
    k, v, q, scale, level = alike(n, 1, d, 8)
    cache = F.empty_kv4_cache(fmt.num_row_windows, 1, d)
    F.store_kv4(k, v, torch.arange(n, dtype=torch.int32, device="cuda"), cache, check_status=True)
    Q = torch.full((n, heads, d), q, dtype=torch.bfloat16, device="cuda")
    o = F.fused3s_forward_kv4(Q, cache, fmt, scale=scale, out_dtype=out_dtype, check_status=True)
    k, v = values(cache, list(range(n // 16)), n)
    for h in range(heads):
        check_alike(o[:16, h], k, v, torch.ones(16, n), level, out_dtype)


# --------------------------------------------- one token above all others --

LOW = 24 - math.log2(22.49)  # the others' weight, 2^-LOW, lies midway between two numbers 2^-24 apart


def one_above(n, kv_heads, d):
    """K and V of n tokens: the first scores LOW above the others and has V = -1, the others +1."""
    k, v = torch.zeros(n, kv_heads, d), torch.ones(n, kv_heads, d)
    k[0], v[0] = 1.0, -1.0
    one = 15 * float(torch.tensor(1 / 15).half())
    return k.half().cuda(), v.half().cuda(), 0.125, LOW * math.log(2) / (d * 0.125 * one)


def check_one_above(got, v, seen, d):
    """got [rows, d] (fp32) of rows that see `seen` tokens.

    The others' share of the weights is s; their scores, LOW ln 2 below the first,
    are off by 3 LOW ln 2 (d / 16 + 4) 2^-22 in numerator and denominator each
    (codes and zeros apart, as in kv4_ref.tolerance), which moves the result by 2 s
    times that.  A weight in two fp16 parts is off by 2^-21 of it or by half of the
    smallest fp16 number, 2^-25, where the largest weight is 2^7 or more: 2^-32
    of it; V's values are 2 apart.  Reciprocals and sums add 64 steps of 2^-23."""
    low = (seen - 1).double() * 2.0 ** -LOW
    one = float(v[1, 0])
    want = one * (low - 1) / (low + 1)
    s = low / (low + 1)
    tol = 2 * s * (2 * 3 * LOW * math.log(2) * (d / 16 + 4) * 2.0 ** -22 + 2.0 ** -21)
    tol = tol + 2 * seen.double() * 2.0 ** -32 + 2 * 64 * 2.0 ** -23
    R.assert_close(got, want[:, None].expand(-1, d), tol[:, None].expand(-1, d))


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_attention_one_token_above_all_others(lib, d):
    """Prompts whose tiles walk 100 pages and more in one piece."""
    context, new, heads = 8000, 2048, 8
    n = context + new
    cache, bt, rows = paged([(context, new)], heads, heads, d, 5)
    assert tile_rows(bt) == 128
    k, v, q, scale = one_above(n, heads, d)
    F.store_kv4(k, v, slots_of(rows[0], n), cache, check_status=True)
    Q = torch.full((new, heads, d), q, dtype=torch.bfloat16, device="cuda")
    o = F.attention_kv4(Q, cache, bt, scale=scale, out_dtype=torch.float32, check_status=True)
    _, v = values(cache, rows[0], 16)
    for h in (0, heads - 1):
        check_one_above(o[:, h], v, context + torch.arange(new) + 1, d)


@gpu
@pytest.mark.parametrize("heads,d", [(1, 64), (4, 128)])
def test_graph_one_token_above_all_others(lib, heads, d):
    """A window that sees 2,500 blocks in one piece (the caller's estimate of the blocks sets its length)."""
    n = 40000
    fmt = star(n)
    k, v, q, scale = one_above(n, 1, d)
    cache = F.empty_kv4_cache(fmt.num_row_windows, 1, d)
    F.store_kv4(k, v, torch.arange(n, dtype=torch.int32, device="cuda"), cache, check_status=True)
    Q = torch.full((16, heads, d), q, dtype=torch.float16, device="cuda")
    o = torch.empty((16, heads, d), device="cuda")
    order, blocks = T.i32([0]), 6 * 160 * 2500
    size = lib.f3s_kv4_forward_scratch_size(1, blocks, heads, 1, d)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    ws = torch.zeros(256, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    st = lib.f3s_kv4_forward(Q.data_ptr(), _lib.F3S_OUT_F16, cache.pages.data_ptr(), cache.num_pages, o.data_ptr(),
                             _lib.F3S_OUT_F32, fmt.window_offsets.data_ptr(), fmt.cols_ptr, order.data_ptr(), 1, blocks,
                             n, heads, 1, d, scale, 0, 16, ws.data_ptr(), 256, scratch.data_ptr(), size, stream)
    assert st == 0 and lib.f3s_workspace_status(ws.data_ptr(), stream) == 0
    _, v = values(cache, [0], 16)
    for h in range(heads):
        check_one_above(o[:, h], v, torch.full((16,), n), d)


# --------------------------------------- query rows of very different sizes --

def check_rows(q, k, v, scale, visible, got, out_dtype, rows):
    """Each of the listed rows by itself: its tolerance comes from its own size."""
    for r in rows:
        want = R.attention(q[r:r + 1], k, v, scale, visible[r:r + 1])
        R.assert_close(got[r:r + 1], want, R.tolerance(q[r:r + 1], k, v, scale, want, out_dtype), f"row {r}")


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ratio", [2.0 ** 30, 2.0 ** 100, 2.0 ** 118])
@pytest.mark.parametrize("new,height", [(3, 8), (30, 16), (150, 128)])
def test_attention_rows_of_very_different_sizes(lib, new, height, ratio, d):
    """A head, and a token of the other head, far larger than the rest of the tile."""
    context, heads = 70, 2
    n = context + new
    cache, bt, rows = paged([(context, new)], heads, 1, d, 5)
    assert tile_rows(bt) == height
    k, v = (T.randn((n, 1, d), s, torch.float16).cuda() for s in (1, 2))
    F.store_kv4(k, v, slots_of(rows[0], n), cache, check_status=True)
    q = T.randn((new, heads, d), 3, torch.bfloat16)
    q[:, 0] *= ratio
    q[1, 1] *= ratio
    o = F.attention_kv4(q.cuda(), cache, bt, scale=d ** -0.5, out_dtype=torch.float32, check_status=True)
    k, v = values(cache, rows[0], n)
    visible = torch.arange(n)[None, :] <= (context + torch.arange(new))[:, None]
    check_rows(q[:, 1].double(), k, v, d ** -0.5, visible, o[:, 1].cpu(), torch.float32, [r for r in range(new) if r != 1])
    assert float(o.abs().max()) <= 1.01 * float(v.abs().max())  # the large ones: an average all the same


@gpu
@pytest.mark.parametrize("heads,kv_heads,d", [(1, 1, 64), (2, 1, 64), (4, 4, 64), (4, 2, 128)])
@pytest.mark.parametrize("ratio", [2.0 ** 30, 2.0 ** 100, 2.0 ** 118])
def test_graph_rows_of_very_different_sizes(lib, heads, kv_heads, d, ratio):
    n = 512
    fmt = star(n)
    cache = T.filled_cache(fmt.num_row_windows, kv_heads, d, 4)
    q = T.randn((n, heads, d), 3, torch.bfloat16)
    q[[3, 8, 13]] *= ratio
    o = F.fused3s_forward_kv4(q.cuda(), cache, fmt, scale=d ** -0.5, check_status=True)
    for h in range(heads):
        k, v = values(cache, list(range(n // 16)), n, h // (heads // kv_heads))
        check_rows(q[:16, h].double(), k, v, d ** -0.5, torch.ones(16, n, dtype=torch.bool), o[:16, h].cpu(), torch.float32,
                   [r for r in range(16) if r not in (3, 8, 13)])
        assert float(o[:16, h].abs().max()) <= 1.01 * float(v.abs().max())


# ----------------------------------------------- scores beyond whole steps --

@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ratio", [2.0 ** 30, 2.0 ** 100, 2.0 ** 118])
def test_attention_scores_too_large_for_fp32s_whole_steps(lib, ratio, d):
    """Scores whose steps in fp32 are larger than the reach of a weight, in 128-row
    tiles: the reference settles all the same, the other rows are right, and what the
    large rows give is an average of V."""
    context, new, heads = 70, 150, 2
    n = context + new
    cache, bt, rows = paged([(context, new)], heads, 1, d, 5)
    assert tile_rows(bt) == 128
    k, v = (T.randn((n, 1, d), s, torch.float16).cuda() for s in (1, 2))
    F.store_kv4(k, v, slots_of(rows[0], n), cache, check_status=True)
    q = T.randn((new, heads, d), 3, torch.bfloat16)
    q[:, 0] *= ratio
    k, v = values(cache, rows[0], n)
    visible = torch.arange(n)[None, :] <= (context + torch.arange(new))[:, None]
    for out_dtype in (torch.float32, torch.bfloat16):
        o = F.attention_kv4(q.cuda(), cache, bt, scale=d ** -0.5, out_dtype=out_dtype, check_status=True).cpu()
        want = R.attention(q[:, 1].double(), k, v, d ** -0.5, visible)
        R.assert_close(o[:, 1], want, R.tolerance(q[:, 1].double(), k, v, d ** -0.5, want, out_dtype))
        assert float(o.abs().max()) <= 1.01 * float(v.abs().max())


# ---------------------------------------------------------- very long sums --

def long_cache(num_pages, kv_heads, d, seed):
    """V of +1 and -1, whose sums cancel where sums of their codes do not; and K, V in 64 bits."""
    n = num_pages * 16
    k = (T.randn((n, kv_heads, d), seed) * 0.3).half().cuda()
    v = torch.where(T.randn((n, kv_heads, d), seed + 1) > 0, 1.0, -1.0).half().cuda()
    cache = F.empty_kv4_cache(num_pages, kv_heads, d)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    F.store_kv4(k, v, slots, cache, check_status=True)
    return (cache, *(x.double() for x in F.load_kv4(cache, slots, torch.float32)))


def check_long(got, q, k, v, scale, counts, out_dtype):
    """got [d] of a row q [d] that sees token t of K, V [n, d] counts[t] times.

    An accumulator takes at most 256 pages, two products each, before it is added to a
    sum in fp32; an addition cuts off at most 2^-23 of the accumulator, and the
    accumulators of a row add up to V's span, 2, at most: 512 * 2^-23 * 2.  Scores as
    in kv4_ref.tolerance.  A lane adds up to 2^16 numbers in fp32, rounded to
    nearest (0.29 steps of 2^-23 each, of a sum that grows): six deviations of that are
    6 * 2^8 * 0.29 / 3^0.5 steps, in the zeros' sum and in the weights'."""
    w = counts * torch.exp((k @ q) * scale)
    want = (w @ v) / w.sum()
    a = 3.0 * scale * float(q.abs().sum()) * float(k.abs().max())
    rel = 2 * a * (k.shape[1] / 16 + 4) * 2.0 ** -22 + 64 * 2.0 ** -23 + 2 * 6 * 2.0 ** 8 * 0.29 / 3 ** 0.5 * 2.0 ** -23
    if out_dtype == torch.bfloat16:
        rel += 2 * 2.0 ** -11 * float(want.abs().max())  # the weights' own rounding, of their average
    tol = 512 * 2.0 ** -23 * 2 + 2 * rel + HALF_STEP[out_dtype] * want.abs()
    R.assert_close(got, want.cpu(), tol.cpu())


@gpu
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("requests,new,heads,kv_heads,d,height", [
    (64, 1, 8, 8, 64, 8), (64, 1, 8, 8, 128, 8), (8, 12, 32, 8, 64, 16), (8, 12, 32, 8, 128, 16),
    (1, 2048, 8, 8, 64, 128), (1, 2048, 8, 8, 128, 128)])
def test_attention_over_a_million_tokens(lib, requests, new, heads, kv_heads, d, height, out_dtype):
    """Tables that list 512 pages again and again, 65,536 entries long."""
    pool, repeats = 512, 128
    tokens = pool * 16
    cache, k, v = long_cache(pool, kv_heads, d, 5)
    order = torch.randperm(pool, generator=T.gen(6)).int()
    tables = order.repeat(requests, repeats).cuda()
    context = pool * repeats * 16 - new
    bt = F.build_block_tables(T.i32([context] * requests), T.i32([new] * requests), tables, tables[0, -new // 16 - 1:].contiguous(),
                              None, requests * new, heads=heads, kv_heads=kv_heads)
    assert tile_rows(bt) == height
    tables.copy_(order.repeat(requests, repeats))  # the new pages are the pool's last again
    q = (T.randn((requests * new, heads, d), 7) * 0.1).bfloat16().cuda()
    o = F.attention_kv4(q, cache, bt, scale=d ** -0.5, out_dtype=out_dtype)
    assert torch.equal(F.attention_kv4(q, cache, bt, scale=d ** -0.5, out_dtype=out_dtype), o)
    at = (order.long()[:, None] * 16 + torch.arange(16)).reshape(-1).cuda()  # tokens of the pool, as the tables list them
    for row, h in ((0, 0), (new - 1, heads - 1), (new // 2, 1), (requests * new - 1, 2)):
        hidden = new - 1 - row % new  # new tokens that come later
        counts = torch.full((tokens,), float(repeats), dtype=torch.float64, device="cuda")
        if hidden:
            counts[at[tokens - hidden:]] -= 1
        g = h // (heads // kv_heads)
        check_long(o[row, h], q[row, h].double(), k[:, g], v[:, g], d ** -0.5, counts, out_dtype)


@gpu
@pytest.mark.parametrize("heads,kv_heads,d", [(1, 1, 64), (2, 1, 128), (4, 1, 64), (4, 4, 64), (4, 2, 128)])
def test_graph_window_of_very_many_blocks(lib, heads, kv_heads, d):
    """A window of 32,000 blocks in one piece (the caller's estimate of the blocks sets its length)."""
    blocks = 32000
    n = blocks * 16
    cache, k, v = long_cache(blocks, kv_heads, d, 5)
    offsets = T.i32([0, blocks] + [blocks] * (blocks - 1))
    cols, order = torch.arange(blocks, dtype=torch.int32, device="cuda"), T.i32([0])
    q = (T.randn((16, heads, d), 7) * 0.1).half().cuda()
    estimate = 900 * blocks
    size = lib.f3s_kv4_forward_scratch_size(1, estimate, heads, kv_heads, d)
    scratch = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")
    ws = torch.zeros(256, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for out_dtype, code in ((torch.float32, _lib.F3S_OUT_F32), (torch.bfloat16, _lib.F3S_OUT_BF16)):
        o = torch.empty((16, heads, d), dtype=out_dtype, device="cuda")
        st = lib.f3s_kv4_forward(q.data_ptr(), _lib.F3S_OUT_F16, cache.pages.data_ptr(), cache.num_pages, o.data_ptr(), code,
                                 offsets.data_ptr(), cols.data_ptr(), order.data_ptr(), 1, estimate, n, heads, kv_heads, d,
                                 d ** -0.5, 0, 16, ws.data_ptr(), 256, scratch.data_ptr(), size, stream)
        assert st == 0 and lib.f3s_workspace_status(ws.data_ptr(), stream) == 0
        for row, h in ((0, 0), (9, heads - 1), (15, heads // 2)):
            g = h // (heads // kv_heads)
            check_long(o[row, h], q[row, h].double(), k[:, g], v[:, g], d ** -0.5,
                       torch.ones(n, dtype=torch.float64, device="cuda"), out_dtype)


# ------------------------------------------------------- tiles of 16 rows --

SIXTEEN = [(20, 33), (0, 25), (33, 31)]  # with two query heads to a K/V head: 59 rows per request


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_16_row_tiles_leave_out_what_is_masked(lib, d):
    assert tile_rows(paged(SIXTEEN, 4, 2, d, 1, tokens=92)[1]) == 16
    T.test_attention_leaves_out_what_is_masked(lib, SIXTEEN, 4, d)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,height", [(1, 8), (30, 16), (150, 128)])
def test_rising_scores_in_every_tile(lib, new, height, d):
    lengths, n = [(800, new)], 800 + new
    cache, bt, rows = paged(lengths, 2, 1, d, 3)
    assert tile_rows(bt) == height
    k = torch.ones(n, 1, d) * (torch.arange(n) / 100.0)[:, None, None]
    F.store_kv4(k.half().cuda(), T.randn((n, 1, d), 2).half().cuda(), slots_of(rows[0], n), cache)
    q = torch.ones(new, 2, d, dtype=torch.float16, device="cuda")
    for out_dtype in (torch.float32, torch.bfloat16):
        o = F.attention_kv4(q, cache, bt, scale=0.5, out_dtype=out_dtype, check_status=True)
        want, pk, pv = T.want_attention(q, cache, rows, lengths, 0.5, 2)
        R.assert_close(o, want, R.tolerance(q.double().cpu(), pk, pv, 0.5, want, out_dtype))


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e-4, 300.0])
def test_extreme_sizes_in_16_row_tiles(lib, size, d):
    tables, free, begin, num_pages = T.make_tables(SIXTEEN, 7)
    cache = T.filled_cache(num_pages, 2, d, 5, size)
    q = T.randn((89, 4, d), 8, torch.bfloat16, 1.0 / max(size, 1.0)).cuda()
    bt = T.build(SIXTEEN, tables, free, begin, 89, heads=4, kv_heads=2)
    assert tile_rows(bt) == 16
    o = F.attention_kv4(q, cache, bt, scale=0.5, out_dtype=torch.float32, check_status=True)
    want, pk, pv = T.want_attention(q, cache, bt.tables.tolist(), SIXTEEN, 0.5, 4)
    R.assert_close(o, want, R.tolerance(q.double().cpu(), pk, pv, 0.5, want, torch.float32))
    for _ in range(5):
        assert torch.equal(F.attention_kv4(q, cache, bt, scale=0.5, out_dtype=torch.float32), o)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,height", [(4, 8), (20, 16), (100, 128)])
def test_nan_reaches_only_who_sees_it_in_every_tile(lib, new, height, d):
    cache, bt, rows = paged([(20, new)], 2, 1, d, 12)
    assert tile_rows(bt) == height
    n = 20 + new
    k, v = (T.randn((n, 1, d), s, torch.float16) for s in (1, 2))
    v[22] = math.nan
    F.store_kv4(k.cuda(), v.cuda(), slots_of(rows[0], n), cache)
    q = T.randn((new, 2, d), 4, torch.float16).cuda()
    for out_dtype in (torch.float32, torch.bfloat16):
        o = F.attention_kv4(q, cache, bt, scale=0.1, out_dtype=out_dtype)
        assert torch.isfinite(o[:2]).all() and torch.isnan(o[2:]).all()
    q[1, 1, 5] = math.nan
    o = F.attention_kv4(q, cache, bt, scale=0.1, out_dtype=torch.float32)
    assert torch.isfinite(o[0]).all() and torch.isfinite(o[1, 0]).all() and torch.isnan(o[1, 1]).all()


@gpu
def test_16_row_tiles_on_two_streams(lib):
    lengths = [(700, 12), (90, 20), (0, 9)]
    assert tile_rows(paged(lengths, 8, 2, 128, 1)[1]) == 16
    T.test_calls_on_two_streams_share_tables_and_cache(lib, lengths)
