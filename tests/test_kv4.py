"""K / V in 4 bits: store, load, block tables, attention over request pages and
over the graph's windows, each against a plain 64-bit implementation
(kv4_ref.py); what the calls refuse; streams and CUDA graphs."""
import math
import random

import numpy as np
import pytest
import torch

import fused3s_b200 as F
import kv4_ref as R
from fused3s_b200 import _lib
from fused3s_b200 import graphs as G

gpu = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(shape, seed, dtype=torch.float32, size=1.0):
    return (torch.randn(shape, generator=gen(seed)) * size).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------- refusals --

def test_python_refuses_before_the_gpu():
    with pytest.raises(TypeError):
        F.KV4Cache(torch.zeros(2, 1, 1152))
    with pytest.raises(TypeError):
        F.KV4Cache(torch.zeros(2, 1152, dtype=torch.uint8))
    with pytest.raises(ValueError):
        F.KV4Cache(torch.zeros(2, 1, 1000, dtype=torch.uint8))
    with pytest.raises(ValueError):
        F.KV4Cache(torch.zeros(2, 1, 1152, dtype=torch.uint8))  # not on a GPU
    with pytest.raises(ValueError):
        F.empty_kv4_cache(2, 1, 96)
    t = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError):
        F.build_block_tables(t[0, :1], t[0, :1], t, t[0], None, 1)


def test_c_calls_refuse_without_touching_the_gpu(lib):
    bad, unsupported, ws, large = (_lib.F3S_ERR_INVALID_VALUE, _lib.F3S_ERR_UNSUPPORTED, _lib.F3S_ERR_WORKSPACE,
                                   _lib.F3S_ERR_TOO_LARGE)
    A = 4096  # an aligned address that is never read

    def store(dtype=1, stride=128, slots=A, n=3, pages=A, num_pages=2, heads=1, d=64, w=A, wb=256, k=A):
        return lib.f3s_kv4_store(k, A, dtype, stride, 64, stride, 64, slots, n, pages, num_pages, heads, d, w, wb, None)

    assert store(dtype=0) == bad and store(dtype=7) == bad
    assert store(stride=129) == bad and store(k=A + 2) == bad and store(k=None) == bad
    assert store(slots=None) == bad and store(pages=None) == bad and store(pages=A + 8) == bad
    assert store(n=-1) == bad and store(heads=0) == bad and store(num_pages=-1) == bad
    assert store(d=96) == unsupported and store(w=None) == bad and store(wb=255) == ws
    assert store(num_pages=1 << 28) == large and store(n=1 << 40) == large
    assert store(n=0) == 0

    def load(dtype=0, slots=A, n=3, d=64, k=A, wb=256):
        return lib.f3s_kv4_load(A, 2, 1, d, slots, n, k, A, dtype, A, wb, None)

    assert load(dtype=3) == bad and load(slots=None) == bad and load(k=None) == bad and load(k=A + 4) == bad
    assert load(d=32) == unsupported and load(wb=0) == ws and load(n=0) == 0

    def tables(ctx=A, new=A, r=2, tab=A, stride=8, width=8, free=A, nfree=4, n=2, h=4, g=2, q=A, pos=A, plan=A,
               pb=1 << 30):
        return lib.f3s_block_tables(ctx, new, r, tab, stride, width, free, nfree, None, n, h, g, q, pos, A, A, plan, pb,
                                    None)

    assert tables(ctx=None) == bad and tables(new=None) == bad and tables(tab=None) == bad
    assert tables(free=None) == bad and tables(q=None) == bad and tables(pos=None) == bad
    assert tables(r=-1) == bad and tables(width=-1) == bad and tables(nfree=-1) == bad and tables(n=-1) == bad
    assert tables(stride=7) == bad and tables(h=3) == bad and tables(h=0) == bad and tables(g=0) == bad
    assert tables(plan=None) == bad and tables(plan=A + 4) == bad and tables(pb=16) == ws and tables(pb=600) == ws
    assert tables(width=1 << 28, stride=1 << 28) == large and tables(n=1 << 31) == large

    def attend(q=A, dt=1, stride=512, pages=A, np_=4, tab=A, plan=A, r=2, n=2, h=4, g=2, d=64, o=A, odt=0, w=A,
               wb=1 << 40):
        return lib.f3s_kv4_attention(q, dt, stride, 64, pages, np_, tab, 8, plan, r, n, h, g, d, 1.0, o, odt, w, wb, None)

    assert attend(q=None) == bad and attend(q=A + 2) == bad and attend(dt=0) == bad and attend(odt=3) == bad
    assert attend(stride=4) == bad and attend(pages=None) == bad and attend(np_=0) == bad and attend(tab=None) == bad
    assert attend(plan=None) == bad and attend(h=3) == bad and attend(g=0) == bad and attend(d=80) == unsupported
    assert attend(o=None) == bad and attend(w=None) == bad and attend(wb=0) == ws and attend(n=-1) == bad
    assert attend(n=0) == 0 and attend(r=0) == 0

    def forward(q=A, dt=1, pages=A, np_=4, o=A, off=A, cols=A, order=A, items=1, nodes=50, h=2, g=2, d=64, base=0,
                rows=50, w=A, wb=256, s=A, sb=1 << 30, blocks=10):
        return lib.f3s_kv4_forward(q, dt, pages, np_, o, 0, off, cols, order, items, blocks, nodes, h, g, d, 1.0, base,
                                   rows, w, wb, s, sb, None)

    assert forward(q=None) == bad and forward(pages=None) == bad and forward(o=None) == bad
    assert forward(off=None) == bad and forward(cols=None) == bad and forward(order=None) == bad
    assert forward(np_=3) == bad and forward(h=3) == bad and forward(d=100) == unsupported
    assert forward(items=-1) == bad and forward(base=-1) == bad and forward(w=None) == bad and forward(wb=1) == ws
    assert forward(s=None) == bad and forward(s=A + 4) == bad and forward(sb=100) == ws and forward(blocks=-1) == bad
    assert forward(items=0) == 0 and forward(nodes=0) == 0 and forward(rows=0) == 0


def test_reference_layout_covers_every_code():
    """The byte layout is a bijection: each code of a page sits in one place."""
    for d in (64, 128):
        seen = set()
        for token in range(16):
            for c in range(d):
                bit = 32 * (token * (d // 8) + c // 8) + 4 * (c % 8 // 2) + 16 * (c % 2)
                seen.add(bit)
                g, w, i = c // (d // 8), c % (d // 8) // 4, c % 4
                half = (((token // 8 * 8 + g) * 4 + token % 8 // 2) * (d // 32) + w) * 2 + token % 2
                seen.add(64 * d + 16 * half + 4 * i)
        assert seen == set(range(0, 128 * d, 4))


@gpu
def test_python_refuses_on_the_gpu(lib):
    cache = F.empty_kv4_cache(4, 2, 64)
    k = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    slots = i32([0, 1, 2])
    for args in ((k.float(), k, slots), (k, k.bfloat16(), slots), (k, k, slots.long())):
        with pytest.raises(TypeError):
            F.store_kv4(*args, cache)
    for args in ((k.cpu(), k, slots), (k[:2], k, slots), (k[:, :1], k, slots), (k, k, slots.cpu()),
                 (torch.zeros(3, 2, 65, dtype=torch.float16, device="cuda")[..., :64], k, slots),
                 (torch.zeros(3 * 2 * 64 + 8, dtype=torch.float16, device="cuda")[4:388].view(3, 2, 64), k, slots)):
        with pytest.raises(ValueError):
            F.store_kv4(*args, cache)
    with pytest.raises(TypeError):
        F.load_kv4(cache, slots, torch.float64)
    tables = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    free = i32([0, 1, 2, 3])
    one = i32([3])
    with pytest.raises(ValueError):
        F.build_block_tables(one, one, tables, free, None, 3, heads=3, kv_heads=2)
    with pytest.raises(ValueError):
        F.build_block_tables(i32([1, 2]), one, tables, free, None, 3)
    with pytest.raises(ValueError):
        F.build_block_tables(one, one, tables.expand(3, 4)[:1].t(), free, None, 3)
    with pytest.raises(TypeError):
        F.build_block_tables(one.long(), one, tables, free, None, 3)
    with pytest.raises(ValueError):
        F.build_block_tables(one, one, tables, free, None, -1)
    bt = F.build_block_tables(i32([0]), one, tables, free, None, 3, heads=4, kv_heads=2)
    q = torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        F.attention_kv4(q[:2], cache, bt)
    with pytest.raises(ValueError):
        F.attention_kv4(q[:, :2], cache, bt)
    with pytest.raises(ValueError):
        F.attention_kv4(q, F.empty_kv4_cache(4, 4, 64), bt)
    with pytest.raises(ValueError):
        F.attention_kv4(q, cache, bt, out=torch.zeros(3, 4, 64, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError):
        F.attention_kv4(q, cache, F.build_block_tables(i32([0]), one, tables, free, None, 3))
    with pytest.raises(TypeError):
        F.attention_kv4(q.float(), cache, bt)
    fmt = F.convert_csr_to_block_sparse(100, np.arange(101, dtype=np.int32), np.arange(100, dtype=np.int32))
    with pytest.raises(ValueError):  # 7 block columns, 4 pages
        F.fused3s_forward_kv4(torch.zeros(100, 2, 64, dtype=torch.float16, device="cuda"), cache, fmt)


# ---------------------------------------------------------- store, load --

@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,kv_heads", [(1, 1), (37, 3), (300, 8)])
def test_store_and_load(lib, d, dtype, n, kv_heads):
    k, v = (randn((n, kv_heads, d), s, dtype, 2.0) for s in (1, 2))
    pages = n // 16 + 3
    slots = torch.randperm(pages * 16, generator=gen(3))[:n].int()
    cache = F.empty_kv4_cache(pages, kv_heads, d)
    F.store_kv4(k.cuda(), v.cuda(), slots.cuda(), cache, check_status=True)
    want_k, want_v = R.dequantise(k), R.dequantise(v)
    # the bytes are where the format says, and nothing else is written
    pk, pv = R.page_values(cache.pages, d)
    flat_k, flat_v = (x.transpose(1, 2).reshape(pages * 16, kv_heads, d) for x in (pk, pv))
    assert torch.equal(flat_k[slots.long()], want_k) and torch.equal(flat_v[slots.long()], want_v)
    others = torch.ones(pages * 16, dtype=torch.bool)
    others[slots.long()] = False
    assert not flat_k[others].any() and not flat_v[others].any()
    for out in (torch.float32, torch.float16, torch.bfloat16):
        got_k, got_v = F.load_kv4(cache, slots.cuda(), out, check_status=True)
        # scale * (code - zero) has at most 15 significant bits: exact in fp32, one rounding in 16 bits
        assert torch.equal(got_k.cpu(), want_k.float().to(out)) and torch.equal(got_v.cpu(), want_v.float().to(out))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_store_rows_of_every_kind(lib, dtype):
    """Zeros, constants of either sign, ties, the type's largest and smallest
    values, infinities, NaN, a value far from the others."""
    d = 64
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = [torch.zeros(d), torch.full((d,), 3.0), torch.full((d,), -2.5), torch.arange(d) / 2 - 7.5,
            torch.arange(d).remainder(16) + 0.5, torch.cat([torch.tensor([15.0]), (torch.arange(d - 1) % 15) + 0.5]),
            torch.full((d,), big), torch.full((d,), -big), torch.tensor([big, -big] * (d // 2)),
            torch.full((d,), tiny), torch.tensor([tiny, -tiny] * (d // 2)),
            torch.cat([torch.tensor([math.inf]), torch.ones(d - 1)]),
            torch.cat([torch.tensor([-math.inf, math.inf]), torch.ones(d - 2)]),
            torch.cat([torch.ones(d - 1), torch.tensor([math.nan])]), torch.full((d,), math.nan),
            torch.cat([torch.tensor([1000.0]), torch.linspace(-1, 1, d - 1)])]
    k = torch.stack(rows).to(dtype)[:, None, :]
    v = k.flip(0)
    cache = F.empty_kv4_cache(1, 1, d)
    slots = torch.arange(16, dtype=torch.int32)
    F.store_kv4(k.cuda(), v.cuda(), slots.cuda(), cache)
    got_k, got_v = F.load_kv4(cache, slots.cuda(), torch.float32)
    for got, x in ((got_k, k), (got_v, v)):
        want = R.dequantise(x).float()
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.cpu()), torch.nan_to_num(want))
        fine = torch.isfinite(x.float()).all(-1) & (x.float().abs().amax(-1) < 60000) & (x.float().abs().amax(-1) > 1e-3)
        # half a step of the row's scale, and what fp16 rounds off the scale over 15 steps
        span = (x.double().amax(-1).clamp(min=0) - x.double().amin(-1).clamp(max=0))[..., None]
        err = (got.cpu().double() - x.double()).abs()
        assert (err <= span / 15 * 0.5 + span * 2.0 ** -10)[fine].all()


@gpu
def test_store_strided_skipped_and_bad_slots(lib):
    d, heads, kv_heads, n = 128, 4, 2, 50
    qkv = randn((n, heads + 2 * kv_heads, d), 5, torch.bfloat16).cuda()
    k, v = qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    slots = torch.arange(n, dtype=torch.int32) + 3
    slots[[4, 17]] = -1
    cache = F.empty_kv4_cache(5, kv_heads, d)
    F.store_kv4(k, v, slots.cuda(), cache, check_status=True)
    got_k, got_v = F.load_kv4(cache, slots.cuda(), torch.float32, check_status=True)
    want_k, want_v = R.dequantise(k.cpu()).float(), R.dequantise(v.cpu()).float()
    want_k[[4, 17]] = 0
    want_v[[4, 17]] = 0
    assert torch.equal(got_k.cpu(), want_k) and torch.equal(got_v.cpu(), want_v)
    before = cache.pages.clone()
    for bad in (80, 2 ** 31 - 1, -2):  # the host's range check of the kernel: nothing is read or written there
        s = i32([bad])
        with pytest.raises(F.Fused3SError) as e:
            F.store_kv4(k[:1], v[:1], s, cache, check_status=True)
        assert e.value.status == _lib.F3S_ERR_BAD_FORMAT and torch.equal(cache.pages, before)
        with pytest.raises(F.Fused3SError):
            F.load_kv4(cache, s, check_status=True)
    empty = i32([])
    F.store_kv4(k[:0], v[:0], empty, cache)
    assert F.load_kv4(cache, empty)[0].shape == (0, kv_heads, d)


# --------------------------------------------------------- block tables --

def make_tables(lengths, seed, spare=3, width=None, pad=0):
    """A cache's tables before a step: (tables, free, begin, num_pages), host lists."""
    rng = random.Random(seed)
    held = [-(-c // 16) for c, _ in lengths]
    need = [-(-(c + n) // 16) for c, n in lengths]
    width = width or max(need + [1]) + 1
    ids = list(range(sum(need) + spare))
    rng.shuffle(ids)
    tables = []
    for h in held:
        tables.append([ids.pop() for _ in range(h)] + [-7] * (width - h))
    return tables, [-9] * 2 + ids, 2, sum(need) + spare


def build(lengths, tables, free, begin, num_tokens, **kw):
    return F.build_block_tables(i32([c for c, _ in lengths]), i32([n for _, n in lengths]), i32(tables), i32(free),
                                i32([begin]), num_tokens, **kw)


LENGTHS = {
    "one": [(0, 1)],
    "edges": [(0, 1), (15, 1), (16, 1), (17, 1), (31, 2), (32, 0), (0, 16), (0, 17), (1, 15), (1, 16)],
    "empty": [(0, 0), (5, 0), (16, 0)],
    "long": [(5000, 1), (0, 3), (70, 777)],
}


@gpu
@pytest.mark.parametrize("name", sorted(LENGTHS) + ["many", "mixed"])
@pytest.mark.parametrize("pad", [0, 5])
def test_block_tables(lib, name, pad):
    rng = random.Random(4)
    lengths = LENGTHS.get(name)
    if name == "many":
        lengths = [(rng.randrange(100), 1) for _ in range(1500)]
    if name == "mixed":
        lengths = [(rng.choice([0, rng.randrange(600)]), rng.choice([0, 1, 1, rng.randrange(300)])) for _ in range(513)]
    tables, free, begin, _ = make_tables(lengths, 1)
    tokens = sum(n for _, n in lengths) + pad
    for kw in ({}, {"heads": 8, "kv_heads": 2}):
        bt = build(lengths, tables, free, begin, tokens, check_status=True, **kw)
        want = R.block_tables([c for c, _ in lengths], [n for _, n in lengths], tables, free, begin, tokens)
        got = (bt.query_offsets, bt.positions, bt.slots, bt.tables, bt.free_begin)
        for g, w in zip(got, want):
            assert torch.equal(g.cpu().reshape(-1), torch.tensor(w, dtype=torch.int32).reshape(-1))


@gpu
def test_block_tables_no_requests(lib):
    empty = i32([])
    bt = F.build_block_tables(empty, empty, torch.zeros((0, 4), dtype=torch.int32, device="cuda"), empty, None, 3,
                              check_status=True)
    assert bt.query_offsets.tolist() == [0] and bt.slots.tolist() == [-1, -1, -1] and bt.free_begin.tolist() == [0]


@gpu
def test_block_tables_report_what_does_not_fit(lib):
    lengths = [(16, 20), (0, 40)]
    tables, free, begin, _ = make_tables(lengths, 2, spare=0)
    # three pages short: the last ones of the second request
    bt = build(lengths, tables, free[:-3], begin, 60, heads=1, kv_heads=1)
    want = R.block_tables([16, 0], [20, 40], tables, free[:-3], begin, 60)
    assert bt.slots.tolist() == want[2] and bt.tables.tolist() == want[3] and bt.free_begin.tolist() == [want[4]]
    assert want[2].count(-1) == 40 and bt.status() == _lib.F3S_ERR_NO_PAGES and bt.status() == 0
    # fewer token rows than tokens: what fits is as without the limit, the rest takes no page
    bt = build(lengths, tables, free, begin, 25, heads=1, kv_heads=1)
    want = R.block_tables([16, 0], [20, 5], tables, free, begin, 25)
    assert bt.slots.tolist() == want[2] and bt.tables.tolist() == want[3] and bt.query_offsets.tolist() == [0, 20, 60]
    assert bt.status() == _lib.F3S_ERR_TOO_LARGE
    # a table row too short for its request
    short = [row[:2] for row in tables]
    bt = build(lengths, short, free, begin, 60, heads=1, kv_heads=1)
    want = R.block_tables([16, 0], [16, 32], short, free, begin, 48)[2]
    assert bt.slots.tolist() == want[:16] + [-1] * 4 + want[16:] + [-1] * 8 and bt.status() == _lib.F3S_ERR_TOO_LARGE
    # a request already longer than its row
    bt = build([(40, 1)], [[3, 4]], [5], 0, 1, heads=1, kv_heads=1)
    assert bt.slots.tolist() == [-1] and bt.tables.tolist() == [[3, 4]] and bt.status() == _lib.F3S_ERR_TOO_LARGE
    # negative lengths count as 0
    bt = build([(-5, 2), (3, -1)], [[-7], [0]], [6], 0, 2)
    assert bt.slots.tolist() == [96, 97] and bt.status() == _lib.F3S_ERR_INVALID_VALUE


@gpu
def test_block_tables_strided_rows(lib):
    lengths = [(20, 3), (0, 40), (47, 2)]
    tables, free, begin, _ = make_tables(lengths, 3, width=5)
    wide = torch.full((6, 9), -5, dtype=torch.int32, device="cuda")
    wide[::2, 2:7] = i32(tables)
    bt = F.build_block_tables(i32([20, 0, 47]), i32([3, 40, 2]), wide[::2, 2:7], i32(free), i32([begin]), 45)
    want = R.block_tables([20, 0, 47], [3, 40, 2], tables, free, begin, 45)
    assert bt.tables.tolist() == want[3] and bt.slots.tolist() == want[2]
    assert (wide[1::2] == -5).all() and (wide[:, :2] == -5).all() and (wide[:, 7:] == -5).all()


# ------------------------------------------------------------ attention --

def filled_cache(num_pages, kv_heads, d, seed, size=1.0):
    cache = F.empty_kv4_cache(num_pages, kv_heads, d)
    n = num_pages * 16
    k, v = (randn((n, kv_heads, d), seed + i, torch.float16, size).cuda() for i in (0, 1))
    F.store_kv4(k, v, torch.arange(n, dtype=torch.int32, device="cuda"), cache)
    return cache


def want_attention(q, cache, tables, lengths, scale, heads):
    """float64 result and tolerances' inputs, from the cache's bytes."""
    d, kv_heads = cache.head_dim, cache.kv_heads
    pk, pv = R.page_values(cache.pages, d)
    out = torch.zeros(q.shape, dtype=torch.float64)
    q = q.double().cpu()
    first = 0
    for (c, n), row in zip(lengths, tables):
        pages = row[:-(-(c + n) // 16)]
        held = torch.tensor([p >= 0 for p in pages]).repeat_interleave(16)
        at = [max(p, 0) for p in pages]
        for h in range(heads):
            g = h // (heads // kv_heads)
            if n:
                visible = (torch.arange(len(at) * 16)[None, :] <= (c + torch.arange(n))[:, None]) & held
                out[first:first + n, h] = R.attention(q[first:first + n, h], pk[at, g].reshape(-1, d),
                                                      pv[at, g].reshape(-1, d), scale, visible)
        first += n
    return out, pk, pv


def run_attention(lengths, heads, kv_heads, d, dtype, out_dtype, seed=1, pad=0, scale=None):
    tables, free, begin, num_pages = make_tables(lengths, seed)
    cache = filled_cache(num_pages, kv_heads, d, seed)
    tokens = sum(n for _, n in lengths) + pad
    q = randn((tokens, heads, d), seed + 9, dtype).cuda()
    scale = d ** -0.5 if scale is None else scale
    bt = build(lengths, tables, free, begin, tokens, heads=heads, kv_heads=kv_heads)
    o = F.attention_kv4(q, cache, bt, scale=scale, out_dtype=out_dtype, check_status=True)
    want, pk, pv = want_attention(q, cache, bt.tables.tolist(), lengths, scale, heads)
    used = tokens - pad
    tol = R.tolerance(q.double().cpu(), pk, pv, scale, want, out_dtype)
    if used:
        R.assert_close(o[:used], want[:used], tol[:used])
    return q, cache, bt, o


@gpu
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,d", [(1, 1, 64), (8, 2, 128), (16, 2, 64), (5, 1, 128)])
def test_attention_single_tokens(lib, heads, kv_heads, d, dtype, out_dtype):
    run_attention([(0, 1), (15, 1), (16, 1), (17, 1), (300, 1), (63, 1), (0, 0), (9, 1)], heads, kv_heads, d, dtype,
                  out_dtype)


@gpu
@pytest.mark.parametrize("lengths", [
    [(0, 1)], [(0, 2), (3, 9), (40, 1), (100, 5)], [(0, 130)], [(0, 16), (0, 17), (0, 33)],
    [(260, 70), (0, 0), (0, 1), (5, 64)], [(4100, 1)], [(3000, 9), (2, 1)], [(2050, 40)]])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (12, 1, 64)])
def test_attention_lengths(lib, lengths, heads, kv_heads, d):
    run_attention(lengths, heads, kv_heads, d, torch.bfloat16, torch.bfloat16, seed=2)
    run_attention(lengths, heads, kv_heads, d, torch.float16, torch.float32, seed=3)


@gpu
def test_attention_large_group_and_long_split(lib):
    run_attention([(1200, 1), (17, 1)], 40, 1, 64, torch.float16, torch.float32)  # 40 rows of one token: two tiles
    run_attention([(12345, 1)], 2, 1, 128, torch.bfloat16, torch.float32)


@gpu
@pytest.mark.parametrize("size", [1e-4, 300.0])
def test_attention_extreme_sizes(lib, size):
    """Scales far from 1 in K and V, scores far apart."""
    lengths = [(100, 1), (37, 5)]
    tables, free, begin, num_pages = make_tables(lengths, 7)
    cache = filled_cache(num_pages, 2, 64, 5, size)
    q = randn((6, 4, 64), 8, torch.bfloat16, 1.0 / max(size, 1.0)).cuda()
    bt = build(lengths, tables, free, begin, 6, heads=4, kv_heads=2)
    o = F.attention_kv4(q, cache, bt, scale=0.5, out_dtype=torch.float32)
    want, pk, pv = want_attention(q, cache, bt.tables.tolist(), lengths, 0.5, 4)
    R.assert_close(o, want, R.tolerance(q.double().cpu(), pk, pv, 0.5, want, torch.float32))


@gpu
@pytest.mark.parametrize("lengths,heads,d", [
    ([(20, 3), (0, 5), (33, 1)], 4, 64),           # tiles of 8 query rows
    ([(20, 13), (0, 5), (33, 11)], 4, 128),        # 32
    ([(70, 90), (0, 130), (33, 60)], 4, 128),      # 128
    ([(40, 41), (0, 50), (63, 70)], 12, 64)])      # 128, groups of 6
def test_attention_leaves_out_what_is_masked(lib, lengths, heads, d):
    """NaN and garbage behind a request's end, in pages without an owner and behind
    table entries of -1; rows behind the last request stay as they were."""
    tables, free, begin, num_pages = make_tables(lengths, 11)
    cache = filled_cache(num_pages, 2, d, 3)
    used = sum(n for _, n in lengths)
    first = lengths[0][1]
    bt = build(lengths, tables, free, begin, used + 3, heads=heads, kv_heads=2)
    rows = bt.tables.tolist()
    q = randn((used + 3, heads, d), 4, torch.float16).cuda()
    out = torch.full((used + 3, heads, d), 7.0, dtype=torch.float16, device="cuda")
    F.attention_kv4(q, cache, bt, scale=0.125, out=out, check_status=True)
    assert (out[used:] == 7.0).all()
    poisoned = F.KV4Cache(torch.full_like(cache.pages, 0xff))  # every scale and zero a NaN
    for (c, n), row in zip(lengths, rows):
        s = torch.tensor([row[p // 16] * 16 + p % 16 for p in range(c + n)], dtype=torch.int32, device="cuda")
        k, v = F.load_kv4(cache, s, torch.float16)
        F.store_kv4(k, v, s, poisoned)
    # storing values that are 4-bit numbers already may move their scale by an fp16 step: compare with the cache's own
    again = torch.full_like(out, 7.0)
    F.attention_kv4(q, poisoned, bt, scale=0.125, out=again, check_status=True)
    want, pk, pv = want_attention(q[:used], poisoned, rows, lengths, 0.125, heads)
    seen = pk[torch.isfinite(pk)], pv[torch.isfinite(pv)]
    R.assert_close(again[:used], want, R.tolerance(q.double().cpu(), seen[0], seen[1], 0.125, want, torch.float16))
    assert (again[used:] == 7.0).all()
    # holes in a table: the first page of request 0, the first page of request 1
    holes = [list(r) for r in rows]
    holes[0][0] = -1
    holes[1][0] = -1
    bt.tables.copy_(i32(holes))
    for dtype in (torch.float32, torch.bfloat16):
        o = F.attention_kv4(q, cache, bt, scale=0.125, out_dtype=dtype, check_status=True)
        want, pk, pv = want_attention(q[:used], cache, holes, lengths, 0.125, heads)
        R.assert_close(o[:used], want, R.tolerance(q.double().cpu(), pk, pv, 0.125, want, dtype))
        assert (o[first:first + min(5, lengths[1][1])] == 0).all()  # their only page is missing
    # a page outside the cache is left out too, and reported
    for bad in (num_pages, 2 ** 31 - 1, -2):
        holes[1][0] = bad
        bt.tables.copy_(i32(holes))
        with pytest.raises(F.Fused3SError) as e:
            F.attention_kv4(q, cache, bt, scale=0.125, check_status=True)
        assert e.value.status == _lib.F3S_ERR_BAD_FORMAT


@gpu
@pytest.mark.parametrize("heads,kv_heads,d,dtype,out_dtype", [
    (4, 4, 64, torch.float16, torch.float16), (8, 1, 128, torch.bfloat16, torch.bfloat16),
    (6, 2, 128, torch.float16, torch.float32), (14, 2, 64, torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("lengths", [
    [(0, 300)], [(500, 129), (3, 200)], [(0, 97), (1, 300), (700, 16)], [(6000, 150)]])
def test_attention_many_new_tokens(lib, lengths, heads, kv_heads, d, dtype, out_dtype):
    """Tiles of 128 query rows: alone, ragged, behind contexts, cut into pieces."""
    run_attention(lengths, heads, kv_heads, d, dtype, out_dtype, seed=6, pad=2)


@gpu
@pytest.mark.parametrize("size", [1e-4, 300.0])
def test_attention_many_new_tokens_extreme_sizes(lib, size):
    lengths = [(60, 200)]
    tables, free, begin, num_pages = make_tables(lengths, 7)
    cache = filled_cache(num_pages, 2, 64, 5, size)
    q = randn((200, 4, 64), 8, torch.bfloat16, 1.0 / max(size, 1.0)).cuda()
    # rows of very different sizes in one tile
    q *= torch.exp2(torch.arange(200, device="cuda") % 23 - 11.0)[:, None, None].to(torch.bfloat16)
    bt = build(lengths, tables, free, begin, 200, heads=4, kv_heads=2)
    o = F.attention_kv4(q, cache, bt, scale=0.01, out_dtype=torch.float32)
    want, pk, pv = want_attention(q, cache, bt.tables.tolist(), lengths, 0.01, 4)
    R.assert_close(o, want, R.tolerance(q.double().cpu(), pk, pv, 0.01, want, torch.float32))
    for _ in range(5):
        assert torch.equal(F.attention_kv4(q, cache, bt, scale=0.01, out_dtype=torch.float32), o)


@gpu
def test_attention_rising_scores(lib):
    """Scores that keep growing along the context: the reference moves again and again."""
    for new, heads in ((1, 2), (11, 2), (150, 2)):
        lengths = [(800, new)]
        tables, free, begin, num_pages = make_tables(lengths, 3)
        cache = F.empty_kv4_cache(num_pages, 1, 64)
        bt = build(lengths, tables, free, begin, new, heads=heads, kv_heads=1)
        row = bt.tables.tolist()[0]
        n = 800 + new
        slots = i32([row[p // 16] * 16 + p % 16 for p in range(n)])
        k = torch.ones(n, 1, 64) * (torch.arange(n) / 100.0)[:, None, None]
        v = randn((n, 1, 64), 2)
        F.store_kv4(k.half().cuda(), v.half().cuda(), slots, cache)
        q = torch.ones(new, heads, 64, dtype=torch.float16, device="cuda")
        o = F.attention_kv4(q, cache, bt, scale=0.5, out_dtype=torch.float32)
        want, pk, pv = want_attention(q, cache, [row], lengths, 0.5, heads)
        R.assert_close(o, want, R.tolerance(q.double().cpu(), pk, pv, 0.5, want, torch.float32))


@gpu
@pytest.mark.parametrize("new", [4, 100])
def test_attention_nan_reaches_only_who_sees_it(lib, new):
    lengths = [(20, new)]
    tables, free, begin, num_pages = make_tables(lengths, 12)
    cache = filled_cache(num_pages, 1, 64, 3)
    bt = build(lengths, tables, free, begin, new, heads=2, kv_heads=1)
    k, v = F.load_kv4(cache, bt.slots, torch.float16)
    v[2] = math.nan
    F.store_kv4(k, v, bt.slots, cache)
    q = randn((new, 2, 64), 4, torch.float16).cuda()
    o = F.attention_kv4(q, cache, bt, out_dtype=torch.float32)
    assert torch.isfinite(o[:2]).all() and torch.isnan(o[2:]).all()
    q[1, 1, 5] = math.nan
    o = F.attention_kv4(q, cache, bt, out_dtype=torch.float32)
    assert torch.isfinite(o[0]).all() and torch.isfinite(o[1, 0]).all() and torch.isnan(o[1, 1]).all()


@gpu
def test_attention_strided_q_out_and_repeats(lib):
    lengths = [(500, 1), (40, 6), (0, 3)]
    tables, free, begin, num_pages = make_tables(lengths, 13)
    cache = filled_cache(num_pages, 2, 128, 3)
    bt = build(lengths, tables, free, begin, 10, heads=4, kv_heads=2)
    qkv = randn((10, 8, 128), 4, torch.bfloat16).cuda()
    a = F.attention_kv4(qkv[:, 2:6], cache, bt, scale=0.1)
    out = torch.empty(10, 4, 128, dtype=torch.bfloat16, device="cuda")
    b = F.attention_kv4(qkv[:, 2:6].contiguous(), cache, bt, scale=0.1, out=out)
    assert b is out and torch.equal(a, b)
    for _ in range(20):
        assert torch.equal(F.attention_kv4(qkv[:, 2:6], cache, bt, scale=0.1), a)


@gpu
@pytest.mark.parametrize("new", [1, 40, 100])
def test_attention_refuses_another_plan(lib, new):
    """A plan made for other sizes, an empty one and one of stray bytes write nothing and are reported."""
    requests, tokens, d = 3, 3 * new, 64
    made = dict(requests=requests, tokens=tokens, heads=8, kv_heads=4)
    tables = torch.zeros(requests + 1, 8, dtype=torch.int32, device="cuda")
    cache = F.empty_kv4_cache(32, 8, d)
    cache.pages.zero_()
    free = torch.arange(32, dtype=torch.int32, device="cuda")
    Q = torch.zeros(tokens + 1, 16, d, dtype=torch.float16, device="cuda")

    def call(bt, requests, tokens, heads, kv_heads):
        out = torch.full((tokens, heads, d), 7.0, device="cuda")
        size = lib.f3s_kv4_attention_scratch_size(requests, tokens, heads, kv_heads, d)
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        st = lib.f3s_kv4_attention(Q.data_ptr(), 1, heads * d, d, cache.pages.data_ptr(), 32 * 8 // kv_heads,
                                   tables.data_ptr(), tables.stride(0), bt.buffer.data_ptr(), requests, tokens, heads,
                                   kv_heads, d, 1.0, out.data_ptr(), 0, scratch.data_ptr(), size,
                                   torch.cuda.current_stream().cuda_stream)
        assert st == _lib.F3S_SUCCESS
        torch.cuda.synchronize()
        return out, bt.status()

    def build():
        return F.build_block_tables(i32([0] * requests), i32([new] * requests), tables[:requests], free, None, tokens,
                                    heads=8, kv_heads=4)

    out, status = call(build(), **made)
    assert status == _lib.F3S_SUCCESS and (out != 7).all()
    for other in (dict(heads=4), dict(heads=16, kv_heads=8), dict(kv_heads=8), dict(requests=requests + 1),
                  dict(requests=requests - 1), dict(tokens=tokens + 1), dict(tokens=tokens - 1)):
        out, status = call(build(), **{**made, **other})
        assert status == _lib.F3S_ERR_BAD_FORMAT and (out == 7).all()
    for byte in (0, 0x7f):
        bt = build()
        bt.buffer[64 : bt.plan_bytes // 4] = byte * 0x01010101  # all but the status
        out, status = call(bt, **made)
        assert status == _lib.F3S_ERR_BAD_FORMAT and (out == 7).all()


@gpu
def test_attention_offsets_beyond_32_bits(lib):
    """A cache of more than 2^32 bytes: pages at its end."""
    d, kv_heads = 128, 8
    record = kv_heads * (16 * d + 128)
    num_pages = 2 ** 32 // record + 40
    pages = torch.empty((num_pages, kv_heads, 16 * d + 128), dtype=torch.uint8, device="cuda")
    cache = F.KV4Cache(pages)
    n = 40
    table = [num_pages - 1, 0, num_pages - 3]
    slots = [table[p // 16] * 16 + p % 16 for p in range(n)]
    k, v = (randn((n, kv_heads, d), s, torch.float16).cuda() for s in (1, 2))
    F.store_kv4(k, v, i32(slots), cache, check_status=True)
    got, _ = F.load_kv4(cache, i32(slots), torch.float32)
    assert torch.equal(got.cpu(), R.dequantise(k.cpu()).float())
    tables = i32([table])
    bt = F.build_block_tables(i32([n - 1]), i32([1]), tables, i32([]), None, 1, heads=8, kv_heads=8)
    assert bt.slots.tolist() == [slots[-1]]
    q = randn((1, 8, d), 3, torch.float16).cuda()
    small = F.KV4Cache(torch.cat([pages[-3:], pages[:1]]))
    o = F.attention_kv4(q, cache, bt, check_status=True)
    bt2 = F.build_block_tables(i32([n - 1]), i32([1]), i32([[2, 3, 0]]), i32([]), None, 1, heads=8, kv_heads=8)
    assert torch.equal(o, F.attention_kv4(q, small, bt2))


# -------------------------------------------------------- graph windows --

def graph_case(n, kv_heads, d, seed, edges=4000, max_degree=200):
    g = G.powerlaw_graph(num_nodes=n, directed_edges=edges, max_degree=max_degree, seed=seed)
    return g, F.convert_csr_to_block_sparse(n, g.row_ptr, g.col_ind)


def want_graph(q, cache, fmt, scale, heads):
    d, n = cache.head_dim, fmt.num_nodes
    pk, pv = R.page_values(cache.pages, d)
    off, cols = fmt.to_host()
    q = q.double().cpu()
    out = torch.zeros(q.shape, dtype=torch.float64)
    for w in range(fmt.num_row_windows):
        at = torch.from_numpy(cols[off[w]:off[w + 1]].astype(np.int64))
        rows = slice(16 * w, min(16 * w + 16, n))
        node = (at[:, None] * 16 + torch.arange(16)).reshape(-1)
        for h in range(heads):
            g = h // (heads // cache.kv_heads)
            if len(at):
                out[rows, h] = R.attention(q[rows, h], pk[at, g].reshape(-1, d), pv[at, g].reshape(-1, d), scale,
                                           (node < n).expand(q[rows].shape[0], -1))
    return out, pk, pv


@gpu
@pytest.mark.parametrize("dtype,out_dtype", [(torch.float16, torch.float32), (torch.float16, torch.float16),
                                             (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("n,heads,kv_heads,d", [(1001, 1, 1, 64), (1001, 4, 2, 128), (640, 3, 3, 64), (17, 2, 1, 128),
                                                (5, 1, 1, 64), (16, 2, 2, 64)])
def test_graph_forward(lib, n, heads, kv_heads, d, dtype, out_dtype):
    _, fmt = graph_case(n, kv_heads, d, 3, edges=min(4000, 4 * n))
    cache = filled_cache(fmt.num_row_windows, kv_heads, d, 4)
    q = randn((n, heads, d), 5, dtype).cuda()
    o = F.fused3s_forward_kv4(q, cache, fmt, scale=d ** -0.5, out_dtype=out_dtype, check_status=True)
    want, pk, pv = want_graph(q, cache, fmt, d ** -0.5, heads)
    R.assert_close(o, want, R.tolerance(q.double().cpu(), pk, pv, d ** -0.5, want, out_dtype))


@gpu
def test_graph_forward_many_units_empty_and_hub_windows(lib):
    """More windows than one wave (one warp each), windows without a block, a hub
    that sees every block column, NaN in the rows past N of the last page."""
    n, d = 40010, 64
    rng = np.random.default_rng(0)
    src = np.concatenate([rng.integers(0, n // 2, 30000), np.full(n, 77), rng.integers(0, n // 2, 500)])
    dst = np.concatenate([rng.integers(0, n, 30000), np.arange(n), np.full(500, n - 1)])
    g = G.csr_from_edges(n, src, dst)
    fmt = F.convert_csr_to_block_sparse(n, g.row_ptr, g.col_ind)
    cache = filled_cache(fmt.num_row_windows, 1, d, 4)
    tail = torch.arange(n, fmt.num_row_windows * 16, dtype=torch.int32, device="cuda")
    nans = torch.full((tail.numel(), 1, d), math.nan, dtype=torch.float16, device="cuda")
    F.store_kv4(nans, nans, tail, cache)
    q = randn((n, 1, d), 5, torch.float16).cuda()
    o = F.fused3s_forward_kv4(q, cache, fmt, scale=0.125, check_status=True)
    want, pk, pv = want_graph(q, cache, fmt, 0.125, 1)
    seen = pk[torch.isfinite(pk)], pv[torch.isfinite(pv)]
    R.assert_close(o, want, R.tolerance(q.double().cpu(), seen[0], seen[1], 0.125, want, torch.float32))
    assert (o[n // 2 + 16:] == 0).all()
    for _ in range(5):
        assert torch.equal(F.fused3s_forward_kv4(q, cache, fmt, scale=0.125), o)
    # the hub alone, and listed more often than the format has blocks for
    for order in ([4], [4] * 300):
        out = torch.zeros_like(o)
        F.fused3s_forward_kv4(q, cache, fmt, order=i32(order), out=out, scale=0.125, check_status=True)
        R.assert_close(out[64:80], want[64:80], R.tolerance(q.double().cpu(), seen[0], seen[1], 0.125, want[64:80], torch.float32))
        assert not out[:64].any() and not out[80:].any()


@gpu
def test_graph_forward_without_edges(lib):
    fmt = F.convert_csr_to_block_sparse(50, np.zeros(51, dtype=np.int32), np.zeros(0, dtype=np.int32))
    cache = filled_cache(4, 2, 64, 1)
    q = randn((50, 2, 64), 5, torch.float16).cuda()
    o = F.fused3s_forward_kv4(q, cache, fmt, check_status=True)
    assert (o == 0).all()
    fmt = F.convert_csr_to_block_sparse(0, np.zeros(1, dtype=np.int32), np.zeros(0, dtype=np.int32))
    assert F.fused3s_forward_kv4(q[:0], cache, fmt).shape == (0, 2, 64)


@gpu
def test_graph_forward_captured_on_several_streams(lib):
    """Two captured graphs and an eager call of the same forward at the same time."""
    n, heads, d = 3000, 4, 64
    _, fmt = graph_case(n, heads, d, 5, edges=20000)
    cache = filled_cache(fmt.num_row_windows, heads, d, 4)
    order = F.generate_balanced_window_order(fmt)
    q = randn((n, heads, d), 5, torch.bfloat16).cuda()
    want = F.fused3s_forward_kv4(q, cache, fmt, order=order, scale=0.125, out_dtype=torch.bfloat16)
    outs = [torch.zeros_like(want) for _ in range(2)]
    graphs = []
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            F.fused3s_forward_kv4(q, cache, fmt, order=order, scale=0.125, out=out)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        again = F.fused3s_forward_kv4(q, cache, fmt, order=order, scale=0.125, out_dtype=torch.bfloat16)
    torch.cuda.synchronize()
    assert torch.equal(again, want) and torch.equal(outs[0], want) and torch.equal(outs[1], want)


@gpu
def test_graph_forward_subsets_and_slabs(lib):
    n, heads, d = 1001, 2, 64
    _, fmt = graph_case(n, heads, d, 9)
    cache = filled_cache(fmt.num_row_windows, heads, d, 4)
    q = randn((n, heads, d), 5, torch.float16).cuda()
    full = F.fused3s_forward_kv4(q, cache, fmt)
    out = torch.full((n, heads, d), 3.0, device="cuda")
    some = i32([5, 60, 62, 0])
    F.fused3s_forward_kv4(q, cache, fmt, order=some, out=out, check_status=True)
    mask = torch.zeros(n, dtype=torch.bool)
    for w in some.tolist():
        mask[16 * w:16 * w + 16] = True
    assert (out[~mask.cuda()] == 3.0).all()
    assert torch.allclose(out[mask.cuda()], full[mask.cuda()], rtol=0, atol=1e-5)  # other split of the blocks: fp32 sums
    for lo, hi in ((0, 320), (320, 1001)):
        slab = F.fused3s_forward_kv4(q[lo:hi], cache, fmt, q_window_base=lo // 16, check_status=True)
        assert torch.allclose(slab, full[lo:hi], rtol=0, atol=1e-5)
    before = out.clone()
    for bad in ([63], [-1], [2 ** 30]):
        with pytest.raises(F.Fused3SError) as e:
            F.fused3s_forward_kv4(q, cache, fmt, order=i32(bad), out=out, check_status=True)
        assert e.value.status == _lib.F3S_ERR_BAD_FORMAT and torch.equal(out, before)
    cols = fmt.block_col_indices.clone()
    cols[3] = 63
    bad_fmt = F.BlockSparseFormat(fmt.num_row_windows, fmt.window_offsets, cols, n)
    with pytest.raises(F.Fused3SError):
        F.fused3s_forward_kv4(q, cache, bad_fmt, check_status=True)


@gpu
def test_graph_forward_is_the_fp16_forward_of_the_loaded_values(lib):
    """The two forwards side by side: fused3s_forward on what the cache holds."""
    n, heads, d = 2708, 4, 64
    _, fmt = graph_case(n, heads, d, 2, edges=10556)
    q, k, v = (t.cuda() for t in G.make_features(n, heads, d, kind="normal", seed=3))
    cache = F.empty_kv4_cache(fmt.num_row_windows, heads, d)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    F.store_kv4(k, v, slots, cache)
    k16, v16 = F.load_kv4(cache, slots, torch.float16)
    a = F.fused3s_forward_kv4(q, cache, fmt)
    b = F.fused3s_forward(q, k16, v16, fmt)
    # K, V and P rounded to fp16 on one side: 2^-11 each of values up to max|v|, scores below 1
    assert float((a - b).abs().max()) <= 4 * 2.0 ** -11 * float(v16.abs().max())


# ------------------------------------------------- together, as in use --

@gpu
@pytest.mark.parametrize("heads,kv_heads,d,dtype", [(8, 2, 128, torch.bfloat16), (4, 4, 64, torch.float16)])
def test_serving_steps(lib, heads, kv_heads, d, dtype):
    """Prompts, then decoding steps with a request that joins and one that ends:
    tables, store and attention together against float64 over what was put in."""
    rng = random.Random(5)
    requests, width, num_pages = 4, 12, 40
    cache = F.empty_kv4_cache(num_pages, kv_heads, d)
    tables = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    ids = list(range(num_pages))
    rng.shuffle(ids)
    free, begin = i32(ids), i32([0])
    context = [0, 0, 0, 0]
    k_all = [torch.zeros(0, kv_heads, d, dtype=torch.float64) for _ in range(requests)]
    v_all = list(k_all)
    scale = d ** -0.5
    for step, new in enumerate([[21, 0, 64, 7], [1, 1, 1, 1], [1, 30, 1, 3], [1, 1, 0, 1], [2, 1, 0, 16]]):
        tokens = sum(new) + (step % 2)
        bt = F.build_block_tables(i32(context), i32(new), tables, free, begin, tokens, heads=heads, kv_heads=kv_heads,
                                  check_status=True)
        begin = bt.free_begin
        qkv = randn((tokens, heads + 2 * kv_heads, d), 100 + step, dtype).cuda()
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        F.store_kv4(k, v, bt.slots, cache, check_status=True)
        o = F.attention_kv4(q, cache, bt, scale=scale, check_status=True)
        first = 0
        for i, n in enumerate(new):
            rows = slice(first, first + n)
            k_all[i] = torch.cat([k_all[i], R.dequantise(k[rows].cpu())])
            v_all[i] = torch.cat([v_all[i], R.dequantise(v[rows].cpu())])
            for h in range(heads if n else 0):
                g = h // (heads // kv_heads)
                visible = torch.arange(context[i] + n)[None, :] <= (context[i] + torch.arange(n))[:, None]
                qh = q[rows, h].double().cpu()
                want = R.attention(qh, k_all[i][:, g], v_all[i][:, g], scale, visible)
                R.assert_close(o[rows, h], want, R.tolerance(qh, k_all[i], v_all[i], scale, want, dtype), f"{step} {i} {h}")
            first += n
        context = [c + n for c, n in zip(context, new)]


@gpu
def test_captured_step_replays_with_new_lengths(lib):
    """A decoding step captured once and replayed with other lengths, tables and
    inputs, between two eager calls; two captured graphs replayed at the same
    time on two streams."""
    requests, heads, kv_heads, d, width = 3, 8, 2, 64, 40
    num_pages = requests * width
    cache = filled_cache(num_pages, kv_heads, d, 3)
    table_rows = torch.arange(num_pages, dtype=torch.int32, device="cuda").view(requests, width)
    context, new, free = i32([5, 17, 300]), i32([1, 1, 1]), i32([0])
    q = randn((requests, heads, d), 4, torch.bfloat16).cuda()

    def step(out):
        bt = F.build_block_tables(context, new, table_rows, free, None, requests, heads=heads, kv_heads=kv_heads)
        return F.attention_kv4(q, cache, bt, scale=0.125, out=out)

    outs = [torch.zeros_like(q) for _ in range(2)]
    side = torch.cuda.Stream()
    graphs = []
    for out in outs:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(out)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(out)
        graphs.append(g)
    for lengths in ([5, 17, 300], [600, 0, 31], [15, 16, 17], [639, 639, 1]):
        context.copy_(i32(lengths))
        q.copy_(randn((requests, heads, d), lengths[0], torch.bfloat16).cuda())
        # pages are in place already: the lengths only say how many are seen
        want = step(torch.zeros_like(q))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(20):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        for out in outs:
            out.zero_()


@gpu
@pytest.mark.parametrize("lengths", [[(700, 1), (90, 2), (0, 5)], [(700, 100), (0, 333)]])
def test_calls_on_two_streams_share_tables_and_cache(lib, lengths):
    tables, free, begin, num_pages = make_tables(lengths, 21)
    cache = filled_cache(num_pages, 2, 128, 3)
    tokens = sum(n for _, n in lengths)
    bt = build(lengths, tables, free, begin, tokens, heads=8, kv_heads=2)
    qs = [randn((tokens, 8, 128), s, torch.bfloat16).cuda() for s in range(4)]
    want = [F.attention_kv4(q, cache, bt, scale=0.1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(10):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(F.attention_kv4(q, cache, bt, scale=0.1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
