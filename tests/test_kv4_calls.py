"""Calls of the 4-bit K / V operators as a program makes them: after an error,
from several threads, in several captured graphs, in place, beside other
kernels."""
import contextlib
import random
import threading
import time

import pytest
import torch

import fused3s_b200 as F
import kv4_ref as R
import test_kv4 as T
from fused3s_b200 import _lib, api, kv4

gpu = pytest.mark.gpu


def test_first_caches_of_two_threads_share_one_status_word(monkeypatch):
    """Two threads that make a device's first cache get the same word, which lives on
    (the device's calls stand-ins that give way to the other thread)."""
    made = []

    class Stream:
        def synchronize(self):
            time.sleep(0.05)

    def zeros(n, dtype=None, device=None):
        made.append(torch.empty(n, dtype=dtype))
        time.sleep(0.05)
        return made[-1]

    monkeypatch.setattr(kv4, "_STATUS", {})
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    monkeypatch.setattr(torch, "zeros", zeros)
    device, got, both = torch.device("cuda", 0), [None, None], threading.Barrier(2)

    def first_cache(i):
        both.wait()
        got[i] = kv4._status(device)

    threads = [threading.Thread(target=first_cache, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and got[0] is made[0] and got[1] is made[0] and kv4._STATUS[0] is made[0]


class OrderLibrary:
    """Stands in for libfused3s.so: notes the scratch of each sort."""

    def __init__(self):
        self.scratch = []

    def f3s_window_order_workspace_size(self, n):
        return 1000 + n

    def f3s_window_order(self, offsets, n, order, ws, ws_bytes, stream):
        self.scratch.append((ws, ws_bytes))
        return 0


def test_the_order_of_windows_keeps_no_scratch(monkeypatch):
    """Nothing that a captured sort writes to stays behind for the next one to share or replace."""
    fake = OrderLibrary()
    monkeypatch.setattr(api._lib, "load", lambda: fake)
    monkeypatch.setattr(api, "_stream_ptr", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(api, "_WS", api._WorkspaceCache())
    for n in (70, 7000):
        offsets = torch.zeros(n + 1, dtype=torch.int32)
        fmt = F.BlockSparseFormat(n, offsets, torch.zeros(0, dtype=torch.int32), 16 * n)
        assert api.generate_balanced_window_order(fmt).shape == (n,)
    assert [size for _, size in fake.scratch] == [1070, 8000] and not api._WS._ws


@gpu
def test_captured_forwards_sort_their_windows_apart(lib):
    """Forwards without an order, of graphs of three sizes, captured one after another
    and replayed at the same time on streams of their own."""
    d, heads, cases = 64, 2, []
    for n, edges in ((3000, 20000), (40000, 90000), (9000, 50000)):
        _, fmt = T.graph_case(n, heads, d, 5, edges=edges)
        cache = T.filled_cache(fmt.num_row_windows, heads, d, 4)
        q = T.randn((n, heads, d), 5, torch.float16).cuda()
        want = F.fused3s_forward_kv4(q, cache, fmt, scale=0.125, check_status=True)
        graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(want)
        with torch.cuda.graph(graph):
            F.fused3s_forward_kv4(q, cache, fmt, scale=0.125, out=out)
        cases.append((graph, out, want, torch.cuda.Stream(), (fmt, cache, q)))  # what the graph reads lives as long
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, out, _, stream, _ in cases:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, want, _, _ in cases)


@gpu
def test_a_cache_keeps_its_status_word(lib):
    cache = F.empty_kv4_cache(2, 1, 64)
    assert cache.status_word.data_ptr() == cache.status_ptr and cache.status_word is kv4._STATUS[cache.device.index]


@gpu
@pytest.mark.parametrize("heads", [1, 2, 4])
def test_an_earlier_timeout_stops_no_later_forward(lib, heads):
    """The device's status word keeps a timeout until it is read; a later forward's
    waits do not go by it."""
    n, d = 3000, 64
    _, fmt = T.graph_case(n, heads, d, 5, edges=20000)
    cache = T.filled_cache(fmt.num_row_windows, heads, d, 4)
    q = T.randn((n, heads, d), 5, torch.float16).cuda()
    want = F.fused3s_forward_kv4(q, cache, fmt, scale=0.125, check_status=True)
    kv4._status(cache.device).view(torch.int32)[2] = _lib.F3S_ERR_TIMEOUT  # as a wait that ran out leaves it
    for _ in range(20):
        assert torch.equal(F.fused3s_forward_kv4(q, cache, fmt, scale=0.125), want)
    with pytest.raises(F.Fused3SError) as e:
        F.fused3s_forward_kv4(q, cache, fmt, check_status=True)
    assert e.value.status == _lib.F3S_ERR_TIMEOUT
    F.fused3s_forward_kv4(q, cache, fmt, check_status=True)


@gpu
@pytest.mark.parametrize("heads,kv_heads", [(0, 0), (32, 8)])
def test_block_tables_in_place(lib, heads, kv_heads):
    """The free list's first page updated in place, for more tokens than one block
    takes, while another stream keeps the SMs busy."""
    rng = random.Random(3)
    lengths = [(rng.choice([0, rng.randrange(3000)]), rng.randrange(400, 1777)) for _ in range(41)]
    tables, free, begin, _ = T.make_tables(lengths, 2)
    tokens, requests, width = sum(n for _, n in lengths), len(lengths), len(tables[0])
    want = R.block_tables([c for c, _ in lengths], [n for _, n in lengths], tables, free, begin, tokens)
    size = lib.f3s_block_tables_workspace_size(requests, tokens, heads, kv_heads)
    context, new, free = T.i32([c for c, _ in lengths]), T.i32([n for _, n in lengths]), T.i32(free)
    offsets, positions, slots = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (requests + 1, tokens, tokens))
    plan = torch.empty(size, dtype=torch.uint8, device="cuda")
    busy, side = torch.randn(4096, 4096, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        table, word = T.i32(tables), T.i32([begin])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            busy @ busy
        st = lib.f3s_block_tables(context.data_ptr(), new.data_ptr(), requests, table.data_ptr(), width, width,
                                  free.data_ptr(), free.numel(), word.data_ptr(), tokens, heads, kv_heads,
                                  offsets.data_ptr(), positions.data_ptr(), slots.data_ptr(), word.data_ptr(),
                                  plan.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        assert st == 0 and lib.f3s_workspace_status(plan.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        got = (offsets.tolist(), positions.tolist(), slots.tolist(), table.tolist(), word.item())
        assert got == want


@gpu
def test_graph_forward_keeps_to_the_sm_limit(lib):
    """Few blocks give the same result and take many times as long as all of them."""
    n, heads, d = 40000, 4, 64
    _, fmt = T.graph_case(n, heads, d, 5, edges=400000)
    cache = T.filled_cache(fmt.num_row_windows, heads, d, 4)
    order = F.generate_balanced_window_order(fmt)
    q = T.randn((n, heads, d), 5, torch.float16).cuda()

    def run():
        out = F.fused3s_forward_kv4(q, cache, fmt, order=order, scale=0.125, check_status=True)
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        F.fused3s_forward_kv4(q, cache, fmt, order=order, scale=0.125, out=out)
        b.record()
        torch.cuda.synchronize()
        return out, a.elapsed_time(b)

    want, all_of_them = run()
    try:
        F.set_forward_sm_limit(8)
        got, eight = run()
    finally:
        F.set_forward_sm_limit(0)
    assert torch.equal(got, want) and eight > 4 * all_of_them
