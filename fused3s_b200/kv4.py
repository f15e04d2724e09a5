"""K / V held in 4 bits: the cache, the store that fills it, the block tables
that address it, and attention over it.

  KV4Cache, empty_kv4_cache   pages of 16 tokens (one block column) per K/V head
  store_kv4, load_kv4         rows of K / V into slots of the cache, and back
  build_block_tables          block tables, slot map and attention plan from
                              request lengths, in one launch
  attention_kv4               causal attention of each request's new tokens,
                              one or many, over its pages
  fused3s_forward_kv4         fused3s_forward with K / V in 4 bits: block column
                              c of the graph's format is page c of the cache

Decoding or prefilling a batch, once per step and then per layer:

    bt = build_block_tables(context_lens, new_lens, tables, free_pages, free_begin, num_tokens,
                            heads=H, kv_heads=G)
    store_kv4(k, v, bt.slots, cache)
    o = attention_kv4(q, cache, bt, scale=d ** -0.5)

A graph's K / V: store_kv4(K, V, torch.arange(N, dtype=torch.int32, ...), cache),
then fused3s_forward_kv4(Q, cache, fmt, order=order).

The byte layout of a page is described in include/fused3s.h.  Every call runs
on the current stream of its tensors' device, allocates its outputs and
scratch from torch's allocator on that stream (so it can be captured into a
CUDA graph) and does not synchronise unless check_status is set.  Errors that
a kernel finds in store_kv4, load_kv4 and fused3s_forward_kv4 are kept in one
status word per device until a call with check_status raises them; those of
build_block_tables and attention_kv4 in the block tables (status()).
"""
from __future__ import annotations

import functools
import threading
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check
from .api import _OUT_DTYPES, BlockSparseFormat, _default_device, generate_balanced_window_order

PAGE_TOKENS = 16
_RECORDS = {16 * d + 128: d for d in (64, 128)}
_IN_DTYPES = {torch.float16: _lib.F3S_OUT_F16, torch.bfloat16: _lib.F3S_OUT_BF16}


def _on(device: torch.device):
    """The device to switch to for a call, or None where it is current already."""
    return None if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the same number without the Stream object, where torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


_STATUS = {}  # one status word per device for store, load and the graph forward
_STATUS_LOCK = threading.Lock()


def _status(device: torch.device) -> torch.Tensor:
    """The device's status word: kernels only set it where it is 0, so all streams
    and captured graphs share it.  Made before any capture, with the first cache,
    once whichever threads ask for it."""
    with _STATUS_LOCK:
        ws = _STATUS.get(device.index)
        if ws is None:
            with torch.cuda.device(device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("make the device's first KV4Cache before capturing a CUDA graph")
                ws = torch.zeros(256, dtype=torch.uint8, device=device)
                torch.cuda.current_stream(device).synchronize()
            _STATUS[device.index] = ws
        return ws


class KV4Cache:
    """4-bit K / V of `num_pages` pages: pages uint8 [num_pages, kv_heads,
    16 * head_dim + 128], contiguous, on a CUDA device.  Wraps the tensor; a
    page of zeros holds zeros."""

    __slots__ = ("pages", "num_pages", "kv_heads", "head_dim", "device", "status_word", "status_ptr")

    def __init__(self, pages: torch.Tensor):
        if pages.dtype != torch.uint8 or pages.dim() != 3:
            raise TypeError("pages must be a uint8 tensor [num_pages, kv_heads, 16 * head_dim + 128]")
        self.num_pages, self.kv_heads, record = pages.shape
        if record not in _RECORDS:
            raise ValueError("a page record has 16 * head_dim + 128 bytes, head_dim 64 or 128")
        if not pages.is_cuda:
            raise ValueError("pages must be on a CUDA device")
        if not pages.is_contiguous():
            raise ValueError("pages must be contiguous")
        if self.num_pages * PAGE_TOKENS >= 2 ** 31:
            raise ValueError("a cache holds fewer than 2^27 pages")
        self.head_dim = _RECORDS[record]
        self.pages = pages
        self.device = pages.device
        self.status_word = _status(self.device)
        self.status_ptr = self.status_word.data_ptr()


def empty_kv4_cache(num_pages: int, kv_heads: int, head_dim: int, device=None) -> KV4Cache:
    """A cache of zeros."""
    if head_dim not in _RECORDS.values():
        raise ValueError("head_dim must be 64 or 128")
    return KV4Cache(torch.zeros((num_pages, kv_heads, 16 * head_dim + 128), dtype=torch.uint8,
                                device=_default_device(device)))


def _check_i32(name: str, t: torch.Tensor, device: torch.device, dim: int = 1) -> None:
    if t.dtype != torch.int32 or t.dim() != dim:
        raise TypeError(f"{name} must be an int32 tensor of {dim} dimension{'s' if dim > 1 else ''}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if dim == 1 and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_rows(name: str, t: torch.Tensor, heads: int, head_dim: int, device: torch.device):
    """(pointer, strides in elements) of [rows, heads, head_dim] fp16 or bf16 with any
    strides that keep 16-byte loads: head_dim contiguous, the others multiples of 8."""
    if t.dtype not in _IN_DTYPES:
        raise TypeError(f"{name} must be float16 or bfloat16")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, with the cache")
    shape, strides, ptr = t.shape, t.stride(), t.data_ptr()
    if len(shape) == 2:
        shape, strides = (shape[0], 1, shape[1]), (strides[0], 0, strides[1])
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim:
        raise ValueError(f"{name} must be [rows, {heads}, {head_dim}]")
    if strides[2] != 1 or (strides[0] | strides[1]) & 7 or ptr & 15:
        raise ValueError(f"{name}: head_dim must be contiguous and rows start on 16-byte boundaries")
    return ptr, strides


def store_kv4(K: torch.Tensor, V: torch.Tensor, slots: torch.Tensor, cache: KV4Cache,
              check_status: bool = False) -> KV4Cache:
    """Quantise row i of K and V (fp16 or bf16 [n, kv_heads, head_dim], strided
    rows allowed) into slot slots[i] (int32; -1: the row is skipped) of the
    cache, in place.  Per row and head: scale = (max - min, zero included) / 15
    in fp16, a whole zero, codes rounded half to even (include/fused3s.h).
    Slots must differ.  check_status: synchronise and raise if a slot lies
    outside the cache (such rows are skipped)."""
    device = cache.device
    _check_i32("slots", slots, device)
    k, ks = _check_rows("K", K, cache.kv_heads, cache.head_dim, device)
    v, vs = _check_rows("V", V, cache.kv_heads, cache.head_dim, device)
    n = slots.shape[0]
    if K.dtype != V.dtype:
        raise TypeError("K and V must have the same type")
    if K.shape[0] != n or V.shape[0] != n:
        raise ValueError("K, V and slots must have the same number of rows")
    switch = _on(device)
    if switch is not None:
        with switch:
            return store_kv4(K, V, slots, cache, check_status)
    lib = _lib.load()
    stream = _raw_stream(device.index)
    ws = cache.status_ptr
    st = lib.f3s_kv4_store(k, v, _IN_DTYPES[K.dtype], ks[0], ks[1], vs[0], vs[1], slots.data_ptr(), n,
                           cache.pages.data_ptr(), cache.num_pages, cache.kv_heads, cache.head_dim, ws, 256, stream)
    if st:
        check(st, "f3s_kv4_store")
    if check_status:
        check(lib.f3s_workspace_status(ws, stream), "f3s_kv4_store (device)")
    return cache


def load_kv4(cache: KV4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
             check_status: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """K and V [n, kv_heads, head_dim] that the cache holds in slots[i] (int32;
    -1: zeros), rounded to `dtype` (float16, bfloat16 or float32)."""
    device = cache.device
    _check_i32("slots", slots, device)
    if dtype not in _OUT_DTYPES:
        raise TypeError("dtype must be float32, float16 or bfloat16")
    switch = _on(device)
    if switch is not None:
        with switch:
            return load_kv4(cache, slots, dtype, check_status)
    n = slots.shape[0]
    k = torch.empty((n, cache.kv_heads, cache.head_dim), dtype=dtype, device=device)
    v = torch.empty_like(k)
    lib = _lib.load()
    stream = _raw_stream(device.index)
    ws = cache.status_ptr
    st = lib.f3s_kv4_load(cache.pages.data_ptr(), cache.num_pages, cache.kv_heads, cache.head_dim, slots.data_ptr(), n,
                          k.data_ptr(), v.data_ptr(), _OUT_DTYPES[dtype], ws, 256, stream)
    if st:
        check(st, "f3s_kv4_load")
    if check_status:
        check(lib.f3s_workspace_status(ws, stream), "f3s_kv4_load (device)")
    return k, v


class BlockTables:
    """What build_block_tables made.

    tables         int32 [requests, width]: the caller's tensor, with the new pages appended
    query_offsets  int32 [requests + 1]: first new token of each request
    positions      int32 [num_tokens]: position of each new token in its request
    slots          int32 [num_tokens]: its slot in the cache, -1: none
    free_begin     int32 [1]: first page of the free list that is still free
    num_tokens, heads, kv_heads: as passed; `buffer` holds the device plan, the
    status and the arrays above."""

    __slots__ = ("tables", "num_tokens", "heads", "kv_heads", "buffer", "plan_bytes", "requests", "_views")

    def __init__(self, tables, num_tokens, heads, kv_heads, buffer, plan_bytes):
        self.tables, self.num_tokens, self.heads, self.kv_heads = tables, num_tokens, heads, kv_heads
        self.buffer, self.plan_bytes, self.requests, self._views = buffer, plan_bytes, tables.shape[0], None

    def _array(self, k: int) -> torch.Tensor:
        if self._views is None:
            n = self.num_tokens
            self._views = self.buffer.split_with_sizes((self.plan_bytes // 4, self.requests + 1, 1, n, n))
        return self._views[k]

    @property
    def query_offsets(self) -> torch.Tensor:
        return self._array(1)

    @property
    def free_begin(self) -> torch.Tensor:
        return self._array(2)

    @property
    def positions(self) -> torch.Tensor:
        return self._array(3)

    @property
    def slots(self) -> torch.Tensor:
        return self._array(4)

    def status(self) -> int:
        """Synchronise and return (and clear) the status of the build and of
        the attentions run with it: F3S_SUCCESS, F3S_ERR_NO_PAGES, ..."""
        device = self.buffer.device
        with torch.cuda.device(device):
            return _lib.load().f3s_workspace_status(self.buffer.data_ptr(), _raw_stream(device.index))


@functools.lru_cache(maxsize=4096)
def _plan_bytes(index: int, requests: int, num_tokens: int, heads: int, kv_heads: int) -> int:
    return _lib.load().f3s_block_tables_workspace_size(requests, num_tokens, heads, kv_heads)


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(index: int, requests: int, num_tokens: int, heads: int, kv_heads: int, head_dim: int) -> int:
    return _lib.load().f3s_kv4_attention_scratch_size(requests, num_tokens, heads, kv_heads, head_dim)


def build_block_tables(context_lens: torch.Tensor, new_lens: torch.Tensor, tables: torch.Tensor,
                       free_pages: torch.Tensor, free_begin: Optional[torch.Tensor], num_tokens: int,
                       heads: int = 0, kv_heads: int = 0, check_status: bool = False) -> BlockTables:
    """Block tables, slot map and attention plan of a step.

    context_lens, new_lens: int32 [requests], tokens cached and tokens to add.
    tables: int32 [requests, width], rows of any stride; row i holds the
    request's ceil(context / 16) pages and gets the new ones appended, in place.
    free_pages: int32, free pages in the order they are handed out, from index
    free_begin[0] (int32 [1]; None: 0) on; the result's free_begin is where the
    next step goes on.  num_tokens: length of the token arrays, at least the new
    tokens (the sum of new_lens; a padded batch may have more).
    heads, kv_heads: what attention_kv4 will be called with (0: no attention).

    One launch; nothing is read back.  status() (or check_status) tells of a
    free list that ran out (those tokens have slot -1) or of lengths that do
    not fit."""
    device = tables.device
    if device.type != "cuda":
        raise ValueError("tables must be on a CUDA device")
    _check_i32("tables", tables, device, 2)
    _check_i32("context_lens", context_lens, device)
    _check_i32("new_lens", new_lens, device)
    _check_i32("free_pages", free_pages, device)
    requests, width = tables.shape
    if context_lens.shape[0] != requests or new_lens.shape[0] != requests:
        raise ValueError("context_lens, new_lens and tables must have one entry per request")
    if width > 1 and tables.stride(1) != 1 or requests > 1 and tables.stride(0) < width:
        raise ValueError("the rows of tables must be contiguous and must not overlap")
    if free_begin is not None:
        _check_i32("free_begin", free_begin, device)
        if free_begin.shape[0] != 1:
            raise ValueError("free_begin must have one entry")
    if heads < 0 or kv_heads < 0 or (heads == 0) != (kv_heads == 0) or (kv_heads and heads % kv_heads):
        raise ValueError("heads must be a multiple of kv_heads")
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    switch = _on(device)
    if switch is not None:
        with switch:
            return build_block_tables(context_lens, new_lens, tables, free_pages, free_begin, num_tokens, heads,
                                      kv_heads, check_status)
    lib = _lib.load()
    size = _plan_bytes(device.index, requests, num_tokens, heads, kv_heads)
    if size == 0:
        raise ValueError("too many tokens or heads for one call")
    buf = torch.empty(size // 4 + requests + 2 + 2 * num_tokens, dtype=torch.int32, device=device)
    base = buf.data_ptr()
    o = base + size
    st = lib.f3s_block_tables(context_lens.data_ptr(), new_lens.data_ptr(), requests, tables.data_ptr(),
                              tables.stride(0), width, free_pages.data_ptr(), free_pages.shape[0],
                              None if free_begin is None else free_begin.data_ptr(), num_tokens, heads, kv_heads,
                              o, o + 4 * (requests + 2), o + 4 * (requests + 2 + num_tokens), o + 4 * (requests + 1),
                              base, size, _raw_stream(device.index))
    if st:
        check(st, "f3s_block_tables")
    bt = BlockTables(tables, num_tokens, heads, kv_heads, buf, size)
    if check_status:
        check(bt.status(), "f3s_block_tables (device)")
    return bt


def attention_kv4(Q: torch.Tensor, cache: KV4Cache, bt: BlockTables, scale: float = 1.0,
                  out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                  check_status: bool = False) -> torch.Tensor:
    """O = softmax(scale * Q K^T) V, causal, over each request's pages.

    Q: fp16 or bf16 [num_tokens, heads, head_dim] (strided rows allowed), the
    new tokens of all requests in a row (bt.query_offsets); the token at
    position p sees positions 0 ... p of its request, whose K / V are in the
    cache already (store_kv4 first).  Query head h reads K/V head
    h // (heads // kv_heads).  Scores are multiplied by `scale` (1.0 as in
    fused3s_forward; language models pass head_dim ** -0.5).
    out: optional contiguous result of Q's shape; rows behind the last new
    token are left as they were.  out_dtype: float32, float16 or bfloat16
    (default Q's).  check_status: synchronise and raise if a table entry lies
    outside the cache (such pages are left out)."""
    device = cache.device
    heads, kv_heads, head_dim = bt.heads, cache.kv_heads, cache.head_dim
    if heads == 0 or bt.kv_heads != kv_heads:
        raise ValueError("the block tables were built for other heads (pass heads and kv_heads to build_block_tables)")
    q, qs = _check_rows("Q", Q, heads, head_dim, device)
    if Q.shape[0] != bt.num_tokens:
        raise ValueError("Q must have num_tokens rows")
    if bt.buffer.device != device:
        raise ValueError("the block tables and the cache must be on the same device")
    out = _result(Q, out, out_dtype or Q.dtype, device)
    if bt.requests == 0 or bt.num_tokens == 0:
        return out
    switch = _on(device)
    if switch is not None:
        with switch:
            return attention_kv4(Q, cache, bt, scale, out, None, check_status)
    lib = _lib.load()
    size = _scratch_bytes(device.index, bt.requests, bt.num_tokens, heads, kv_heads, head_dim)
    scratch = torch.empty(size, dtype=torch.uint8, device=device)
    st = lib.f3s_kv4_attention(q, _IN_DTYPES[Q.dtype], qs[0], qs[1], cache.pages.data_ptr(), cache.num_pages,
                               bt.tables.data_ptr(), bt.tables.stride(0), bt.buffer.data_ptr(), bt.requests,
                               bt.num_tokens, heads, kv_heads, head_dim, scale, out.data_ptr(), _OUT_DTYPES[out.dtype],
                               scratch.data_ptr(), size, _raw_stream(device.index))
    if st:
        check(st, "f3s_kv4_attention")
    if check_status:
        check(bt.status(), "f3s_kv4_attention (device)")
    return out


def _result(Q: torch.Tensor, out: Optional[torch.Tensor], dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if out is None:
        if dtype not in _OUT_DTYPES:
            raise ValueError("O must be float32, float16 or bfloat16")
        return torch.empty(Q.shape, dtype=dtype, device=device)
    if out.shape != Q.shape or not out.is_contiguous() or out.device != device or out.data_ptr() & 15:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor shaped like Q, with the cache")
    if out.dtype not in _OUT_DTYPES:
        raise ValueError("O must be float32, float16 or bfloat16")
    return out


def fused3s_forward_kv4(Q: torch.Tensor, cache: KV4Cache, fmt: BlockSparseFormat,
                        order: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                        q_window_base: int = 0, check_status: bool = False, scale: float = 1.0,
                        out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """fused3s_forward with K / V held in 4 bits: O = block-sparse
    softmax(scale * Q K^T) V over the graph's row windows.

    Q: fp16 or bf16 [q_rows, heads, head_dim] (or [q_rows, head_dim] for one
    head), contiguous, rows 16 * q_window_base ...  cache: page c holds the nodes
    16 c ... 16 c + 15 (node v in slot v), at least ceil(N / 16) pages; heads
    may be a multiple of its kv_heads (query head h reads K/V head
    h // (heads // kv_heads)).  order, out, q_window_base, check_status and
    out_dtype as in fused3s_forward."""
    device = cache.device
    q_rows, heads, head_dim = Q.shape if Q.dim() == 3 else (Q.shape[0], 1, Q.shape[-1])
    if Q.dim() not in (2, 3) or head_dim != cache.head_dim or heads == 0 or heads % cache.kv_heads:
        raise ValueError("Q must be [rows, heads, head_dim] with the cache's head_dim and heads a multiple of its kv_heads")
    q, _ = _check_rows("Q", Q, heads, head_dim, device)
    if not Q.is_contiguous():
        raise ValueError("Q must be contiguous")
    if fmt.window_offsets.device != device:
        raise ValueError("the format and the cache must be on the same device")
    if cache.num_pages < fmt.num_row_windows:
        raise ValueError("the cache must have a page for every block column of the graph")
    switch = _on(device)
    if switch is not None:
        with switch:
            return fused3s_forward_kv4(Q, cache, fmt, order, out, q_window_base, check_status, scale, out_dtype)
    if order is None:
        if q_window_base == 0 and q_rows == fmt.num_nodes:
            order = generate_balanced_window_order(fmt)
        else:
            order = torch.arange(q_window_base, q_window_base + (q_rows + 15) // 16, dtype=torch.int32, device=device)
    elif order.dtype != torch.int32 or order.device != device or not order.is_contiguous():
        order = order.to(device=device, dtype=torch.int32).contiguous()
    out = _result(Q, out, out_dtype, device)
    lib = _lib.load()
    stream = _raw_stream(device.index)
    ws = cache.status_ptr
    items, blocks = order.numel(), fmt.num_blocks
    size = lib.f3s_kv4_forward_scratch_size(items, blocks, heads, cache.kv_heads, head_dim)
    scratch = torch.empty(size, dtype=torch.uint8, device=device)
    st = lib.f3s_kv4_forward(q, _IN_DTYPES[Q.dtype], cache.pages.data_ptr(), cache.num_pages, out.data_ptr(),
                             _OUT_DTYPES[out.dtype], fmt.window_offsets.data_ptr(), fmt.cols_ptr, order.data_ptr(), items,
                             blocks, fmt.num_nodes, heads, cache.kv_heads, head_dim, scale, q_window_base, q_rows, ws, 256,
                             scratch.data_ptr(), size, stream)
    if st:
        check(st, "f3s_kv4_forward")
    if check_status:
        check(lib.f3s_workspace_status(ws, stream), "f3s_kv4_forward (device)")
    return out
