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
CUDA graph) and does not synchronise unless check_status is set.
"""
from __future__ import annotations

import dataclasses
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check
from .api import _OUT_DTYPES, _WS, BlockSparseFormat, _as_nhd, _default_device, generate_balanced_window_order

PAGE_TOKENS = 16
_RECORDS = {16 * d + 128: d for d in (64, 128)}
_IN_DTYPES = {torch.float16: _lib.F3S_OUT_F16, torch.bfloat16: _lib.F3S_OUT_BF16}


class KV4Cache:
    """4-bit K / V of `num_pages` pages: pages uint8 [num_pages, kv_heads,
    16 * head_dim + 128], contiguous, on a CUDA device.  Wraps the tensor; a
    page of zeros holds zeros."""

    __slots__ = ("pages", "num_pages", "kv_heads", "head_dim")

    def __init__(self, pages: torch.Tensor):
        if pages.dtype != torch.uint8 or pages.dim() != 3:
            raise TypeError("pages must be a uint8 tensor [num_pages, kv_heads, 16 * head_dim + 128]")
        self.num_pages, self.kv_heads, record = pages.shape
        if record not in _RECORDS:
            raise ValueError("a page record has 16 * head_dim + 128 bytes, head_dim 64 or 128")
        if pages.device.type != "cuda":
            raise ValueError("pages must be on a CUDA device")
        if not pages.is_contiguous():
            raise ValueError("pages must be contiguous")
        if self.num_pages * PAGE_TOKENS >= 2 ** 31:
            raise ValueError("a cache holds fewer than 2^27 pages")
        self.head_dim = _RECORDS[record]
        self.pages = pages


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


def _check_rows(name: str, t: torch.Tensor, heads: int, head_dim: int, device: torch.device) -> torch.Tensor:
    """[rows, heads, head_dim] of fp16 or bf16 with any strides that keep
    16-byte loads: head_dim contiguous, the others multiples of 8."""
    if t.dtype not in _IN_DTYPES:
        raise TypeError(f"{name} must be float16 or bfloat16")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, with the cache")
    t = _as_nhd(t)
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != head_dim:
        raise ValueError(f"{name} must be [rows, {heads}, {head_dim}]")
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name}: head_dim must be contiguous and rows start on 16-byte boundaries")
    return t


def _rows_workspace(device: torch.device) -> torch.Tensor:
    return _WS.get(device, "kv4", 256)


def store_kv4(K: torch.Tensor, V: torch.Tensor, slots: torch.Tensor, cache: KV4Cache,
              check_status: bool = False) -> KV4Cache:
    """Quantise row i of K and V (fp16 or bf16 [n, kv_heads, head_dim], strided
    rows allowed) into slot slots[i] (int32; -1: the row is skipped) of the
    cache, in place.  Per row and head: scale = (max - min, zero included) / 15
    in fp16, a whole zero, codes rounded half to even (include/fused3s.h).
    Slots must differ.  check_status: synchronise and raise if a slot lies
    outside the cache (such rows are skipped)."""
    device = cache.pages.device
    _check_i32("slots", slots, device)
    k = _check_rows("K", K, cache.kv_heads, cache.head_dim, device)
    v = _check_rows("V", V, cache.kv_heads, cache.head_dim, device)
    n = slots.shape[0]
    if k.dtype != v.dtype:
        raise TypeError("K and V must have the same type")
    if k.shape[0] != n or v.shape[0] != n:
        raise ValueError("K, V and slots must have the same number of rows")
    lib = _lib.load()
    with torch.cuda.device(device):
        ws = _rows_workspace(device)
        stream = torch.cuda.current_stream(device).cuda_stream
        st = lib.f3s_kv4_store(k.data_ptr(), v.data_ptr(), _IN_DTYPES[k.dtype], k.stride(0), k.stride(1), v.stride(0),
                               v.stride(1), slots.data_ptr(), n, cache.pages.data_ptr(), cache.num_pages,
                               cache.kv_heads, cache.head_dim, ws.data_ptr(), ws.numel(), stream)
        check(st, "f3s_kv4_store")
        if check_status:
            check(lib.f3s_workspace_status(ws.data_ptr(), stream), "f3s_kv4_store (device)")
    return cache


def load_kv4(cache: KV4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
             check_status: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """K and V [n, kv_heads, head_dim] that the cache holds in slots[i] (int32;
    -1: zeros), rounded to `dtype` (float16, bfloat16 or float32)."""
    device = cache.pages.device
    _check_i32("slots", slots, device)
    if dtype not in _OUT_DTYPES:
        raise TypeError("dtype must be float32, float16 or bfloat16")
    n = slots.shape[0]
    k = torch.empty((n, cache.kv_heads, cache.head_dim), dtype=dtype, device=device)
    v = torch.empty_like(k)
    lib = _lib.load()
    with torch.cuda.device(device):
        ws = _rows_workspace(device)
        stream = torch.cuda.current_stream(device).cuda_stream
        st = lib.f3s_kv4_load(cache.pages.data_ptr(), cache.num_pages, cache.kv_heads, cache.head_dim,
                              slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), _OUT_DTYPES[dtype], ws.data_ptr(),
                              ws.numel(), stream)
        check(st, "f3s_kv4_load")
        if check_status:
            check(lib.f3s_workspace_status(ws.data_ptr(), stream), "f3s_kv4_load (device)")
    return k, v


@dataclasses.dataclass
class BlockTables:
    """What build_block_tables made: the tables (the caller's tensor, with the
    new pages appended), int32 per-token arrays and the attention plan."""
    tables: torch.Tensor         # int32 [requests, width]
    query_offsets: torch.Tensor  # int32 [requests + 1]: first new token of each request
    positions: torch.Tensor      # int32 [num_tokens]: position of each new token in its request
    slots: torch.Tensor          # int32 [num_tokens]: its slot in the cache, -1: none
    free_begin: torch.Tensor     # int32 [1]: first page of the free list that is still free
    plan: torch.Tensor           # device plan and status
    num_tokens: int
    heads: int
    kv_heads: int

    def status(self) -> int:
        """Synchronise and return (and clear) the status of the build and of
        the attentions run with it: F3S_SUCCESS, F3S_ERR_NO_PAGES, ..."""
        with torch.cuda.device(self.plan.device):
            return _lib.load().f3s_workspace_status(self.plan.data_ptr(),
                                                    torch.cuda.current_stream(self.plan.device).cuda_stream)


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
    lib = _lib.load()
    with torch.cuda.device(device):
        size = lib.f3s_block_tables_workspace_size(requests, num_tokens, heads, kv_heads)
        if size == 0:
            raise ValueError("too many tokens or heads for one call")
        ints = size // 4
        buf = torch.empty(ints + requests + 2 + 2 * num_tokens, dtype=torch.int32, device=device)
        plan, offsets, begin, positions, slots = buf.split((ints, requests + 1, 1, num_tokens, num_tokens))
        base = buf.data_ptr()
        o = base + size
        st = lib.f3s_block_tables(context_lens.data_ptr(), new_lens.data_ptr(), requests, tables.data_ptr(),
                                  tables.stride(0), width, free_pages.data_ptr(), free_pages.shape[0],
                                  None if free_begin is None else free_begin.data_ptr(), num_tokens, heads, kv_heads,
                                  o, o + 4 * (requests + 2), o + 4 * (requests + 2 + num_tokens),
                                  o + 4 * (requests + 1), base, size, torch.cuda.current_stream(device).cuda_stream)
        check(st, "f3s_block_tables")
    bt = BlockTables(tables, offsets, positions, slots, begin, plan, num_tokens, heads, kv_heads)
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
    device = cache.pages.device
    heads, head_dim = bt.heads, cache.head_dim
    if heads == 0 or bt.kv_heads != cache.kv_heads:
        raise ValueError("the block tables were built for other heads (pass heads and kv_heads to build_block_tables)")
    q = _check_rows("Q", Q, heads, head_dim, device)
    if q.shape[0] != bt.num_tokens:
        raise ValueError("Q must have num_tokens rows")
    if bt.tables.device != device:
        raise ValueError("the block tables and the cache must be on the same device")
    if out is None:
        out = torch.empty(Q.shape, dtype=out_dtype or Q.dtype, device=device)
    elif out.shape != Q.shape or not out.is_contiguous() or out.device != device or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor shaped like Q, with the cache")
    if out.dtype not in _OUT_DTYPES:
        raise ValueError("O must be float32, float16 or bfloat16")
    requests = bt.tables.shape[0]
    lib = _lib.load()
    if requests == 0 or bt.num_tokens == 0:
        return out
    with torch.cuda.device(device):
        size = lib.f3s_kv4_attention_scratch_size(requests, bt.num_tokens, heads, cache.kv_heads, head_dim)
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        st = lib.f3s_kv4_attention(q.data_ptr(), _IN_DTYPES[q.dtype], q.stride(0), q.stride(1), cache.pages.data_ptr(),
                                   cache.num_pages, bt.tables.data_ptr(), bt.tables.stride(0), bt.plan.data_ptr(),
                                   requests, bt.num_tokens, heads, cache.kv_heads, head_dim, scale, out.data_ptr(),
                                   _OUT_DTYPES[out.dtype], ws.data_ptr(), size,
                                   torch.cuda.current_stream(device).cuda_stream)
        check(st, "f3s_kv4_attention")
    if check_status:
        check(bt.status(), "f3s_kv4_attention (device)")
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
    device = cache.pages.device
    q3 = _as_nhd(Q)
    if q3.dim() != 3 or q3.shape[2] != cache.head_dim or q3.shape[1] == 0 or q3.shape[1] % cache.kv_heads:
        raise ValueError("Q must be [rows, heads, head_dim] with the cache's head_dim and heads a multiple of its kv_heads")
    q_rows, heads, head_dim = q3.shape
    _check_rows("Q", Q, heads, head_dim, device)
    if not Q.is_contiguous():
        raise ValueError("Q must be contiguous")
    if fmt.window_offsets.device != device:
        raise ValueError("the format and the cache must be on the same device")
    if cache.num_pages < fmt.num_row_windows:
        raise ValueError("the cache must have a page for every block column of the graph")
    if order is None:
        if q_window_base == 0 and q_rows == fmt.num_nodes:
            order = generate_balanced_window_order(fmt)
        else:
            order = torch.arange(q_window_base, q_window_base + (q_rows + 15) // 16, dtype=torch.int32, device=device)
    order = order.to(device=device, dtype=torch.int32).contiguous()
    if out is None:
        out = torch.empty(Q.shape, dtype=out_dtype, device=device)
    elif out.shape != Q.shape or not out.is_contiguous() or out.device != device or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor shaped like Q, with the cache")
    if out.dtype not in _OUT_DTYPES:
        raise ValueError("O must be float32, float16 or bfloat16")
    lib = _lib.load()
    with torch.cuda.device(device):
        ws = _rows_workspace(device)
        stream = torch.cuda.current_stream(device).cuda_stream
        items = order.shape[0]
        blocks = fmt.num_blocks
        size = lib.f3s_kv4_forward_scratch_size(items, blocks, heads, head_dim)
        scratch = torch.empty(size, dtype=torch.uint8, device=device)
        st = lib.f3s_kv4_forward(q3.data_ptr(), _IN_DTYPES[Q.dtype], cache.pages.data_ptr(), cache.num_pages,
                                 out.data_ptr(), _OUT_DTYPES[out.dtype], fmt.window_offsets.data_ptr(), fmt.cols_ptr,
                                 order.data_ptr(), items, blocks, fmt.num_nodes, heads, cache.kv_heads, head_dim,
                                 scale, q_window_base, q_rows, ws.data_ptr(), ws.numel(), scratch.data_ptr(), size,
                                 stream)
        check(st, "f3s_kv4_forward")
        if check_status:
            check(lib.f3s_workspace_status(ws.data_ptr(), stream), "f3s_kv4_forward (device)")
    return out
