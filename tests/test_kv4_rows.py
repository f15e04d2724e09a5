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


# ----------------------------------------------- scores beyond whole steps --

@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ratio", [2.0 ** 30, 2.0 ** 100])
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
