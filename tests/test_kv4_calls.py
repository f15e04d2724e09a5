"""Calls of the 4-bit K / V operators as a program makes them: after an error,
from several threads, in several captured graphs, in place, beside other
kernels."""
import pytest
import torch

import fused3s_b200 as F
import test_kv4 as T
from fused3s_b200 import _lib, kv4

gpu = pytest.mark.gpu


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
