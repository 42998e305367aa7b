"""Tokens one at a time over a cache beside the whole sequence at once: the outputs of the one are those of the
other, each within its tolerance of float64 (test_masked_attention_gpu.py), so within the sum of both."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention, prefix_attention

from test_masked_attention_gpu import DTYPES, heads, i32, reference
from test_prefix_attention_gpu import joined, shared
from test_window_attention_gpu import see

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('t,window,sinks', [(70, 12, 2), (200, 90, 1)])
def test_windows(device, t, window, sinks, dtype):
    q, k, v = heads(device, dtype, 1, t, t, 4, 2, 64)
    at = torch.arange(t)
    side = Tokens(i32(at * 0, device), i32(at, device))
    whole = masked_attention(q, k, v, 0.125, keys=side, window=window, sinks=sinks)
    tol = reference(q, k, v, 0.125, seen=see(at * 0, at * 0, at, at, window, sinks))[1]
    cache_k, cache_v = torch.full_like(k, float('nan')), torch.full_like(v, float('inf'))   # never written
    for i in range(t):
        cache_k[:, i], cache_v[:, i] = k[:, i], v[:, i]
        last = i32(at[i:i + 1], device)
        one = masked_attention(q[:, i:i + 1], cache_k, cache_v, 0.125, keys=side, window=window, sinks=sinks,
                               queries=Tokens(torch.zeros_like(last), last, queries_only=True))
        assert ((one - whole[:, i:i + 1]).double().abs().cpu() <= 2 * tol[:, i:i + 1]).all()


@pytest.mark.parametrize('dtype', DTYPES)
def test_prefixes(device, dtype):
    b, t, p = 3, 60, 150
    q, k, v = heads(device, dtype, b, t, t, 4, 2, 64)
    pk, pv = shared(device, dtype, p, 2, 64)
    at = torch.arange(t)
    side = Tokens(i32(at * 0, device), i32(at, device))
    whole = prefix_attention(q, k, v, pk, pv, 0.125, keys=side)
    seen = torch.cat([torch.ones((1, t, p), dtype=torch.bool), see(at * 0, at * 0, at, at, t, 0)], 2)
    tol = reference(q, joined(pk, k), joined(pv, v), 0.125, seen=seen)[1]
    for i in range(t):
        last = i32(at[i:i + 1], device)
        one = prefix_attention(q[:, i:i + 1], k, v, pk, pv, 0.125, keys=side,
                               queries=Tokens(torch.zeros_like(last), last, queries_only=True))
        assert ((one - whole[:, i:i + 1]).double().abs().cpu() <= 2 * tol[:, i:i + 1]).all()
