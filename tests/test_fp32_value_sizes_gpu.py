"""fp32 windows and prefixes over V whose keys differ in size, one document alone: a row's output keeps its digits
whatever the keys hold that only other rows see.  Tolerance as in test_fp32_value_scales_gpu.py."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention, prefix_attention

from test_fp32_value_scales_gpu import check
from test_masked_attention_gpu import heads, i32
from test_prefix_attention_gpu import joined, shared
from test_window_attention_gpu import see

pytestmark = pytest.mark.gpu


def causal(device, t):
    at = torch.arange(t)
    return at, Tokens(i32(at * 0, device), i32(at, device))


@pytest.mark.parametrize('d', [64, 72, 96, 128])
@pytest.mark.parametrize('window', [1, 2, 40])
@pytest.mark.parametrize('per_key', [1.0, 0.5, 0.25, 0.1, -0.1, -0.25, -0.5, -1.0])
def test_values_that_grow_or_fall_key_by_key(device, per_key, window, d):
    t = 110
    q, k, v = heads(device, torch.float32, 1, t, t, 2, 1, d)
    at, side = causal(device, t)
    v = v * (2.0 ** (per_key * (at - t // 2)).floor()).to(device)[None, :, None, None]
    got = masked_attention(q, k, v, 1e-3, keys=side, window=window)
    check(got, q, k, v, 1e-3, seen=see(at * 0, at * 0, at, at, window, 0))


@pytest.mark.parametrize('d', [64, 96])
@pytest.mark.parametrize('tq', [1, 20, 160])
@pytest.mark.parametrize('power', [3, 7, 12, 20, 28, 40, 60, 100, -12, -40])
def test_one_key_of_another_size(device, power, tq, d):
    # in the middle of a tile: some rows see it and others do not
    t = 160
    q, k, v = heads(device, torch.float32, 1, tq, t, 2, 1, d)
    at = torch.arange(t)
    new = at[:tq] if tq > 1 else at[72:73]
    v[:, 8], v[:, 75], v[:, 140] = v[:, 8] * 2.0 ** power, v[:, 75] * 2.0 ** power, v[:, 140] * 2.0 ** power
    side, queries = Tokens(i32(at * 0, device), i32(at, device)), Tokens(i32(new * 0, device), i32(new, device), queries_only=True)
    for window in (1, 30, 200):
        got = masked_attention(q, k, v, 1e-3, keys=side, queries=queries, window=window)
        check(got, q, k, v, 1e-3, seen=see(new * 0, at * 0, new, at, window, 0))


@pytest.mark.parametrize('b,t', [(2, 40), (12, 6), (2, 140)])
@pytest.mark.parametrize('power', [20, 40, 100])
def test_own_keys_after_a_prefix(device, power, b, t):
    q, k, v = heads(device, torch.float32, b, t, t, 2, 2, 64)
    pk, pv = shared(device, torch.float32, 70, 2, 64)
    at, side = causal(device, t)
    v[:, 4] *= 2.0 ** power
    own = see(at * 0, at * 0, at, at, t, 0)
    seen = torch.cat([torch.ones((1, t, 70), dtype=torch.bool), own], 2)
    got = prefix_attention(q, k, v, pk, pv, 1e-3, keys=side)
    check(got, q, joined(pk, k), joined(pv, v), 1e-3, seen=seen)


@pytest.mark.parametrize('d', [64, 80])
def test_one_channel_of_another_size(device, d):
    # channels of a block that are large in all keys leave the others their digits by key
    t = 200
    q, k, v = heads(device, torch.float32, 1, t, t, 2, 1, d)
    at, side = causal(device, t)
    v[..., 5] *= 1000
    v[..., 40] /= 1000
    got = masked_attention(q, k, v, 1e-3, keys=side, window=60)
    check(got, q, k, v, 1e-3, seen=see(at * 0, at * 0, at, at, 60, 0))
