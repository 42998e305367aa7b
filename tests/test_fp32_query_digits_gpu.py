"""fp32 windows and prefixes whose keys differ in size go by fp32 instructions on Q as it is, against float64
(the tolerance is masked attention's, test_masked_attention_gpu.py)."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention, prefix_attention

from test_masked_attention_gpu import check, heads, i32
from test_prefix_attention_gpu import joined, shared
from test_window_attention_gpu import see

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('scale', [0.3, -0.3, 0.0])
@pytest.mark.parametrize('tq', [1, 20, 130])
@pytest.mark.parametrize('d', [64, 72, 128])
def test_small_numbers_of_q_meet_large_ones_of_k(device, d, tq, scale):
    t = 130
    q, k, v = heads(device, torch.float32, 2, tq, t, 2, 1, d)
    q[..., 7] *= 2.0 ** -30                 # as much of the score as the others, for every other key
    k[:, ::2, :, 7] *= 2.0 ** 30
    at, new = torch.arange(t), torch.arange(t)[-tq:]
    keys = Tokens(i32(at * 0, device), i32(at, device))
    queries = Tokens(i32(new * 0, device), i32(new, device), queries_only=True)
    got = masked_attention(q, k, v, scale, keys=keys, queries=queries, window=50, sinks=1)
    check(got, q, k, v, scale, seen=see(new * 0, at * 0, new, at, 50, 1))


@pytest.mark.parametrize('b,tq', [(1, 1), (40, 1), (3, 90)])
def test_after_a_prefix(device, b, tq):
    q, k, v = heads(device, torch.float32, b, tq, 50, 2, 2, 64)
    pk, pv = shared(device, torch.float32, 700, 2, 64)
    q[..., 7] *= 2.0 ** -30
    k[:, ::2, :, 7] *= 2.0 ** 30
    pk[::3, :, 7] *= 2.0 ** 30
    check(prefix_attention(q, k, v, pk, pv, 0.3), q, joined(pk, k), joined(pv, v), 0.3)


def test_infinities_beside_small_numbers(device):
    # a query and a key that are not finite leave the other rows as they are
    t = 100
    q, k, v = heads(device, torch.float32, 1, t, t, 1, 1, 64)
    q[..., 7] *= 2.0 ** -30
    k[:, ::2, :, 7] *= 2.0 ** 30
    q[0, 50, 0, 3] = float('inf')
    at = torch.arange(t)
    side = Tokens(i32(at * 0, device), i32(at, device))
    got = masked_attention(q, k, v, 0.3, keys=side, window=30)
    rest = at != 50
    check(got[:, rest], q[:, rest], k, v, 0.3, seen=see(at * 0, at * 0, at, at, 30, 0)[:, rest])
    assert torch.isnan(got[0, 50]).all()
