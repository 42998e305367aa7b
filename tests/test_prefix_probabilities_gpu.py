"""Few rows an entry keep their probabilities in two numbers, alone or together with other entries after a shared
prefix, in 16-bit types.

Tolerance: masked attention's (test_masked_attention_gpu.py) with, in place of a probability's rounding to the storage
type (eps / 2), that to two such numbers: eps^2 / 2."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention, prefix_attention

from test_masked_attention_gpu import heads, i32, reference, see as see_own
from test_prefix_attention_gpu import joined, shared
from test_window_attention_gpu import see

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


def check(got, q, k, v, scale, **kw):
    out, tol = reference(q.float(), k, v, scale, **kw)     # without the storage type's roundings
    eps = torch.finfo(q.dtype).eps
    w = reference(q.float(), k, v.abs(), scale, **kw)[0]
    tol = tol + eps * eps / 2 * w
    if q.dtype == torch.float16:
        tol = tol + k.shape[1] * 2.0 ** -32 * v.abs().max().item() + 2.0 ** -25
    tol = tol + eps / 2 * (out.abs() + tol)
    bad = (got.double().cpu() - out).abs() > tol
    assert not bad.any(), (((got.double().cpu() - out).abs() / tol).max().item(), bad.sum().item())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('cap', [0.0, 20.0, 300.0])
@pytest.mark.parametrize('b,tq', [(1, 1), (3, 2), (12, 1), (40, 1), (33, 3), (9, 8)])
@pytest.mark.parametrize('d', [64, 80, 128])
def test_entries_of_few_rows(device, d, b, tq, cap, dtype):
    h, hk, tk, p = 8, 2, 70, 2300        # past what the waves of one workgroup share
    q, k, v = heads(device, dtype, b, tq, tk, h, hk, d)
    pk, pv = shared(device, dtype, p, hk, d)
    at, last = torch.arange(tk), torch.randint(tq, tk, (b, 1), generator=torch.Generator().manual_seed(b)) + torch.arange(tq) - tq
    keys = Tokens(i32(at * 0, device), i32(at, device))
    queries = Tokens(i32(last * 0, device), i32(last, device), queries_only=True)
    own = see_own(last * 0, at * 0, last, at)
    seen = torch.cat([torch.ones((b, tq, p), dtype=torch.bool), own], 2)
    got = prefix_attention(q, k, v, pk, pv, 0.1, keys=keys, queries=queries, cap=cap)
    check(got, q, joined(pk, k), joined(pv, v), 0.1, seen=seen, cap=cap)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('d', [64, 128])
def test_with_a_bias(device, d, dtype):
    b, p, h = 40, 2300, 8
    q, k, _ = heads(device, dtype, b, 1, 0, h, 2, d)
    pk, pv = shared(device, dtype, p, 2, d)
    slopes, ppos, qpos = 2.0 ** -torch.arange(3, 3 + h).float()[:, None], torch.arange(p).float()[:, None], torch.full((b, 1, 1), 2310.0)
    none = torch.empty((b, 0, 1), device=device)
    got = prefix_attention(q, k, k, pk, pv, 0.1, keys=Tokens(positions=none), queries=Tokens(positions=qpos.to(device)),
                           slopes=slopes.to(device), prefix_positions=ppos.to(device))
    check(got, q, joined(pk, k), joined(pv, k), 0.1, slopes=slopes, qpos=qpos, kpos=ppos[None].expand(b, -1, -1))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('b,tq', [(1, 1), (40, 1), (9, 8)])
def test_windows_of_few_rows(device, b, tq, dtype):
    tk = 900
    q, k, v = heads(device, dtype, b, tq, tk, 8, 2, 128)
    at, new = torch.arange(tk), torch.arange(tk)[-tq:]
    got = masked_attention(q, k, v, 0.1, keys=Tokens(i32(at * 0, device), i32(at, device)), window=500, sinks=4,
                           queries=Tokens(i32(new * 0, device), i32(new, device), queries_only=True))
    check(got, q, k, v, 0.1, seen=see(new * 0, at * 0, new, at, 500, 4))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('b,tq', [(2, 1), (12, 1), (40, 1), (9, 8)])
def test_errors_are_the_roundings_of_the_output(device, b, tq, d, dtype):
    """Before its rounding an output is within about 2^-17 of itself, so the root mean square of the errors is that of
    rounding the exact values; over the 1000 to 80000 outputs here it scatters by 1 / sqrt(2000) at most, of which a
    tenth is four.  Probabilities of one number each give 1.3 times as much."""
    h, hk, tk, p = 8, 2, 60, 2300
    q, k, v = heads(device, dtype, b, tq, tk, h, hk, d)
    pk, pv = shared(device, dtype, p, hk, d)
    got = prefix_attention(q, k, v, pk, pv, 0.1)
    out = reference(q, joined(pk, k), joined(pv, v), 0.1)[0]
    rms = lambda x: (x - out).pow(2).mean().sqrt().item()  # noqa: E731
    assert rms(got.double().cpu()) <= 1.1 * rms(out.to(dtype).double())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('cap', [0.0, 300.0])
def test_stacked_entries_beside_unseen_values(device, cap, dtype):
    # NaN and infinities behind the prefix in its last tile, in caches that were never written, and in padding
    b, h, hk, tk, p, d = 40, 8, 2, 90, 2301, 128
    q, k, v = heads(device, dtype, b, 1, tk, h, hk, d)
    room_k, room_v = shared(device, dtype, p + 30, hk, d)
    room_k[p:], room_v[p:] = float('nan'), float('inf')
    at, last = torch.arange(tk), (torch.arange(b)[:, None] * 7) % tk
    qd = torch.where(torch.arange(b)[:, None] % 9 == 8, -1, 0)
    unseen = (at[None] > last)[..., None, None].to(device)
    full_k, full_v = k.masked_fill(unseen, float('inf')), v.masked_fill(unseen, float('nan'))
    q[qd[:, 0].to(device) < 0] = float('nan')
    keys = Tokens(i32(at * 0, device), i32(at, device))
    queries = Tokens(i32(qd, device), i32(last, device), queries_only=True)
    got = prefix_attention(q, full_k, full_v, room_k[:p], room_v[:p], 0.1, keys=keys, queries=queries, cap=cap)
    live = qd[:, 0] >= 0
    own = see_own(qd, at * 0, last, at)
    seen = torch.cat([torch.ones((b, 1, p), dtype=torch.bool), own], 2)[live]
    check(got[live], q[live], joined(room_k[:p], k)[live], joined(room_v[:p], v)[live], 0.1, seen=seen, cap=cap)
    assert (got[~live] == 0).all()
