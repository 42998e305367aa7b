"""fp32 windows and prefixes over V that is not finite, large, or of different sizes, against float64.

Tolerance: masked attention's (test_masked_attention_gpu.py), and for V held in two fp16 numbers by 32 keys and
32 channels, whose keys are within 2^6 of the largest by their largest entries there, 2^-39 of the block's
largest: 2^-33 sum_j p_j max_c |v_jc| / sum_j p_j over the block's channels."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention, prefix_attention

from test_masked_attention_gpu import heads, i32, reference
from test_prefix_attention_gpu import joined, shared
from test_window_attention_gpu import see

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (40, 1), (9, 5), (3, 90), (1, 300)]       # teams, stacked, stacked, four waves, splits


def blocks(v):
    """each entry's place taken by the largest of its key and block of 32 channels"""
    d = v.shape[-1]
    parts = [v[..., c:c + 32].abs().amax(-1, keepdim=True).expand(*v.shape[:-1], min(32, d - c)) for c in range(0, d, 32)]
    return torch.cat(parts, -1)


def check(got, q, k, v, scale, channels=slice(None), **kw):
    v = torch.nan_to_num(v.cpu(), 0, 0, 0)
    out, tol = reference(q, k, v, scale, **kw)
    tol = tol + 2.0 ** -33 * reference(q, k, blocks(v), scale, **kw)[0].abs()
    got = got.double().cpu()
    assert torch.isfinite(got[..., channels]).all()
    bad = ((got - out).abs() > tol)[..., channels]
    off = ((got - out).abs() / tol)[..., channels]
    assert not bad.any(), (off.max().item(), bad.nonzero()[:4])


@pytest.mark.parametrize('b,tq,p', [(b, tq, p) for b, tq in SHAPES for p in (32, 64, 1024)] + [(1, 2, 16384), (3, 30, 16384)])
@pytest.mark.parametrize('what', [float('-inf'), float('nan')])
@pytest.mark.parametrize('size', [4.0, 100.0])
def test_one_entry_of_whole_tiles_is_not_finite(device, size, what, b, tq, p):
    q, k, _ = heads(device, torch.float32, b, tq, 0, 2, 1, 64)
    pk, pv = shared(device, torch.float32, p, 1, 64)
    pv = size * (1 + pv.abs() / 8)
    pv[3, 0, 5] = what
    got = prefix_attention(q, k, k, pk, pv, 0.05)
    others = [c for c in range(64) if c != 5]
    check(got, q, joined(pk, k), joined(pv, k), 0.05, others)
    assert torch.equal(got[..., 5].cpu().nan_to_num(7, 8, 9), torch.full(got.shape[:-1], what).nan_to_num(7, 8, 9))


@pytest.mark.parametrize('b,tq', SHAPES)
@pytest.mark.parametrize('p', [32, 96, 2048])
def test_one_channel_is_not_finite(device, p, b, tq):
    q, k, _ = heads(device, torch.float32, b, tq, 0, 2, 1, 96)
    pk, pv = shared(device, torch.float32, p, 1, 96)
    pv *= 200
    pv[..., 0], pv[..., 70] = float('nan'), float('inf')
    got = prefix_attention(q, k, k, pk, pv, 0.05)
    check(got, q, joined(pk, k), joined(pv, k), 0.05, [c for c in range(96) if c not in (0, 70)])
    assert torch.isnan(got[..., 0]).all() and (got[..., 70] == float('inf')).all()


@pytest.mark.parametrize('tq', [1, 40, 200])
@pytest.mark.parametrize('tk', [32, 64, 1024])
def test_whole_tiles_of_a_window(device, tk, tq):
    # every order the same: all keys are seen by all queries
    q, k, v = heads(device, torch.float32, 2, tq, tk, 4, 2, 64)
    v = 100 * (1 + v.abs() / 8)
    v[:, 1, :, 40], v[:, 2, :, 9] = float('inf'), float('nan')
    zeros = lambda t: i32(torch.zeros(t), device)  # noqa: E731
    got = masked_attention(q, k, v, 0.05, keys=Tokens(zeros(tk), zeros(tk)), queries=Tokens(zeros(tq), zeros(tq), queries_only=True),
                           window=1)
    check(got, q, k, v, 0.05, [c for c in range(64) if c not in (9, 40)])


@pytest.mark.parametrize('d', [32, 64, 72])
@pytest.mark.parametrize('largest', [1e-25, 1e12, 1e24, 1e32])
def test_the_largest_numbers_after_small_ones(device, largest, d):
    # documents of very large and of ordinary V in one tile, and in tiles after one another
    docs = torch.repeat_interleave(torch.arange(6), torch.tensor([20, 40, 70, 30, 33, 64]))
    t = len(docs)
    q, k, v = heads(device, torch.float32, 1, t, t, 2, 1, d)
    sizes = torch.tensor([1.0, largest, 1.0, largest, 1.0, largest])[docs].to(device)
    v = v.clamp(-4, 4) * sizes[None, :, None, None]
    at = torch.arange(t)
    side = Tokens(i32(docs, device), i32(at, device))
    got = masked_attention(q, k, v, 0.05, keys=side, window=50)
    check(got, q, k, v, 0.05, seen=see(docs, docs, at, at, 50, 0))


@pytest.mark.parametrize('tq', [1, 20, 200])
@pytest.mark.parametrize('d', [64, 128])
def test_values_near_the_end_of_the_type(device, d, tq):
    # four keys of up to 2^125 each: their sum is a number
    t = 230
    q, k, v = heads(device, torch.float32, 1, tq, t, 2, 1, d)
    v = v.clamp(-1, 1) * 2.0 ** 125
    at, new = torch.arange(t), torch.arange(t)[-tq:]
    got = masked_attention(q, k, v, 1e-3, keys=Tokens(i32(at * 0, device), i32(at, device)), window=4,
                           queries=Tokens(i32(new * 0, device), i32(new, device), queries_only=True))
    check(got, q, k, v, 1e-3, seen=see(new * 0, at * 0, new, at, 4, 0))


@pytest.mark.parametrize('b,tq', SHAPES)
def test_values_near_the_end_of_the_type_after_a_prefix(device, b, tq):
    q, k, v = heads(device, torch.float32, b, tq, 2, 2, 1, 64)
    pk, pv = shared(device, torch.float32, 3000, 1, 64)
    v, pv = v.clamp(-1, 1) * 2.0 ** 114, pv.clamp(-1, 1) * 2.0 ** 114       # the sum over 3002 keys below 2^126
    check(prefix_attention(q, k, v, pk, pv, 1e-3), q, joined(pk, k), joined(pv, v), 1e-3)
