"""Several-axis rotary positions against complex float64 rotation of the same stored inputs.

Tolerance of an output a cos - b sin: the angle's fraction of a turn is rounded to fp32 (at
most 1/2, so pi 2^-24 radians), cosine and sine are within 2 units of 2^-24 each, two products
and a sum round once each: (|a| + |b|) (pi + 2 + 3) 2^-24, and the rounding to the type.  The
float64 turns of both sides are within 3 * 2^-53 of the number of turns."""
import math

import pytest
import torch

from musc_hip._rotary_hip import RotaryAxes, rotary

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def expected(x, positions, sections, base, shared, adjacent, inverse=False):
    """(values, tolerance) in float64."""
    x64 = x.double().cpu()
    p = positions.double().cpu()
    p = p if p.dim() == 3 else p[None].expand(x.shape[0], -1, -1)
    total, rates, axis = sum(sections), [], []
    for a, n in enumerate(sections):
        for i in range(n):
            rates.append(base ** -(len(rates) / total if shared else i / n))
            axis.append(a)
    angle = p[..., axis] * torch.tensor(rates, dtype=torch.float64)
    slack = 2 * math.pi * 3 * 2.0 ** -53 * (angle.abs() / (2 * math.pi))[:, :, None]
    turn = torch.polar(torch.ones_like(angle), -angle if inverse else angle)[:, :, None]
    if adjacent:
        a, b = x64[..., 0:2 * total:2], x64[..., 1:2 * total:2]
    else:
        a, b = x64[..., :total], x64[..., total:2 * total]
    z = torch.complex(a, b) * turn
    off = (a.abs() + b.abs()) * ((math.pi + 5) * 2.0 ** -24 + slack)
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if adjacent else (lambda u, v: torch.cat([u, v], -1))
    y = torch.cat([join(z.real, z.imag), x64[..., 2 * total:]], -1)
    tol = torch.cat([join(off, off), torch.zeros_like(x64[..., 2 * total:])], -1)
    return y, tol + (y.abs() + tol) * torch.finfo(x.dtype).eps / 2 + TINY[x.dtype]


def check(got, x, *args, **kw):
    y, tol = expected(x, *args, **kw)
    assert got.shape == x.shape and got.dtype == x.dtype
    assert ((got.double().cpu() - y).abs() <= tol).all()


def normal(shape, dtype, seed, device):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('adjacent', [False, True])
@pytest.mark.parametrize('b,t,h,hk,dim,sections', [
    (1, 1, 1, 1, 2, (1,)), (2, 5, 3, 1, 6, (1, 2)), (2, 37, 4, 4, 64, (0, 16, 16)), (1, 100, 8, 2, 128, (16, 24, 24)),
    (3, 9, 2, 2, 80, (8, 16, 16)), (1, 21, 2, 1, 72, (0, 16, 16)), (2, 3, 1, 1, 512, (100, 56, 100)), (1, 7, 5, 5, 33, (5, 6))])
def test_sections_and_layouts(device, b, t, h, hk, dim, sections, adjacent, dtype):
    g = torch.Generator().manual_seed(dim + t)
    q, k = normal((b, t, h, dim), dtype, 1, device), normal((b, t, hk, dim), dtype, 2, device)
    pos = torch.randint(-50, 500, (b, t, len(sections)), generator=g)
    for shared, base in ((False, 100.0), (True, 1e6)):
        axes = RotaryAxes(dim, sections, base=base, shared=shared, adjacent=adjacent, device=device)
        for p in (pos.float(), pos.int(), pos[0].float() + 0.25):
            qr, kr = rotary(q, k, p.to(device), axes)
            check(qr, q, p, sections, base, shared, adjacent)
            check(kr, k, p, sections, base, shared, adjacent)


@pytest.mark.parametrize('position', [2 ** 24 - 1, 2 ** 31 - 1, -(2 ** 31)])
def test_far_positions(device, position):
    q = normal((1, 4, 2, 64), torch.float32, 3, device)
    pos = torch.tensor([[position], [position // 2], [0], [1]], dtype=torch.int32)
    axes = RotaryAxes(64, (32,), base=10000.0, device=device)
    check(rotary(q, None, pos.to(device), axes), q, pos, (32,), 10000.0, False, False)


@pytest.mark.parametrize('dtype', DTYPES)
def test_packed_projection_in_place_and_back(device, dtype):
    t, b, heads = 50, 3, 4
    qkv = normal((t, b, 3 * heads * 64), dtype, 4, device)     # the in-projection's (T, B, 3E)
    before = qkv.clone()
    parts = qkv.view(t, b, 3, heads, 64).permute(2, 1, 0, 3, 4)
    q, k, v = parts[0], parts[1], parts[2]
    pos = torch.stack([torch.arange(t) // 7, torch.arange(t) % 7], -1).float()
    axes = RotaryAxes(64, (16, 16), base=100.0, device=device)
    apart = rotary(q, k, pos.to(device), axes)
    out = rotary(q, k, pos.to(device), axes, out=(q, k))
    assert out[0].data_ptr() == q.data_ptr()
    assert torch.equal(q, apart[0]) and torch.equal(k, apart[1])
    was = before.view(t, b, 3, heads, 64).permute(2, 1, 0, 3, 4)
    check(q, was[0], pos, (16, 16), 100.0, False, False)
    assert torch.equal(v, was[2])
    back = rotary(q, None, pos.to(device), axes, inverse=True)
    check(back, q, pos, (16, 16), 100.0, False, False, inverse=True)


@pytest.mark.parametrize('dtype', DTYPES)
def test_unaligned_views(device, dtype):
    whole = normal((2, 11, 3, 70), dtype, 5, device)
    for first in (1, 2, 6):
        q = whole[..., first:first + 64]
        axes = RotaryAxes(64, (8, 20), device=device)
        pos = torch.arange(22).reshape(11, 2).float()
        check(rotary(q, None, pos.to(device), axes), q, pos, (8, 20), 10000.0, False, False)
    q = normal((2, 64, 11, 3), dtype, 6, device).permute(0, 2, 3, 1)   # last dimension not contiguous
    check(rotary(q, None, pos.to(device), axes), q, pos, (8, 20), 10000.0, False, False)


def test_many_heads_and_tokens(device):
    q = normal((2, 1500, 65, 32), torch.float16, 7, device)
    pos = torch.arange(1500).float()[:, None]
    axes = RotaryAxes(32, (16,), device=device)
    check(rotary(q, q[:, :, :3], pos.to(device), axes)[0], q, pos, (16,), 10000.0, False, False)
    assert rotary(q[:, :0], None, pos[:0].to(device), axes).shape == (2, 0, 65, 32)
    # 1024 heads of 508 single-stepped channels: the largest index arithmetic
    q = normal((1, 2, 1024, 509), torch.bfloat16, 8, device)
    axes = RotaryAxes(509, (1,), device=device)
    check(rotary(q, None, pos[:2].to(device), axes), q, pos[:2], (1,), 10000.0, False, False)


def test_not_a_number_stays_in_its_token(device):
    q = normal((1, 6, 2, 64), torch.float32, 9, device)
    axes = RotaryAxes(64, (32,), device=device)
    pos = torch.arange(6).float()[:, None]
    clean = rotary(q, None, pos.to(device), axes)
    pos[3] = float('nan')
    q2 = q.clone()
    q2[0, 1] = float('inf')
    got = rotary(q2, None, pos.to(device), axes)
    for t in (0, 2, 4, 5):
        assert torch.equal(got[0, t], clean[0, t])
    assert torch.isnan(got[0, 3]).all()


def test_graph_follows_positions(device):
    q, k = normal((2, 1, 8, 128), torch.bfloat16, 10, device), normal((2, 1, 2, 128), torch.bfloat16, 11, device)
    axes = RotaryAxes(128, (16, 24, 24), shared=True, base=1e6, device=device)
    pos = torch.zeros((2, 1, 3), device=device)
    rotary(q, k, pos, axes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = rotary(q, k, pos, axes)
    for step in range(3):
        pos.fill_(1000.0 + step)
        eager = rotary(q, k, pos, axes)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept[0], eager[0]) and torch.equal(kept[1], eager[1])


def test_refusals(device):
    q = torch.zeros((1, 4, 2, 64), device=device)
    pos = torch.zeros((4, 2), device=device)
    axes = RotaryAxes(64, (16, 16), device=device)
    with pytest.raises(ValueError, match='positions'):
        rotary(q, None, pos[:3], axes)
    with pytest.raises(ValueError, match='positions'):
        rotary(q, None, pos.double(), axes)
    with pytest.raises(ValueError, match='heads, 64'):
        rotary(q[..., :32], None, pos, axes)
    with pytest.raises(ValueError, match='match q'):
        rotary(q, q.half(), pos, axes)
    with pytest.raises(ValueError, match='share memory'):
        rotary(q, None, pos, axes, out=q[:, :1].expand(1, 4, 2, 64))
    with pytest.raises(ValueError, match='backward'):
        rotary(q.clone().requires_grad_(), None, pos, axes)
    for bad in ((), (33,), (-1, 5), (0,)):
        with pytest.raises(ValueError, match='sections'):
            RotaryAxes(64, bad, device=device)
    with pytest.raises(RuntimeError, match='implemented range'):
        rotary(torch.zeros((1, 1, 1, 1024), device=device), None, pos[:1], RotaryAxes(1024, (4, 4), device=device))


def test_refuses_gradients_of_positions_and_out(device):
    q, pos = torch.zeros((1, 4, 2, 64), device=device), torch.zeros((4, 2), device=device)
    axes = RotaryAxes(64, (16, 16), device=device)
    for out in (torch.empty_like(q).requires_grad_(), None):
        with pytest.raises(ValueError, match='backward'):
            rotary(q, None, pos if out is not None else pos.clone().requires_grad_(), axes, out=out)
    with pytest.raises(ValueError, match='backward'):
        rotary(q, q.clone(), pos, axes, out=(torch.empty_like(q), torch.empty_like(q).requires_grad_()))


def test_keys_without_queries(device):
    q, k = normal((2, 5, 0, 64), torch.float16, 12, device), normal((2, 5, 3, 64), torch.float16, 13, device)
    pos = torch.arange(10).float().view(5, 2)
    axes = RotaryAxes(64, (16, 16), device=device)
    q_out, k_out = rotary(q, k, pos.to(device), axes)
    assert q_out.shape == q.shape
    check(k_out, k, pos, (16, 16), 10000.0, False, False)
