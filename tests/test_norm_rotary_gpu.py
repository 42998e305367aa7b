"""Per-head root-mean-square norms of q and k with rotary positions in the same pass, against float64 on
the same stored inputs.

Tolerance: the D squares are added in fp32, so their sum is off by (D + 1) 2^-24 of itself and its
inverse root by half that, and by 2^-24 for each of the mean, eps, root and reciprocal; two products make
y = x rstd w of it: r = ((D + 1) / 2 + 6) 2^-24 relative.  An output a cos - b sin of it is then off by
(|a| + |b|) (r + (pi + 5) 2^-24), as for rotary alone, and by the rounding to the type."""
import math

import pytest
import torch

from musc_hip._rotary_hip import RotaryAxes, norm_rotary, rotary

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}
U = 2.0 ** -24


def expected(x, weight, eps, positions, sections, base, shared, adjacent):
    """(values, tolerance) in float64."""
    x64 = x.double().cpu()
    y = x64 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double().cpu()
    p = positions.double().cpu()
    p = p if p.dim() == 3 else p[None].expand(x.shape[0], -1, -1)
    total, rates, axis = sum(sections), [], []
    for a, n in enumerate(sections):
        for i in range(n):
            rates.append(base ** -(len(rates) / total if shared else i / n))
            axis.append(a)
    angle = p[..., axis] * torch.tensor(rates, dtype=torch.float64)
    slack = 3 * 2.0 ** -53 * angle.abs()[:, :, None]
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]
    a, b = (y[..., 0:2 * total:2], y[..., 1:2 * total:2]) if adjacent else (y[..., :total], y[..., total:2 * total])
    z = torch.complex(a, b) * turn
    r = ((x.shape[-1] + 1) / 2 + 6) * U
    off = (a.abs() + b.abs()) * (r + (math.pi + 5) * U + slack)
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if adjacent else (lambda u, v: torch.cat([u, v], -1))
    out = torch.cat([join(z.real, z.imag), y[..., 2 * total:]], -1)
    tol = torch.cat([join(off, off), y[..., 2 * total:].abs() * r], -1)
    return out, tol + (out.abs() + tol) * torch.finfo(x.dtype).eps / 2 + TINY[x.dtype]


def check(got, x, weight, eps, *args):
    y, tol = expected(x, weight, eps, *args)
    assert got.shape == x.shape and got.dtype == x.dtype
    bad = ~((got.double().cpu() - y).abs() <= tol)
    assert not bad.any(), (bad.nonzero()[:4], ((got.double().cpu() - y).abs() / tol).max())


def normal(shape, dtype, seed, device, size=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * size).to(dtype).to(device)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('adjacent', [False, True])
@pytest.mark.parametrize('b,t,h,hk,dim,sections', [
    (1, 1, 1, 1, 2, (1,)), (2, 5, 3, 1, 6, (1, 2)), (2, 37, 4, 4, 64, (0, 16, 16)), (1, 100, 8, 2, 128, (16, 24, 24)),
    (3, 9, 2, 2, 80, (8, 16, 16)), (1, 21, 2, 1, 72, (0, 18, 18)), (2, 3, 1, 1, 512, (100, 56, 100)), (1, 7, 5, 5, 33, (5, 6)),
    (1, 40, 33, 3, 96, (44,)), (1, 3, 2, 1, 8, (4,)), (1, 5, 2, 1, 256, (2, 2))])
def test_sections_and_layouts(device, b, t, h, hk, dim, sections, adjacent, dtype):
    g = torch.Generator().manual_seed(dim + t)
    q, k = normal((b, t, h, dim), dtype, 1, device, 3.0), normal((b, t, hk, dim), dtype, 2, device, 0.2)
    pos = torch.randint(-50, 500, (b, t, len(sections)), generator=g)
    axes = RotaryAxes(dim, sections, base=100.0, shared=h % 2 == 0, adjacent=adjacent, device=device)
    args = (sections, 100.0, h % 2 == 0, adjacent)
    qw, kw = 1 + normal((dim,), torch.float32, 3, device, 0.3), 1 + normal((hk, dim), dtype, 4, device, 0.3)
    for p, q_weight, k_weight, eps in ((pos.float(), qw, kw, 1e-6), (pos.int(), qw.to(dtype), None, 0.5),
                                       (pos[0].float() + 0.25, None, kw.float(), 0.0)):
        qr, kr = norm_rotary(q, k, p.to(device), axes, q_weight, k_weight, eps)
        check(qr, q, q_weight, eps, p, *args)
        check(kr, k, k_weight, eps, p, *args)
    assert torch.equal(norm_rotary(q, None, pos.int().to(device), axes, qw.to(dtype), None, 0.5),
                       norm_rotary(q, k, pos.int().to(device), axes, qw.to(dtype), None, 0.5)[0])


@pytest.mark.parametrize('dtype', DTYPES)
def test_heads_of_zeros_small_and_large_values(device, dtype):
    x = normal((1, 6, 4, 64), dtype, 5, device)
    x[0, 0, 0] = 0
    x[0, 1] *= 1e-3
    x[0, 2] *= 1000
    axes, pos = RotaryAxes(64, (32,), device=device), torch.arange(6).float()[:, None]
    for eps in (1e-6, 1e-12):
        got = norm_rotary(x, None, pos.to(device), axes, None, None, eps)
        check(got, x, None, eps, pos, (32,), 10000.0, False, False)
        assert (got[0, 0, 0] == 0).all()
    # infinities and NaN stay in their head
    x[0, 3, 1, 7], x[0, 4, 2, 60] = float('inf'), float('nan')
    got = norm_rotary(x, None, pos.to(device), axes)
    bad = torch.isnan(got).any(-1)
    assert bad[0, 3, 1] and bad[0, 4, 2] and bad.sum() == 2
    if dtype != torch.float16:
        x[0, 5] = 1e20                              # squares past fp32
        assert (norm_rotary(x, None, pos.to(device), axes)[0, 5] == 0).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('adjacent', [False, True])
def test_packed_projection_in_place(device, dtype, adjacent):
    t, b, heads = 50, 3, 4
    qkv = normal((t, b, 3 * heads * 64), dtype, 6, device)
    parts = qkv.view(t, b, 3, heads, 64).permute(2, 1, 0, 3, 4)
    q, k, v = parts[0], parts[1], parts[2]
    was = parts.clone()
    pos = torch.stack([torch.arange(t) // 7, torch.arange(t) % 7], -1).float()
    axes = RotaryAxes(64, (12, 16), base=100.0, adjacent=adjacent, device=device)
    w = 1 + normal((heads, 64), torch.float32, 7, device, 0.2)
    apart = norm_rotary(q, k, pos.to(device), axes, w, w[0], 1e-6)
    out = norm_rotary(q, k, pos.to(device), axes, w, w[0], 1e-6, out=(q, k))
    assert out[0].data_ptr() == q.data_ptr()
    assert torch.equal(q, apart[0]) and torch.equal(k, apart[1]) and torch.equal(v, was[2])
    check(q, was[0], w, 1e-6, pos, (12, 16), 100.0, False, adjacent)
    check(k, was[1], w[0], 1e-6, pos, (12, 16), 100.0, False, adjacent)


@pytest.mark.parametrize('dtype', DTYPES)
def test_unaligned_views_and_weights(device, dtype):
    whole = normal((2, 11, 3, 70), dtype, 8, device)
    pos = torch.arange(22).reshape(11, 2).float()
    axes = RotaryAxes(64, (8, 20), device=device)
    w = 1 + normal((67,), torch.float32, 9, device, 0.2)[1:65]
    for first in (1, 2, 4, 6):
        q = whole[..., first:first + 64]
        check(norm_rotary(q, None, pos.to(device), axes, w), q, w, 1e-6, pos, (8, 20), 10000.0, False, False)
        k = q[:, :, :1].clone()
        check(norm_rotary(q, k, pos.to(device), axes, w, w.to(dtype))[1], k, w.to(dtype), 1e-6, pos, (8, 20), 10000.0, False, False)
    q = normal((2, 64, 11, 3), dtype, 10, device).permute(0, 2, 3, 1)   # last dimension not contiguous
    check(norm_rotary(q, None, pos.to(device), axes), q, None, 1e-6, pos, (8, 20), 10000.0, False, False)
    one = whole[:, :1, :1, :64].expand(2, 11, 3, 64)                    # heads and tokens that share memory
    check(norm_rotary(one, None, pos.to(device), axes), one, None, 1e-6, pos, (8, 20), 10000.0, False, False)


def test_many_heads_and_tokens_and_none(device):
    q = normal((2, 1500, 65, 32), torch.float16, 11, device)
    pos = torch.arange(1500).float()[:, None]
    axes = RotaryAxes(32, (16,), device=device)
    qr, kr = norm_rotary(q, q[:, :, :3], pos.to(device), axes)
    check(qr, q, None, 1e-6, pos, (16,), 10000.0, False, False)
    assert torch.equal(kr, qr[:, :, :3])
    assert norm_rotary(q[:, :0], None, pos[:0].to(device), axes).shape == (2, 0, 65, 32)
    none, kr = norm_rotary(q[:, :, :0], q[:, :, :3], pos.to(device), axes)
    assert none.shape == (2, 1500, 0, 32) and torch.equal(kr, qr[:, :, :3])
    q = normal((1, 2, 1024, 509), torch.bfloat16, 12, device)
    axes = RotaryAxes(509, (1,), device=device)
    check(norm_rotary(q[:, :, :1000], q[:, :, 1000:], pos[:2].to(device), axes)[0], q[:, :, :1000], None, 1e-6, pos[:2], (1,),
          10000.0, False, False)


def test_captured_and_on_another_stream(device):
    q, k = normal((1, 200, 8, 64), torch.float16, 13, device), normal((1, 200, 2, 64), torch.float16, 14, device)
    pos = torch.arange(200).float()[:, None].to(device)
    axes, w = RotaryAxes(64, (32,), device=device), 1 + normal((64,), torch.float32, 15, device, 0.2)
    want = norm_rotary(q, k, pos, axes, w, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm_rotary(q, k, pos, axes, w, w)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = norm_rotary(q, k, pos, axes, w, w)
    for turn in range(3):
        q.copy_(normal(q.shape, torch.float16, 20 + turn, device))
        pos.add_(1000)
        want = norm_rotary(q, k, pos, axes, w, w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept[0], want[0]) and torch.equal(kept[1], want[1])


def test_agrees_with_rotary_of_a_normed_head(device):
    # fp32: the norm in torch and rotary by itself differ by roundings only, counted as above for both
    q = normal((2, 60, 4, 64), torch.float32, 16, device)
    pos = torch.arange(60).float()[:, None]
    axes = RotaryAxes(64, (32,), device=device)
    y = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6)
    _, tol = expected(q, None, 1e-6, pos, (32,), 10000.0, False, False)
    off = (norm_rotary(q, None, pos.to(device), axes) - rotary(y, None, pos.to(device), axes)).abs().double().cpu()
    assert (off <= 2 * tol).all()


def test_refusals(device):
    q = normal((1, 4, 2, 64), torch.float16, 17, device)
    axes, pos = RotaryAxes(64, (32,), device=device), torch.zeros((4, 1), device=device)
    for bad in (torch.ones(63, device=device), torch.ones((3, 64), device=device), torch.ones(64, dtype=torch.bfloat16, device=device),
                torch.ones(64), torch.ones(64, dtype=torch.float64, device=device), [1.0] * 64):
        with pytest.raises(ValueError, match='q_weight'):
            norm_rotary(q, None, pos, axes, bad)
        with pytest.raises(ValueError, match='k_weight'):
            norm_rotary(q, q, pos, axes, None, bad)
    with pytest.raises(ValueError, match='backward'):
        norm_rotary(q, None, pos, axes, torch.ones(64, device=device, requires_grad=True))
    for eps in (-1.0, float('nan')):
        with pytest.raises(ValueError):
            norm_rotary(q, None, pos, axes, eps=eps)
    with pytest.raises(ValueError):
        norm_rotary(q, None, pos[:3], axes)
    with pytest.raises(ValueError):
        norm_rotary(q[..., :32], None, pos, axes)
