"""Root-mean-square norm, residual sum and 8-bit output against float64 on the same stored inputs.

Tolerances.  A rounding to type t is off by at most eps_t / 2 of the value (and half a
subnormal step below the normal numbers).  The sum of squares has positive terms: a thread
adds at most 32 of them, then at most 10 + 16 partial sums meet, so it is within 58 * 2^-24 of
exact, its inverse root within half of that, and division, root and two products add five
roundings: 34 * 2^-24 on y in fp32 before its own rounding."""
import pytest
import torch

from musc_hip import _layers_hip

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
Y_FP32 = 34 * F32
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}   # half a subnormal step
EIGHT = {torch.float8_e4m3fn: (448.0, 2.0 ** -4, 2.0 ** -10), torch.float8_e5m2: (57344.0, 2.0 ** -3, 2.0 ** -17)}


def inputs(rows, width, dtype, seed, device, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, width), generator=g) * torch.exp(torch.randn((rows, 1), generator=g))).to(dtype)
    r = torch.randn((rows, width), generator=g).to(dtype) if residual else None
    w = 1 + 0.3 * torch.randn((width,), generator=g)
    return x.to(device), None if r is None else r.to(device), w.to(device)


def formula(s, w, eps):
    s = s.double()
    return s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * (1.0 if w is None else w.double())


def check_sum(s, x, r):
    exact = x.double() + r.double()
    tol = exact.abs() * (torch.finfo(x.dtype).eps / 2 + F32) + TINY[x.dtype]
    assert ((s.double() - exact).abs() <= tol).all()


def check_norm(y, s, w, eps=1e-6):
    ref = formula(s, w, eps)
    tol = ref.abs() * (torch.finfo(y.dtype).eps / 2 * (1 + Y_FP32) + Y_FP32) + TINY[y.dtype]
    assert ((y.double() - ref).abs() <= tol).all()


def check_eight(y8, scales, s, w, group, dtype, eps=1e-6):
    largest, half, tiny = EIGHT[dtype]
    ref = formula(s, w, eps)
    blocks = ref.unflatten(-1, (-1, group or ref.shape[-1]))
    top = blocks.abs().amax(-1)
    want = torch.where(top > 0, top / largest, 1.0)
    assert scales.shape == want.shape and scales.dtype == torch.float32
    assert ((scales.double() - want).abs() <= want * (Y_FP32 + F32)).all()
    value = y8.double().unflatten(-1, (-1, group or ref.shape[-1])) * scales.double()[..., None]
    # half a step of the format at y / scale, and what y / scale itself is off by in fp32
    tol = blocks.abs() * (half * (1 + 3 * Y_FP32) + 3 * Y_FP32) + tiny * scales.double()[..., None]
    assert ((value - blocks).abs() <= tol).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,width', [(1, 1), (3, 7), (5, 64), (2, 513), (7, 1024), (4, 1000), (3, 2056), (2, 4096),
                                        (2, 8191), (1, 16384), (300, 72)])
def test_norm_and_residual(device, rows, width, dtype):
    x, r, w = inputs(rows, width, dtype, rows * 7 + width, device)
    check_norm(_layers_hip.rms_norm(x, w, 1e-6), x, w)
    s, y = _layers_hip.rms_norm(x, w, 1e-6, residual=r)
    check_sum(s, x, r)
    check_norm(y, s, w)
    check_norm(_layers_hip.rms_norm(x, w.to(dtype), 1e-6), x, w.to(dtype))
    check_norm(_layers_hip.rms_norm(x, None, 1e-3), x, None, 1e-3)


@pytest.mark.parametrize('width', [16392, 32768])
def test_widest_rows(device, width):
    x, r, w = inputs(2, width, torch.bfloat16, 3, device)
    s, y = _layers_hip.rms_norm(x, w, 1e-6, residual=r)
    check_norm(y, s, w)
    with pytest.raises(RuntimeError, match='implemented range'):
        _layers_hip.rms_norm(torch.zeros((1, 32769), dtype=torch.float16, device=device), None, 1e-6)


@pytest.mark.parametrize('fmt', list(EIGHT))
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,width,group', [(1, 1, 0), (3, 33, 0), (5, 1024, 0), (8, 4096, 0), (2, 9000, 0), (4, 32, 32),
                                              (3, 192, 64), (6, 1024, 128), (2, 8192, 128), (2, 768, 256), (3, 10240, 32)])
def test_eight_bits(device, rows, width, group, dtype, fmt):
    x, r, w = inputs(rows, width, dtype, rows + width, device)
    y8, scales = _layers_hip.rms_norm_quantized(x, w, 1e-6, dtype=fmt, group=group)
    assert y8.dtype == fmt
    check_eight(y8, scales, x, w, group, fmt)
    s, y8, scales = _layers_hip.rms_norm_quantized(x, w, 1e-6, residual=r, dtype=fmt, group=group)
    check_sum(s, x, r)
    check_eight(y8, scales, s, w, group, fmt)


@pytest.mark.parametrize('dtype', DTYPES)
def test_strided_rows_and_unaligned_starts(device, dtype):
    x, r, w = inputs(9, 264, dtype, 5, device)
    for cols in (slice(0, 128), slice(8, 136), slice(1, 129), slice(3, 260)):
        xs, rs, ws = x[:, cols], r[:, cols], w[cols]
        s, y = _layers_hip.rms_norm(xs, ws, 1e-6, residual=rs)
        check_sum(s, xs, rs)
        check_norm(y, s, ws)
    y8, scales = _layers_hip.rms_norm_quantized(x[:, 1:129], w[1:129], 1e-6, group=32)
    check_eight(y8, scales, x[:, 1:129], w[1:129], 32, torch.float8_e4m3fn)
    y = _layers_hip.rms_norm(x.t()[:9, :9], None, 1e-6)
    check_norm(y, x.t()[:9, :9], None)
    y = _layers_hip.rms_norm(x.view(3, 3, 264), w, 1e-6)
    assert y.shape == (3, 3, 264)
    check_norm(y, x.view(3, 3, 264), w)


def test_zero_rows_and_zero_groups(device):
    x = torch.zeros((3, 256), device=device, dtype=torch.float16)
    x[1, 64:128] = 2.0
    assert (_layers_hip.rms_norm(x, None, 1e-6)[0] == 0).all()
    y8, scales = _layers_hip.rms_norm_quantized(x, None, 1e-6, group=64)
    assert torch.equal(scales[0].cpu(), torch.ones(4)) and (y8.float()[0] == 0).all()
    assert scales[1, 1] != 1 and (y8.float()[1, 64:128] == 448).all()
    assert _layers_hip.rms_norm(x[:0], None, 1e-6).shape == (0, 256)
    y8, scales = _layers_hip.rms_norm_quantized(x[:0], None, 1e-6)
    assert y8.shape == (0, 256) and scales.shape == (0, 1)
    # values too small for a normal scale: the scale stays a normal number
    y8, scales = _layers_hip.rms_norm_quantized(x[1:2], torch.full((256,), 1e-42, device=device), 1e-6)
    assert (scales >= 2.0 ** -126).all() and torch.isfinite(y8.float()).all()


def test_not_a_number_stays_in_its_row(device):
    x, _, w = inputs(6, 512, torch.bfloat16, 9, device, residual=False)
    clean = _layers_hip.rms_norm(x, w, 1e-6)
    clean8, clean_scales = _layers_hip.rms_norm_quantized(x, w, 1e-6)
    x[2, 17], x[4, 5] = float('nan'), float('inf')
    y = _layers_hip.rms_norm(x, w, 1e-6)
    y8, scales = _layers_hip.rms_norm_quantized(x, w, 1e-6)
    for row in (0, 1, 3, 5):
        assert torch.equal(y[row], clean[row]) and torch.equal(scales[row], clean_scales[row])
        assert torch.equal(y8[row].view(torch.uint8), clean8[row].view(torch.uint8))
    assert torch.isnan(y[2]).all() and torch.isnan(y8.float()[2]).all() and torch.isnan(scales[2]).all()
    # an infinite entry: its own value is inf * 0, its neighbours' are x * 0
    assert torch.isnan(y[4, 5]) and (y[4, :5] == 0).all()


def test_side_stream_and_graph(device):
    x, r, w = inputs(64, 2048, torch.float16, 11, device)
    eager = _layers_hip.rms_norm_quantized(x, w, 1e-6, residual=r, group=128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _layers_hip.rms_norm_quantized(x, w, 1e-6, residual=r, group=128)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = _layers_hip.rms_norm_quantized(x, w, 1e-6, residual=r, group=128)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(eager, again, kept):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))


def test_eight_bit_rows_feed_a_scaled_product(device):
    # the pair (y8, scales) is what a row-scaled 8-bit product takes
    x, _, w = inputs(32, 256, torch.bfloat16, 13, device, residual=False)
    g = torch.Generator().manual_seed(14)
    m = torch.randn((64, 256), generator=g).to(device)
    y8, scales = _layers_hip.rms_norm_quantized(x, w, 1e-6)
    got = (y8.float() * scales) @ m.t()
    ref = formula(x, w, 1e-6) @ m.double().t()
    # each of 256 terms is off by at most 2^-4 of it (and 2^-10 of the scale)
    tol = (formula(x, w, 1e-6).abs() * (2.0 ** -4 + 256 * F32) + scales.double() * 2.0 ** -10) @ m.double().abs().t()
    assert ((got.double() - ref).abs() <= tol + 1e-6).all()


def test_refusals(device):
    x = torch.zeros((2, 64), device=device)
    with pytest.raises(ValueError, match='float32, float16 or bfloat16'):
        _layers_hip.rms_norm(x.double(), None, 1e-6)
    with pytest.raises(ValueError, match='weight'):
        _layers_hip.rms_norm(x, torch.ones(63, device=device), 1e-6)
    with pytest.raises(ValueError, match='weight'):
        _layers_hip.rms_norm(x, torch.ones(64, device=device, dtype=torch.float16), 1e-6)
    with pytest.raises(ValueError, match='residual'):
        _layers_hip.rms_norm(x, None, 1e-6, residual=x[:1])
    with pytest.raises(ValueError, match='group'):
        _layers_hip.rms_norm_quantized(x, None, 1e-6, group=48)
    with pytest.raises(ValueError, match='group'):
        _layers_hip.rms_norm_quantized(x, None, 1e-6, group=128)
    with pytest.raises(ValueError, match='dtype'):
        _layers_hip.rms_norm_quantized(x, None, 1e-6, dtype=torch.int8)
    with pytest.raises(ValueError, match='backward'):
        _layers_hip.rms_norm(x.clone().requires_grad_(), None, 1e-6)
    with pytest.raises(ValueError, match='invalid argument'):
        _layers_hip.rms_norm(x, None, -1.0)
