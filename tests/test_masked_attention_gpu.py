"""Attention over documents, orders, caps and distances against float64 on the same inputs.

Tolerance of an output o = sum_j p_j v_j / sum_j p_j, with W = sum_j p_j |v_j| / sum_j p_j:
  - a score is within d of exact, d = 2^-24 ((D + 8) scale sum_c |q_c k_c| + 8 cap + 6 bias +
    4): products added in fp32, the factors, tanh and distance rounded; its exponential within
    d + 2^-22 (relative), in the numerator and the denominator:
    sum_j p_j (d_j + 2^-22) (|v_j| + |o|) / sum_j p_j;
  - n terms are added in fp32: n 2^-24 W in the numerator, as much in the denominator;
  - 16-bit types round each probability: half a step, eps / 2 W; fp16 below its normal numbers
    (the largest probability is at least 2^7) n 2^-32 max|v|;
  - the output's own rounding: eps / 2 |o| (and half a subnormal step)."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def reference(q, k, v, scale, seen=None, cap=0.0, slopes=None, qpos=None, kpos=None):
    """(out, tolerance), float64 on the CPU; seen (B or 1, Tq, Tk) bool; positions (B or 1, T, A)."""
    dtype = q.dtype
    q, k, v = (x.double().cpu().transpose(1, 2) for x in (q, k, v))
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    keep = torch.ones((1, q.shape[2], k.shape[2]), dtype=torch.bool) if seen is None else seen.cpu()
    keep = keep[:, None]
    k0, v0 = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
    s = q @ k0.transpose(2, 3) * scale
    size = (q.abs() @ k0.abs().transpose(2, 3)) * abs(scale)
    d = (q.shape[3] + 8) * size + 4
    if cap:
        s = cap * torch.tanh(s / cap)
        d = d + 8 * cap
    if slopes is not None:
        apart = (qpos.double().cpu()[:, :, None] - kpos.double().cpu()[:, None]).abs()
        bias = torch.einsum('bqka,ha->bhqk', apart, slopes.double().cpu())
        s = s - bias
        d = d + 6 * bias.abs()
    s = s.masked_fill(~keep, -torch.inf)
    top = s.amax(-1, keepdim=True)
    empty = top == -torch.inf
    p = torch.exp(s - torch.where(empty, 0.0, top))
    total = p.sum(-1, keepdim=True)
    total = torch.where(empty, 1.0, total)
    out, w = p @ v0 / total, p @ v0.abs() / total
    # a score that is off by d_j moves o by p_j d_j (v_j - o): numerator and denominator
    d = d * U + 2.0 ** -22
    moved = (p * d) @ v0.abs() / total + (p * d).sum(-1, keepdim=True) / total * out.abs()
    n = keep.sum(-1, keepdim=True).double()
    tol = moved + 2 * n * U * w
    half = torch.finfo(dtype).eps / 2
    if dtype != torch.float32:
        tol = tol + half * w
    if dtype == torch.float16:
        tol = tol + n * 2.0 ** -32 * v0.abs().amax() + 2.0 ** -25
    tol = tol + half * (out.abs() + tol)
    return out.transpose(1, 2), tol.transpose(1, 2)


def check(got, *args, **kw):
    out, tol = reference(*args, **kw)
    got = got.double().cpu()
    assert got.shape == out.shape
    assert torch.isfinite(got).all()
    bad = (got - out).abs() > tol
    assert not bad.any(), ((got - out).abs().max().item(), ((got - out).abs() / tol).max().item(), bad.nonzero()[:4])


def heads(device, dtype, b, tq, tk, h, hk, d, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed * 1000 + tq * 31 + tk * 7 + h + d)
    make = lambda t, n: (torch.randn((b, t, n, d), generator=g) * size).to(dtype).to(device)  # noqa: E731
    return make(tq, h), make(tk, hk), make(tk, hk)


def see(qd, kd, qo=None, ko=None):
    qd, kd = (x if x.dim() == 2 else x[None] for x in (qd, kd))
    m = (qd[:, :, None] == kd[:, None]) & (kd >= 0)[:, None]
    if qo is not None:
        qo, ko = (x if x.dim() == 2 else x[None] for x in (qo, ko))
        m = m & (ko[:, None] <= qo[:, :, None])
    return m


def i32(x, device):
    return torch.as_tensor(x, dtype=torch.int32).to(device)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('b,tq,tk,h,hk,d', [
    (1, 1, 1, 1, 1, 64), (2, 1, 2, 4, 2, 128), (1, 3, 31, 2, 2, 32), (2, 33, 32, 2, 1, 64), (1, 64, 65, 3, 3, 96),
    (1, 129, 63, 4, 1, 128), (1, 130, 200, 2, 2, 8), (2, 40, 100, 5, 1, 72), (1, 5, 300, 8, 2, 80), (1, 200, 130, 2, 2, 104),
    (1, 2, 70, 40, 1, 64), (1, 257, 97, 6, 2, 88)])
def test_every_key(device, b, tq, tk, h, hk, d, dtype):
    q, k, v = heads(device, dtype, b, tq, tk, h, hk, d)
    check(masked_attention(q, k, v, 0.3), q, k, v, 0.3)
    check(masked_attention(q, k, v, 0.8, cap=2.0), q, k, v, 0.8, cap=2.0)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('sizes', [[1], [5, 1, 30], [64, 64, 64], [33, 95, 2, 70], [300], [20] * 17])
@pytest.mark.parametrize('d', [64, 128])
def test_packed_documents(device, sizes, d, dtype):
    docs = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes))
    q, k, v = heads(device, dtype, 1, len(docs), len(docs), 4, 2, d)
    ids = i32(docs * 1000003 % 2147483647, device)
    got = masked_attention(q, k, v, 0.25, keys=Tokens(ids))
    check(got, q, k, v, 0.25, seen=see(docs, docs))
    # in any order of the tokens
    mixed = torch.randperm(len(docs), generator=torch.Generator().manual_seed(3))
    got = masked_attention(q, k, v, 0.25, keys=Tokens(i32(docs[mixed], device)))
    check(got, q, k, v, 0.25, seen=see(docs[mixed], docs[mixed]))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('t', [1, 31, 64, 65, 200, 333])
def test_causal_prefix_and_frames(device, t, dtype):
    q, k, v = heads(device, dtype, 2, t, t, 4, 1, 64)
    docs, at = torch.zeros((t,), dtype=torch.int64), torch.arange(t)
    for order in (at, torch.where(at < t // 2, 0, at), at // 13, at - t, (at // 13) * (2 ** 31 // 40)):
        got = masked_attention(q, k, v, 0.2, keys=Tokens(i32(docs, device), i32(order, device)))
        check(got, q, k, v, 0.2, seen=see(docs, docs, order, order))


@pytest.mark.parametrize('dtype', DTYPES)
def test_padded_batch_and_empty_rows(device, dtype):
    t, lengths = 150, [150, 1, 0, 77]
    at = torch.arange(t)
    docs = torch.stack([torch.where(at < n, 0, -1 - at) for n in lengths])   # any negative id is padding
    q, k, v = heads(device, dtype, 4, t, t, 2, 2, 64)
    side = Tokens(i32(docs, device), i32(at.expand(4, t).contiguous(), device))
    got = masked_attention(q, k, v, 0.3, keys=side)
    check(got, q, k, v, 0.3, seen=see(docs, docs, at, at))
    for i, n in enumerate(lengths):
        assert (got[i, n:] == 0).all()
    # queries of a document that has no keys, and queries before every key
    qd, kd = torch.tensor([5, 0, 1, 0]), torch.tensor([0] * 70 + [1] * 30)
    qo, ko = torch.tensor([0, -1, 500, 200]), torch.arange(100)
    q, k, v = heads(device, dtype, 1, 4, 100, 2, 2, 64)
    got = masked_attention(q, k, v, 0.3, keys=Tokens(i32(kd, device), i32(ko, device)),
                           queries=Tokens(i32(qd, device), i32(qo, device), queries_only=True))
    check(got, q, k, v, 0.3, seen=see(qd, kd, qo, ko))
    assert (got[0, :2] == 0).all() and (got[0, 2:] != 0).any()
    assert (masked_attention(q, k[:, :0], v[:, :0], 0.3) == 0).all()
    assert masked_attention(q[:, :0], k, v, 0.3).shape == (1, 0, 2, 64)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('axes', [1, 2, 3])
@pytest.mark.parametrize('tq,tk,d', [(1, 90, 64), (100, 100, 64), (45, 130, 128)])
def test_distance_bias(device, axes, tq, tk, d, dtype):
    g = torch.Generator().manual_seed(axes + tq)
    q, k, v = heads(device, dtype, 2, tq, tk, 4, 2, d)
    qpos = torch.randint(0, 30, (2, tq, axes), generator=g).float()
    kpos = torch.randint(0, 30, (1, tk, axes), generator=g).float() + 0.5
    slopes = torch.rand((4, axes), generator=g) * torch.tensor([1.0, 0.1, -0.05, 0.0])[:, None]
    kd = torch.zeros(tk, dtype=torch.int64)
    kd[tk // 2:] = 1
    qd = torch.randint(0, 2, (2, tq), generator=g)
    for cap in (0.0, 4.0):
        got = masked_attention(q, k, v, 0.3, keys=Tokens(i32(kd, device), positions=kpos.to(device)),
                               queries=Tokens(i32(qd, device), positions=qpos.to(device)), cap=cap, slopes=slopes.to(device))
        check(got, q, k, v, 0.3, seen=see(qd, kd), cap=cap, slopes=slopes, qpos=qpos, kpos=kpos)
    # positions alone: every key is seen
    got = masked_attention(q, k, v, 0.3, keys=Tokens(positions=kpos[0].to(device)),
                           queries=Tokens(positions=qpos.to(device)), slopes=slopes.to(device))
    check(got, q, k, v, 0.3, slopes=slopes, qpos=qpos, kpos=kpos)


def test_far_positions_keep_their_distance(device):
    t = 70
    q, k, v = heads(device, torch.float32, 1, t, t, 2, 2, 64)
    pos = (torch.arange(t) + 2 ** 24 - 100).float()[:, None]
    slopes = torch.tensor([[0.5], [0.01]])
    got = masked_attention(q, k, v, 0.2, keys=Tokens(positions=pos.to(device)), slopes=slopes[:, 0].to(device))
    check(got, q, k, v, 0.2, slopes=slopes, qpos=pos[None], kpos=pos[None])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tk,b,h,hk', [(1000, 1, 4, 4), (4099, 3, 8, 2), (9000, 1, 16, 1)])
@pytest.mark.parametrize('d', [64, 128])
def test_single_tokens_over_long_keys(device, tk, b, h, hk, d, dtype):
    q, k, v = heads(device, dtype, b, 1, tk, h, hk, d)
    last = torch.tensor([[tk - 1], [10], [tk // 2]])[:b]
    at = torch.arange(tk)
    keys = Tokens(i32(torch.zeros(tk), device), i32(at, device), positions=at.float()[:, None].to(device))
    queries = Tokens(i32(torch.zeros((b, 1)), device), i32(last, device), last.float()[..., None].to(device), queries_only=True)
    slopes = 2.0 ** -torch.arange(2, 2 + h).float()[:, None]
    seen = see(torch.zeros((b, 1)), torch.zeros(tk), last, at)
    check(masked_attention(q, k, v, 0.3, keys=keys, queries=queries), q, k, v, 0.3, seen=seen)
    got = masked_attention(q, k, v, 0.3, keys=keys, queries=queries, cap=20.0, slopes=slopes.to(device))
    check(got, q, k, v, 0.3, seen=seen, cap=20.0, slopes=slopes, qpos=last.float()[..., None], kpos=at.float()[None, :, None])
    again = masked_attention(q, k, v, 0.3, keys=keys, queries=queries, cap=20.0, slopes=slopes.to(device))
    assert torch.equal(got, again)


@pytest.mark.parametrize('dtype', DTYPES)
def test_pooling_latents_of_packed_images(device, dtype):
    sizes = [100, 7, 0, 300, 64]
    kd = torch.repeat_interleave(torch.arange(5), torch.tensor(sizes))
    for latents in (1, 3, 12):
        qd = torch.arange(5).repeat_interleave(latents)
        q, k, v = heads(device, dtype, 1, len(qd), len(kd), 4, 4, 64)
        got = masked_attention(q, k, v, 0.3, keys=Tokens(i32(kd, device)), queries=Tokens(i32(qd, device), queries_only=True))
        check(got, q, k, v, 0.3, seen=see(qd, kd))
        assert (got[0, 2 * latents:3 * latents] == 0).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tq', [1, 90])
def test_what_unseen_keys_hold_does_not_matter(device, tq, dtype):
    # infinities and NaN in K and V of other documents, behind the order and in padding
    tk = 300
    kd = torch.tensor([0] * 100 + [1] * 100 + [-1] * 50 + [0] * 50)
    ko = torch.arange(tk)
    qd, qo = torch.tensor([0, 1, 0] * 30)[:tq], torch.full((tq,), 270)
    q, k, v = heads(device, dtype, 1, tq, tk, 2, 2, 64)
    keys, queries = Tokens(i32(kd, device), i32(ko, device)), Tokens(i32(qd, device), i32(qo, device), queries_only=True)
    seen = see(qd, kd, qo, ko)
    clean = masked_attention(q, k, v, 0.3, keys=keys, queries=queries)
    check(clean, q, k, v, 0.3, seen=seen)
    k2, v2 = k.clone(), v.clone()
    for at, x in ((210, float('nan')), (249, float('inf')), (271, float('-inf')), (299, float('nan'))):
        k2[:, at], v2[:, at] = x, x
    got = masked_attention(q, k2, v2, 0.3, keys=keys, queries=queries)
    check(got, q, k2, v2, 0.3, seen=seen)
    if tq > 1:
        v2[:, 150] = float('nan')     # seen by document 1, not by document 0
        k2[:, 160] = float('inf')
        got = masked_attention(q, k2, v2, 0.3, keys=keys, queries=queries)
        rows = qd == 0
        check(got[:, rows], q[:, rows], k2, v2, 0.3, seen=seen[:, rows])
        assert torch.isnan(got[:, ~rows]).all()


@pytest.mark.parametrize('dtype', DTYPES)
def test_seen_infinities_show(device, dtype):
    q, k, v = heads(device, dtype, 1, 40, 100, 1, 1, 64)
    docs = torch.zeros(100, dtype=torch.int64)
    docs[50:] = 1
    v[0, 3, 0, 5], v[0, 60, 0, 6] = float('inf'), float('nan')
    qd = torch.zeros(40, dtype=torch.int64)
    qd[20:] = 1
    got = masked_attention(q, k, v, 0.1, keys=Tokens(i32(docs, device)), queries=Tokens(i32(qd, device)))
    assert (got[0, :20, 0, 5] == float('inf')).all() and torch.isfinite(got[0, :20, 0, 6:]).all()
    assert torch.isnan(got[0, 20:, 0, 6]).all() and torch.isfinite(got[0, 20:, 0, :6]).all()


@pytest.mark.parametrize('dtype', DTYPES)
def test_sharp_growing_and_huge_scores(device, dtype):
    t = 260
    q, k, v = heads(device, dtype, 1, t, t, 1, 1, 64)
    q = torch.zeros_like(q)
    q[..., 0] = 1.0
    k = k * 0.05
    k[0, :, 0, 0] = torch.arange(t, device=device).to(dtype) * 0.5
    at = torch.arange(t)
    side = Tokens(i32(torch.zeros(t), device), i32(at, device))
    check(masked_attention(q, k, v, 1.0, keys=side), q, k, v, 1.0, seen=see(at * 0, at * 0, at, at))
    check(masked_attention(q, -k, v, 1.0, keys=side), q, -k, v, 1.0, seen=see(at * 0, at * 0, at, at))
    # scores near 2^13, and capped ones at the cap's two ends
    check(masked_attention(q * 64, k, v, 1.0, keys=side), q * 64, k, v, 1.0, seen=see(at * 0, at * 0, at, at))
    check(masked_attention(q * 64, k, v, 1.0, keys=side, cap=30.0), q * 64, k, v, 1.0, seen=see(at * 0, at * 0, at, at), cap=30.0)
    check(masked_attention(-q * 64, k, v, 1.0, cap=50.0), -q * 64, k, v, 1.0, cap=50.0)


@pytest.mark.parametrize('dtype', DTYPES)
def test_layouts(device, dtype):
    t, b, h, d = 77, 2, 3, 64
    g = torch.Generator().manual_seed(8)
    qkv = torch.randn((t, b, 3 * h * d), generator=g).to(dtype).to(device)      # the in-projection's (T, B, 3E)
    q, k, v = qkv.view(t, b, 3, h, d).permute(2, 1, 0, 3, 4)
    check(masked_attention(q, k, v, 0.125), q, k, v, 0.125)
    out = torch.full((t, b, h * d), 7.0, dtype=dtype, device=device)             # the out-projection's (T, B, E)
    view = out.view(t, b, h, d).transpose(0, 1)
    assert masked_attention(q, k, v, 0.125, out=view) is view
    check(view, q, k, v, 0.125)
    # rows off 16 bytes, a last dimension that is not contiguous, heads shared by expansion
    wide = torch.randn((b, t, h, d + 3), generator=g).to(dtype).to(device)
    check(masked_attention(wide[..., 1:1 + d], wide[..., 3:], wide[..., :d], 0.125), wide[..., 1:1 + d], wide[..., 3:],
          wide[..., :d], 0.125)
    turned = torch.randn((b, d, t, h), generator=g).to(dtype).to(device).permute(0, 2, 3, 1)
    one = k[:, :1, :1].expand(b, t, h, d)
    check(masked_attention(turned, one, v, 0.125), turned, one, v, 0.125)


def test_refuses_gradients_of_positions_and_out(device):
    q, k, v = heads(device, torch.float16, 1, 4, 4, 2, 2, 64)
    pos, slopes = torch.zeros((4, 1), device=device, requires_grad=True), torch.ones((2, 1), device=device)
    with pytest.raises(ValueError, match='backward'):
        masked_attention(q, k, v, 1.0, keys=Tokens(positions=pos), slopes=slopes)
    with pytest.raises(ValueError, match='backward'):
        masked_attention(q, k, v, 1.0, out=torch.empty_like(q).requires_grad_())
    with torch.no_grad():
        masked_attention(q, k, v, 1.0, keys=Tokens(positions=pos), slopes=slopes)


def test_more_batch_entries_than_a_schedule_takes(device):
    b = (1 << 20) + 5                                            # one token each: its output is its value
    docs = torch.zeros((b, 1), dtype=torch.int32, device=device)
    docs[::3] = -1
    v = torch.randn((b, 1, 1, 8), device=device).half()
    out = masked_attention(v, v, v, 1.0, keys=Tokens(docs))
    assert torch.equal(out, v * (docs >= 0)[..., None, None])


@pytest.mark.parametrize('tq,tk', [(1, 40), (1, 5000), (200, 200)])
def test_scores_of_minus_infinity(device, tq, tk):
    q, k, v = heads(device, torch.float16, 1, tq, tk, 1, 1, 64)
    q[..., 0] = 1.0
    q[0, 0, 0, 0] = 0.5
    k[0, :, 0, 0] = float('-inf')
    assert (masked_attention(q, k, v, 0.125) == 0).all()
    k[0, tk // 2, 0, 0] = 0.0                                    # one key left: its value
    assert torch.equal(masked_attention(q, k, v, 0.125), v[:, tk // 2:tk // 2 + 1].expand(1, tq, 1, 64))


def test_contiguous_inputs_off_16_bytes(device):
    b, t, h, d = 2, 40, 3, 64
    g = torch.Generator().manual_seed(18)
    flat = torch.randn(3 * b * t * h * d + 4, generator=g).to(torch.float16).to(device)
    q, k, v = (flat[1 + i + i * b * t * h * d:][:b * t * h * d].view(b, t, h, d) for i in range(3))
    check(masked_attention(q, k, v, 0.125), q, k, v, 0.125)


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
def test_agrees_with_unmasked_attention(device, dtype):
    from musc_hip import _attention_hip
    q, k, v = heads(device, dtype, 2, 300, 300, 4, 4, 64)
    flat = [x.transpose(1, 2).reshape(8, 300, 64) for x in (q, k, v)]
    old = _attention_hip.attention(*flat, 0.125).view(2, 4, 300, 64).transpose(1, 2)
    out, tol = reference(q, k, v, 0.125)
    new = masked_attention(q, k, v, 0.125)
    # both are within the tolerance (the unmasked fp16 kernel also rounds its scaled queries)
    assert ((new.double().cpu() - out).abs() <= tol).all()
    assert (new - old).abs().max() <= (2e-3 if dtype == torch.float16 else 1e-5)


def test_offsets_past_32_bits(device):
    # 2.3e9 elements of K (and V): the last heads and tokens lie past 2^31 elements
    tk, h, d = 70000, 256, 128
    g = torch.Generator(device=device).manual_seed(1)
    kv = torch.randn((1, tk, h, d), generator=g, device=device, dtype=torch.float16)
    q = torch.randn((1, 1, h, d), generator=g, device=device, dtype=torch.float16)
    got = masked_attention(q, kv, kv, 0.5)
    for at in (0, 131, 255):
        x = kv[0, :, at].double()
        p = torch.softmax(x @ q[0, 0, at].double() * 0.5, 0)
        ref, w = p @ x, p @ x.abs()
        assert ((got[0, 0, at].double() - ref).abs() <= 2.0 ** -10 * (w + ref.abs()) + 1e-5).all()


def test_graph_follows_tokens(device):
    # a captured step whose length and cache change between replays, beside eager calls
    b, tk, h, hk, d = 3, 2000, 8, 2, 128
    q, k, v = heads(device, torch.bfloat16, b, 1, tk, h, hk, d)
    at = torch.arange(tk)
    keys = Tokens(i32(torch.zeros(tk), device), i32(at, device))
    last = i32([[5], [700], [1999]], device)
    queries = Tokens(i32(torch.zeros((b, 1)), device), last, queries_only=True)
    masked_attention(q, k, v, 0.3, keys=keys, queries=queries)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keys.refresh()
        kept = masked_attention(q, k, v, 0.3, keys=keys, queries=queries)
    for step in range(4):
        last.copy_(i32([[step], [701 + step], [40 * step]], device))
        k[:, step] += 1
        if step == 2:
            keys.documents[:100] = -1
            keys.refresh()
        eager = masked_attention(q, k, v, 0.3, keys=keys, queries=queries)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, eager)
        seen = see(torch.zeros((b, 1)), keys.documents.cpu(), last.cpu(), at)
        check(kept, q, k, v, 0.3, seen=seen)


def test_two_streams_and_threads(device):
    import threading
    docs = torch.repeat_interleave(torch.arange(4), 100)
    q, k, v = heads(device, torch.float16, 1, 400, 400, 4, 4, 64)
    one = heads(device, torch.float16, 2, 1, 3000, 4, 4, 64)
    keys = Tokens(i32(docs, device))
    want = masked_attention(q, k, v, 0.3, keys=keys), masked_attention(*one, 0.3)
    torch.cuda.synchronize()
    got = {}

    def work(name):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[name] = [(masked_attention(q, k, v, 0.3, keys=keys), masked_attention(*one, 0.3)) for _ in range(5)]
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for results in got.values():
        for a, b in results:
            assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_no_tokens(device):
    empty = Tokens(torch.zeros((0,), dtype=torch.int32, device=device), torch.zeros((0,), dtype=torch.int32, device=device))
    q, k, v = (x.half().to(device) for x in torch.zeros((3, 2, 0, 4, 64)))
    assert masked_attention(q, k, v, 1.0, keys=empty).shape == (2, 0, 4, 64)
    one = torch.ones((2, 3, 4, 64), dtype=torch.float16, device=device)
    docs = i32([0, 0, 0], device)
    side = Tokens(docs, docs, queries_only=True)
    assert (masked_attention(one, k, v, 1.0, keys=empty, queries=side) == 0).all()
    assert masked_attention(one[:0], one[:0], one[:0], 1.0, keys=Tokens(docs)).shape == (0, 3, 4, 64)


def test_refusals(device):
    q, k, v = heads(device, torch.float16, 1, 4, 4, 2, 2, 64)
    docs = i32([0, 0, 1, 1], device)
    pos = torch.zeros((4, 2), device=device)
    for bad in (lambda: masked_attention(q[0], k, v, 1.0), lambda: masked_attention(q, k.float(), v, 1.0),
                lambda: masked_attention(q, k, v[:, :3], 1.0), lambda: masked_attention(q[:, :, :1], k, v, 1.0),
                lambda: masked_attention(q[..., :4], k[..., :4], v[..., :4], 1.0),
                lambda: masked_attention(q, k, v, 1.0, keys=Tokens(docs[:3])),
                lambda: masked_attention(q, k, v, 1.0, keys=Tokens(docs), queries=Tokens(docs, docs)),
                lambda: masked_attention(q, k, v, 1.0, keys=Tokens(docs, queries_only=True)),
                lambda: masked_attention(q, k, v, 1.0, keys=Tokens(docs), queries=Tokens()),
                lambda: masked_attention(q, k, v, 1.0, slopes=torch.ones(2, device=device)),
                lambda: masked_attention(q, k, v, 1.0, keys=Tokens(positions=pos), slopes=torch.ones((2, 1), device=device)),
                lambda: masked_attention(q, k, v, 1.0, cap=-1.0), lambda: masked_attention(q, k, v, float('nan')),
                lambda: masked_attention(q, k, v, 1.0, out=q[:, :1].expand_as(q)),
                lambda: masked_attention(q.clone().requires_grad_(), k, v, 1.0),
                lambda: Tokens(docs.long()), lambda: Tokens(None, docs), lambda: Tokens(docs, docs[:2]),
                lambda: Tokens(docs[::2]), lambda: Tokens(docs, positions=pos[:2].contiguous()),
                lambda: Tokens(positions=torch.zeros((4, 4), device=device))):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros((1, 4, 1, 136), device=device, dtype=torch.float16)
    with pytest.raises(ValueError, match='head width'):
        masked_attention(wide, wide, wide, 1.0)


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
@pytest.mark.parametrize('sizes', [[1000, 10, 20, 700, 5], [64] * 12 + [900], [1800, 400, 30], [3000]])
@pytest.mark.parametrize('h,hk', [(2, 2), (4, 2), (8, 2), (16, 2), (6, 2)])
def test_long_documents_among_short_ones(device, sizes, h, hk, dtype):
    # row tiles in parts (few of them, of very different work), with 1, 2, 4, 8 and 3 heads a key head
    docs = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes))
    t = len(docs)
    q, k, v = heads(device, dtype, 1, t, t, h, hk, 64)
    pos = torch.arange(t).float()[:, None]
    order = torch.arange(t)
    slopes = torch.full((h, 1), 0.01)
    tokens = Tokens(i32(docs, device), i32(order, device), pos.to(device))
    got = masked_attention(q, k, v, 0.3, keys=tokens, slopes=slopes.to(device), cap=30.0)
    rows = torch.randperm(t, generator=torch.Generator().manual_seed(1))[:300]
    check(got[:, rows], q[:, rows], k, v, 0.3, seen=see(docs[rows], docs, order[rows], order), cap=30.0, slopes=slopes,
          qpos=pos[rows][None], kpos=pos[None])
    assert torch.equal(got, masked_attention(q, k, v, 0.3, keys=tokens, slopes=slopes.to(device), cap=30.0))
    v[0, 5, 0, 3] = float('nan')          # seen by later rows of the first document only
    got = masked_attention(q, k, v, 0.3, keys=tokens)
    bad = torch.isnan(got).any(-1).any(-1)[0].cpu()
    assert bad[5:sizes[0]].all() and not bad[:5].any() and not bad[sizes[0]:].any()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('h,hk,d', [(2, 2, 64), (4, 1, 128), (8, 1, 96)])
def test_row_tiles_of_two_documents(device, h, hk, d, dtype):
    # long documents that meet inside row tiles, with padding and a single token between them
    sizes = [[330, 6, 517, 1, 490], [200, 0, 500, 300, 344]]
    docs = torch.stack([torch.repeat_interleave(torch.tensor([4, -1, 2, 9, 3]), torch.tensor(n)) for n in sizes])
    t = docs.shape[1]
    q, k, v = heads(device, dtype, 2, t, t, h, hk, d)
    tokens = Tokens(i32(docs, device))
    seen = see(docs, docs)
    out = torch.full_like(q, 7.0)
    got = masked_attention(q, k, v, 0.1, keys=tokens, out=out)
    check(got, q, k, v, 0.1, seen=seen)
    assert (got[docs.to(device) < 0] == 0).all()
    v[0, 3], k[1, 300] = float('nan'), float('inf')       # of the first document, and of the second entry's second
    held = masked_attention(q, k, v, 0.1, keys=tokens)
    same = torch.ones((2, t), dtype=torch.bool)
    same[0, :330], same[1, 200:700] = False, False
    # not to the bit: a workgroup that meets an unseen NaN adds its mixed tiles' products one by one, in
    # fp32 as the matrix instructions do but in another order, which the tolerance's n 2^-24 W covers
    for b in range(2):
        rows = same[b].nonzero()[:, 0]
        check(held[b:b + 1, rows], q[b:b + 1, rows], k[b:b + 1], v[b:b + 1], 0.1, seen=seen[b:b + 1, rows])
    assert torch.isnan(held[0, :330]).all() and torch.isnan(held[1, 200:700]).any(-1).all()


def test_schedule_is_a_permutation(device):
    for sizes in ([1], [128], [129, 300, 4], [2000] + [10] * 100, [700, 900, 1000], [300, -1, 77] * 30, [3000, 2500, 1200, 90], [150] * 109, [16384]):
        docs = i32(torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes).abs()), device)
        docs[::50] -= sum(n < 0 for n in sizes)                  # some padding
        tokens = Tokens(docs)
        at = 0
        for group in (1, 2, 4, 8):
            n = -(-len(docs) * group // 128)
            block = tokens._schedule[at:at + 4 + 5 * n + (9 * n + 4) // 5 + n // 4].cpu()
            at += len(block)
            work, order, first, jobs = block[4:4 + n], block[4 + n:4 + 2 * n], block[4 + 2 * n:4 + 3 * n], block[4 + 3 * n:]
            cuts, pieces = jobs[(9 * n + 4) // 5:][:n].tolist(), jobs[(9 * n + 4) // 5 + n:][:block[1]].tolist()
            assert sorted(order.tolist()) == list(range(n)) and (work[order.long()].diff() <= 0).all()
            jobs = jobs[:block[0]].tolist()
            parts = [x >> 24 for x in first.tolist()]
            assert sum(parts) == len(jobs) and max(parts) <= 8
            for tile, x in enumerate(first.tolist()):
                assert jobs[x & 0xffffff:(x & 0xffffff) + (x >> 24)] == [
                    tile | p << 20 | ((x >> 24) - 1) << 23 for p in range(x >> 24)]
            # pieces: every row of every tile once, those of the most work first, cut between documents
            rows = sorted((x & 1023, x >> 10 & 127, x >> 17) for x in pieces)
            whole = [(t, 0, 127) for t in range(n)]
            for t, low, high in rows:
                if low:
                    assert (t, 0, low - 1) in rows and high == 127 and not low % group
                    token = t * 128 // group + low // group
                    assert docs[token] != docs[token - 1] and cuts[t] & 127 == low
                    whole[t] = (t, 0, low - 1)
            assert rows == sorted(whole + [x for x in rows if x[1]]) and len(rows) <= n + n // 4
            of = {(t, bool(low)): cuts[t] >> 17 if low else cuts[t] >> 7 & 1023 if high < 127 else int(work[t]) for t, low, high in rows}
            sizes_of = [of[x & 1023, bool(x >> 10 & 127)] for x in pieces]
            assert sizes_of == sorted(sizes_of, reverse=True)
            if sizes == [700, 900, 1000]:
                assert len(rows) > n
