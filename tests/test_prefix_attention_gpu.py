"""Attention of a batch after a prefix that all entries share, against float64 on the same inputs with the
prefix's keys in front of each entry's: the tolerance is masked attention's (test_masked_attention_gpu.py)."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention, prefix_attention

from test_masked_attention_gpu import DTYPES, check, heads, i32
from test_masked_attention_gpu import see as see_own

pytestmark = pytest.mark.gpu


def shared(device, dtype, p, hk, d, seed=5):
    g = torch.Generator().manual_seed(seed * 100 + p + d)
    return tuple(torch.randn((p, hk, d), generator=g).to(dtype).to(device) for _ in range(2))


def joined(pk, k):
    return torch.cat([pk[None].expand(k.shape[0], -1, -1, -1), k], 1)


def check_prefix(got, q, k, v, pk, pv, scale, own=None, live=None, kpos=None, ppos=None, **kw):
    """own (B or 1, Tq, Tk): own keys that are seen; live (B or 1, Tq): queries that see the prefix"""
    seen, tq, p = None, q.shape[1], pk.shape[0]
    if own is not None:
        live = torch.ones(own.shape[:2], dtype=torch.bool) if live is None else live
        seen = torch.cat([live[:, :, None].expand(-1, -1, p), own], 2)
    if ppos is not None:
        kpos = torch.cat([ppos[None].expand(kpos.shape[0], -1, -1), kpos], 1)
    check(got, q, joined(pk, k), joined(pv, v), scale, seen=seen, kpos=kpos, **kw)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('b,tq,tk,p,h,hk,d', [
    (1, 1, 1, 1, 1, 1, 64), (2, 1, 5, 33, 4, 2, 128), (3, 1, 40, 300, 2, 2, 64), (40, 1, 70, 129, 8, 2, 96), (5, 7, 7, 64, 3, 1, 72),
    (2, 33, 33, 100, 2, 1, 64), (3, 64, 64, 65, 4, 4, 32), (2, 129, 129, 63, 4, 2, 128), (2, 140, 140, 500, 1, 1, 64),
    (3, 300, 300, 200, 2, 1, 80), (1, 50, 200, 1000, 2, 2, 64), (1, 3, 10, 5000, 4, 1, 128), (70, 1, 3, 2100, 4, 1, 64),
    (2, 1, 0, 77, 2, 2, 64), (1, 200, 0, 64, 2, 1, 64), (6, 20, 0, 300, 2, 1, 128), (2, 5, 9, 0, 2, 1, 64), (2, 130, 9, 0, 2, 1, 64)])
def test_every_key(device, b, tq, tk, p, h, hk, d, dtype):
    q, k, v = heads(device, dtype, b, tq, tk, h, hk, d)
    pk, pv = shared(device, dtype, p, hk, d)
    got = prefix_attention(q, k, v, pk, pv, 0.3)
    check_prefix(got, q, k, v, pk, pv, 0.3)
    assert torch.equal(got, prefix_attention(q, k, v, pk, pv, 0.3))
    check_prefix(prefix_attention(q, k, v, pk, pv, 0.8, cap=2.0), q, k, v, pk, pv, 0.8, cap=2.0)
    check_prefix(prefix_attention(q, k, v, pk, pv, 0.8, cap=200.0), q, k, v, pk, pv, 0.8, cap=200.0)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('t,p', [(1, 100), (30, 64), (77, 31), (200, 190)])
def test_padded_causal_batch(device, t, p, dtype):
    b, lengths = 4, [t, 0, 1, (t + 1) // 2]
    at = torch.arange(t)
    docs = torch.stack([torch.where(at < n, 3, -7) for n in lengths])
    q, k, v = heads(device, dtype, b, t, t, 4, 2, 64)
    pk, pv = shared(device, dtype, p, 2, 64)
    side = Tokens(i32(docs, device), i32(at.expand(b, t).contiguous(), device))
    got = prefix_attention(q, k, v, pk, pv, 0.3, keys=side)
    check_prefix(got, q, k, v, pk, pv, 0.3, see_own(docs, docs, at, at), docs >= 0)
    for i, n in enumerate(lengths):
        assert (got[i, n:] == 0).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('b,cache,p', [(1, 50, 40), (3, 600, 100), (33, 90, 1000), (9, 2500, 64)])
def test_single_tokens_after_a_prefix(device, b, cache, p, dtype):
    # caches filled to their own lengths, one query whose own keys are all behind it, one without a document
    h, hk, d = 8, 2, 128
    q, k, v = heads(device, dtype, b, 1, cache, h, hk, d)
    pk, pv = shared(device, dtype, p, hk, d)
    at = torch.arange(cache)
    last = torch.randint(0, cache, (b, 1), generator=torch.Generator().manual_seed(b))
    qd = torch.zeros((b, 1), dtype=torch.int64)
    if b > 1:
        last[1] = -1
        qd[-1] = -1
    keys = Tokens(i32(torch.zeros(cache), device), i32(at, device), (at.float() + p)[:, None].to(device))
    queries = Tokens(i32(qd, device), i32(last, device), (last.float() + p)[..., None].to(device), queries_only=True)
    own = see_own(qd, torch.zeros(cache), last, at)
    got = prefix_attention(q, k, v, pk, pv, 0.3, keys=keys, queries=queries)
    check_prefix(got, q, k, v, pk, pv, 0.3, own, qd >= 0)
    slopes, ppos = 2.0 ** -torch.arange(2, 2 + h).float()[:, None], torch.arange(p).float()[:, None]
    got = prefix_attention(q, k, v, pk, pv, 0.3, keys=keys, queries=queries, cap=20.0, slopes=slopes.to(device),
                           prefix_positions=ppos.to(device))
    check_prefix(got, q, k, v, pk, pv, 0.3, own, qd >= 0, (at.float() + p)[None, :, None], ppos, cap=20.0, slopes=slopes,
                 qpos=(last.float() + p)[..., None])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tq,d', [(1, 64), (20, 96), (200, 128)])
@pytest.mark.parametrize('axes', [1, 3])
def test_distance_bias(device, axes, tq, d, dtype):
    b, tk, p = 3, 60, 70
    g = torch.Generator().manual_seed(axes + tq)
    q, k, v = heads(device, dtype, b, tq, tk, 4, 2, d)
    pk, pv = shared(device, dtype, p, 2, d)
    qpos, kpos = torch.randint(0, 30, (b, tq, axes), generator=g).float(), torch.randint(0, 30, (b, tk, axes), generator=g).float()
    ppos = torch.randint(0, 30, (p, axes), generator=g).float() + 0.5
    slopes = torch.rand((4, axes), generator=g) * torch.tensor([1.0, 0.1, -0.05, 0.0])[:, None]
    for cap in (0.0, 4.0):
        got = prefix_attention(q, k, v, pk, pv, 0.3, keys=Tokens(positions=kpos.to(device)),
                               queries=Tokens(positions=qpos.to(device)), cap=cap, slopes=slopes.to(device),
                               prefix_positions=ppos.to(device))
        check_prefix(got, q, k, v, pk, pv, 0.3, kpos=kpos, ppos=ppos, cap=cap, slopes=slopes, qpos=qpos)


@pytest.mark.parametrize('dtype', DTYPES)
def test_packed_documents_after_a_prefix(device, dtype):
    sizes = [5, 1, 30, 64, 100]
    docs = torch.repeat_interleave(torch.arange(5), torch.tensor(sizes))
    q, k, v = heads(device, dtype, 1, 200, 200, 4, 4, 64)
    pk, pv = shared(device, dtype, 90, 4, 64)
    got = prefix_attention(q, k, v, pk, pv, 0.25, keys=Tokens(i32(docs * 1000003, device)))
    check_prefix(got, q, k, v, pk, pv, 0.25, see_own(docs, docs))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tq', [1, 90])
def test_what_unseen_keys_hold_does_not_matter(device, tq, dtype):
    b, tk, p = 3, 150, 45
    at, new = torch.arange(tk), torch.full((b, tq), 60)
    q, k, v = heads(device, dtype, b, tq, tk, 2, 2, 64)
    room_k, room_v = shared(device, dtype, 64, 2, 64)
    room_k[p:], room_v[p:] = float('nan'), float('inf')     # behind the prefix, in its own last tile
    keys, queries = Tokens(i32(at * 0, device), i32(at, device)), Tokens(i32(new * 0, device), i32(new, device), queries_only=True)
    k2, v2 = k.clone(), v.clone()
    k2[:, 61:], v2[:, 61:] = float('inf'), float('nan')
    got = prefix_attention(q, k2, v2, room_k[:p], room_v[:p], 0.3, keys=keys, queries=queries)
    check_prefix(got, q, k, v, room_k[:p], room_v[:p], 0.3, see_own(new * 0, at * 0, new, at))
    room_v[3, 0, 5] = float('nan')                          # seen by all
    got = prefix_attention(q, k2, v2, room_k[:p], room_v[:p], 0.3, keys=keys, queries=queries)
    assert torch.isnan(got[..., 0, 5]).all() and torch.isfinite(got[..., 1, :]).all() and torch.isfinite(got[..., 0, :5]).all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('b,tq,p', [(3, 1, 45), (40, 1, 900), (3, 90, 45)])
def test_huge_numbers_in_unseen_keys(device, b, tq, p, dtype):
    tk = 150
    at, new = torch.arange(tk), torch.full((b, tq), 60)
    qd = torch.zeros((b, tq), dtype=torch.int64)
    qd[:, tq // 2 + 1:] = -1
    q, k, v = heads(device, dtype, b, tq, tk, 2, 2, 64)
    pk, pv = shared(device, dtype, p, 2, 64)
    k[:, 61:] *= 1e30
    v[:, 61:] *= 1e30
    keys, queries = Tokens(i32(at * 0, device), i32(at, device)), Tokens(i32(qd, device), i32(new, device), queries_only=True)
    got = prefix_attention(q, k, v, pk, pv, 0.3, keys=keys, queries=queries)
    k, v = k.cpu(), v.cpu()
    k[:, 61:] = v[:, 61:] = 0
    check_prefix(got, q.cpu(), k, v, pk.cpu(), pv.cpu(), 0.3, see_own(qd, at * 0, new, at), qd >= 0)


@pytest.mark.parametrize('tq', [1, 60])
def test_documents_without_own_keys(device, tq):
    b, p = 3, 70
    qd = torch.zeros((b, tq), dtype=torch.int64)
    qd[1] = -1
    q, k, v = heads(device, torch.float16, b, tq, 4, 2, 2, 64)
    pk, pv = shared(device, torch.float16, p, 2, 64)
    none = torch.empty((b, 0), dtype=torch.int32, device=device)
    side, queries = Tokens(none, none.clone()), Tokens(i32(qd, device), i32(qd * 0, device), queries_only=True)
    got = prefix_attention(q, k[:, :0], v[:, :0], pk, pv, 0.3, keys=side, queries=queries)
    check_prefix(got, q, k[:, :0], v[:, :0], pk, pv, 0.3, torch.ones((b, tq, 0), dtype=torch.bool), qd >= 0)
    assert (got[1] == 0).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('t', [3, 150])
def test_layouts(device, t, dtype):
    b, h, d, p = 3, 3, 64, 50
    g = torch.Generator().manual_seed(8)
    make = lambda *s: torch.randn(s, generator=g).to(dtype).to(device)  # noqa: E731
    qkv, pkv = make(t, b, 3 * h * d), make(p, 2 * h * d)                # projections' layouts
    q, k, v = qkv.view(t, b, 3, h, d).permute(2, 1, 0, 3, 4)
    pk, pv = pkv.view(p, 2, h, d).unbind(1)
    out = torch.full((t, b, h * d), 7.0, dtype=dtype, device=device)
    view = out.view(t, b, h, d).transpose(0, 1)
    assert prefix_attention(q, k, v, pk, pv, 0.125, out=view) is view
    check_prefix(view, q, k, v, pk, pv, 0.125)
    wide, wide_p = make(b, t, h, d + 3), make(p, h, d + 3)              # rows off 16 bytes
    q, k, v = wide[..., 1:1 + d], wide[..., 3:], wide[..., :d]
    check_prefix(prefix_attention(q, k, v, wide_p[..., 2:2 + d], pv, 0.125), q, k, v, wide_p[..., 2:2 + d], pv, 0.125)
    one = pk[:1].expand(p, h, d)                                        # one key as the whole prefix
    turned = make(h, d, p).permute(2, 0, 1)
    check_prefix(prefix_attention(q, k, v, one, turned, 0.125), q, k, v, one, turned, 0.125)


@pytest.mark.parametrize('dtype', DTYPES)
def test_agrees_with_masked_attention_of_the_copies(device, dtype):
    q, k, v = heads(device, dtype, 5, 4, 30, 4, 2, 64)
    pk, pv = shared(device, dtype, 100, 2, 64)
    a, b = prefix_attention(q, k, v, pk, pv, 0.3), masked_attention(q, joined(pk, k), joined(pv, v), 0.3)
    check_prefix(a, q, k, v, pk, pv, 0.3)
    check_prefix(b, q, k, v, pk, pv, 0.3)


@pytest.mark.parametrize('tq', [1, 200])
def test_captured(device, tq):
    b, tk, p = 6, 200, 300
    q, k, v = heads(device, torch.bfloat16, b, tq, tk, 8, 2, 64)
    pk, pv = shared(device, torch.bfloat16, p, 2, 64)
    keys = Tokens(i32(torch.zeros((b, tk)), device), i32(torch.arange(tk).expand(b, tk), device).contiguous())
    last = i32(torch.arange(tq).expand(b, tq), device).contiguous()
    queries = Tokens(torch.zeros_like(last), last, queries_only=True)
    prefix_attention(q, k, v, pk, pv, 0.1, keys=keys, queries=queries)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = prefix_attention(q, k, v, pk, pv, 0.1, keys=keys, queries=queries)
    for turn in range(3):
        if tq == 1:
            last.add_(40)
        for n, x in enumerate((q, pk, pv, v)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * turn + n)))
        eager = prefix_attention(q, k, v, pk, pv, 0.1, keys=keys, queries=queries)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, eager)
        check_prefix(kept, q, k, v, pk, pv, 0.1, see_own(torch.zeros((b, tq)), torch.zeros((b, tk)), last.cpu(), torch.arange(tk).expand(b, tk)))


def test_refusals(device):
    q, k, v = heads(device, torch.float16, 2, 4, 8, 4, 2, 64)
    pk, pv = shared(device, torch.float16, 10, 2, 64)
    for bad in (pk[:, :1], pk[..., :32], pk.float(), pk.cpu(), pk[None], None):
        with pytest.raises(ValueError, match='prefix_k'):
            prefix_attention(q, k, v, bad, pv, 1.0)
    with pytest.raises(ValueError, match='prefix_v'):
        prefix_attention(q, k, v, pk, pv[:9], 1.0)
    with pytest.raises(ValueError, match='backward'):
        prefix_attention(q, k, v, pk.clone().requires_grad_(), pv, 1.0)
    pos = Tokens(positions=torch.zeros((8, 1), device=device))
    qpos = Tokens(positions=torch.zeros((4, 1), device=device))
    for bad in (None, torch.zeros((9, 1), device=device), torch.zeros((10, 2), device=device), torch.zeros((10, 1)),
                torch.zeros((10, 1), dtype=torch.float64, device=device)):
        with pytest.raises(ValueError, match='prefix_positions'):
            prefix_attention(q, k, v, pk, pv, 1.0, keys=pos, queries=qpos, slopes=torch.ones(4, device=device), prefix_positions=bad)
    empty = prefix_attention(q[:, :0], k, v, pk, pv, 1.0)
    assert empty.shape == (2, 0, 4, 64)
    assert (prefix_attention(q, k[:, :0], v[:, :0], pk[:0], pv[:0], 1.0) == 0).all()


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
@pytest.mark.parametrize('b,tq', [(2, 1), (3, 200)])
def test_prefixes_past_32_bit_offsets(device, b, tq, dtype):
    """Heads of a wide prefix whose last tokens lie more than 2^32 bytes after the first."""
    p, apart, d = 2100, (1 << 20) + 512, 64
    wide = torch.empty((p, apart * (2 if dtype == torch.float16 else 1)), dtype=dtype, device=device)
    q, k, v = heads(device, dtype, b, tq, 9, 2, 1, d)
    pk, pv = shared(device, dtype, p, 1, d)
    wide[:, 512:576], wide[:, -128:-64] = pk[:, 0], pv[:, 0]
    assert (p - 64) * wide.stride(0) * wide.element_size() > 1 << 32
    got = prefix_attention(q, k, v, wide[:, None, 512:576], wide[:, None, -128:-64], 0.3)
    check_prefix(got, q, k, v, pk, pv, 0.3)
