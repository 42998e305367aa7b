"""Attention with a sliding window and sinks against float64 on the same inputs: the tolerance is
masked attention's (test_masked_attention_gpu.py), the keys that are seen are fewer."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention

from test_masked_attention_gpu import DTYPES, check, heads, i32
from test_masked_attention_gpu import see as see_all

pytestmark = pytest.mark.gpu


def see(qd, kd, qo, ko, window, sinks):
    qo, ko = (x.long() if x.dim() == 2 else x.long()[None] for x in (qo, ko))
    back = qo[:, :, None] - ko[:, None]
    first = ((ko >= 0) & (ko < sinks))[:, None]
    return see_all(qd, kd, qo, ko) & ((back < window) | first)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('t,window,sinks', [
    (1, 1, 0), (31, 1, 0), (64, 5, 1), (65, 64, 0), (200, 63, 64), (333, 17, 100), (333, 1, 3), (200, 1000, 2), (130, 2147483647, 0)])
def test_causal(device, t, window, sinks, dtype):
    q, k, v = heads(device, dtype, 2, t, t, 4, 2, 64)
    docs, at = torch.zeros((t,), dtype=torch.int64), torch.arange(t)
    got = masked_attention(q, k, v, 0.2, keys=Tokens(i32(docs, device), i32(at, device)), window=window, sinks=sinks)
    check(got, q, k, v, 0.2, seen=see(docs, docs, at, at, window, sinks))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('d', [32, 80, 96, 128])
def test_orders(device, d, dtype):
    # frames, a prefix that sees itself, negative orders, the ends of int32, tokens in any order
    t = 150
    q, k, v = heads(device, dtype, 1, t, t, 6, 3, d)
    docs, at = torch.arange(t) // 90, torch.arange(t) % 90
    mixed = torch.randperm(t, generator=torch.Generator().manual_seed(d))
    for order, window, sinks in ((at // 13, 2, 1), (torch.where(at < 40, 0, at), 20, 0), (at - 60, 7, 5), (at - 60, 30, 0),
                                 (at[mixed], 11, 4), (at + 2 ** 31 - 90, 9, 2 ** 31 - 85), (at - 2 ** 31, 9, 3),
                                 (at * (2 ** 32 // 90) - 2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1)):
        got = masked_attention(q, k, v, 0.2, keys=Tokens(i32(docs, device), i32(order, device)), window=window, sinks=sinks)
        check(got, q, k, v, 0.2, seen=see(docs, docs, order, order, window, sinks))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('cap', [0.0, 20.0, 300.0])
@pytest.mark.parametrize('d', [64, 72, 128])
def test_caps_and_distance(device, d, cap, dtype):
    t = 140
    q, k, v = heads(device, dtype, 2, t, t, 4, 1, d)
    docs, at = torch.zeros(t, dtype=torch.int64), torch.arange(t)
    pos = at.float()[:, None]
    slopes = 2.0 ** -torch.arange(1, 5).float()[:, None]
    seen = see(docs, docs, at, at, 30, 5)
    side = Tokens(i32(docs, device), i32(at, device), pos.to(device))
    check(masked_attention(q, k, v, 0.3, keys=side, cap=cap, window=30, sinks=5), q, k, v, 0.3, seen=seen, cap=cap)
    got = masked_attention(q, k, v, 0.3, keys=side, cap=cap, slopes=slopes.to(device), window=30, sinks=5)
    check(got, q, k, v, 0.3, seen=seen, cap=cap, slopes=slopes, qpos=pos[None], kpos=pos[None])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tk,b,h,hk', [(40, 2, 2, 1), (1000, 1, 4, 4), (4099, 3, 8, 2), (20000, 2, 16, 1)])
@pytest.mark.parametrize('d', [64, 128])
def test_single_tokens_over_long_keys(device, tk, b, h, hk, d, dtype):
    q, k, v = heads(device, dtype, b, 1, tk, h, hk, d)
    last = torch.tensor([[tk - 1], [10], [tk // 2]])[:b]
    at = torch.arange(tk)
    keys = Tokens(i32(torch.zeros(tk), device), i32(at, device), positions=at.float()[:, None].to(device))
    queries = Tokens(i32(torch.zeros((b, 1)), device), i32(last, device), last.float()[..., None].to(device), queries_only=True)
    slopes = 2.0 ** -torch.arange(2, 2 + h).float()[:, None]
    for window, sinks in ((1, 0), (33, 4), (700, 1), (3001, 100), (tk, 0)):
        seen = see(torch.zeros((b, 1)), torch.zeros(tk), last, at, window, sinks)
        got = masked_attention(q, k, v, 0.3, keys=keys, queries=queries, window=window, sinks=sinks)
        check(got, q, k, v, 0.3, seen=seen)
        assert torch.equal(got, masked_attention(q, k, v, 0.3, keys=keys, queries=queries, window=window, sinks=sinks))
    got = masked_attention(q, k, v, 0.3, keys=keys, queries=queries, cap=20.0, slopes=slopes.to(device), window=700, sinks=3)
    check(got, q, k, v, 0.3, seen=see(torch.zeros((b, 1)), torch.zeros(tk), last, at, 700, 3), cap=20.0, slopes=slopes,
          qpos=last.float()[..., None], kpos=at.float()[None, :, None])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tq,tk,h,hk', [(40, 5000, 1, 1), (100, 9000, 2, 1), (300, 4500, 4, 4)])
def test_some_rows_over_long_keys(device, tq, tk, h, hk, dtype):
    # a stretch of new tokens over a cache: tiles in more than one 64, shared out between workgroups
    q, k, v = heads(device, dtype, 1, tq, tk, h, hk, 64)
    at, new = torch.arange(tk), torch.arange(tk - 200 - tq, tk - 200)
    keys = Tokens(i32(torch.zeros(tk), device), i32(at, device))
    queries = Tokens(i32(torch.zeros(tq), device), i32(new, device), queries_only=True)
    for window, sinks in ((1, 0), (50, 4), (2500, 300), (tk, 0)):
        got = masked_attention(q, k, v, 0.3, keys=keys, queries=queries, window=window, sinks=sinks)
        check(got, q, k, v, 0.3, seen=see(torch.zeros(tq), torch.zeros(tk), new, at, window, sinks))


@pytest.mark.parametrize('tq,tk', [(1, 140000), (40, 270000)])
def test_more_tiles_than_a_word_tells_apart(device, tq, tk):
    q, k, v = heads(device, torch.float16, 1, tq, tk, 1, 1, 8)
    at = torch.arange(tk)
    keys = Tokens(i32(torch.zeros(tk), device), i32(at, device))
    for last, window, sinks in ((tk - 1, 100, 2), (tk - 1, 6000, 0), (tk // 2, 70, 0), (500, 100, 5)):
        new = torch.arange(last - tq + 1, last + 1)
        queries = Tokens(i32(torch.zeros(tq), device), i32(new, device), queries_only=True)
        got = masked_attention(q, k, v, 0.3, keys=keys, queries=queries, window=window, sinks=sinks)
        check(got, q, k, v, 0.3, seen=see(torch.zeros(tq), torch.zeros(tk), new, at, window, sinks))


@pytest.mark.parametrize('dtype', DTYPES)
def test_padded_batch_and_empty_rows(device, dtype):
    t, lengths = 150, [150, 1, 0, 77]
    at = torch.arange(t)
    docs = torch.stack([torch.where(at < n, 0, -1 - at) for n in lengths])
    q, k, v = heads(device, dtype, 4, t, t, 2, 2, 64)
    side = Tokens(i32(docs, device), i32(at.expand(4, t).contiguous(), device))
    got = masked_attention(q, k, v, 0.3, keys=side, window=20, sinks=2)
    check(got, q, k, v, 0.3, seen=see(docs, docs, at, at, 20, 2))
    for i, n in enumerate(lengths):
        assert (got[i, n:] == 0).all()
    # queries of other documents, before every key, and far behind the last key without sinks
    qd, kd = torch.tensor([5, 0, 1, 0, 1]), torch.tensor([0] * 70 + [1] * 30)
    qo, ko = torch.tensor([0, -1, 500, 75, 105]), torch.arange(100)
    q, k, v = heads(device, dtype, 1, 5, 100, 2, 2, 64)
    got = masked_attention(q, k, v, 0.3, keys=Tokens(i32(kd, device), i32(ko, device)),
                           queries=Tokens(i32(qd, device), i32(qo, device), queries_only=True), window=10)
    check(got, q, k, v, 0.3, seen=see(qd, kd, qo, ko, 10, 0))
    assert (got[0, :3] == 0).all() and (got[0, 3:] != 0).any(-1).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tq', [1, 90])
def test_what_unseen_keys_hold_does_not_matter(device, tq, dtype):
    tk = 300
    at, new = torch.arange(tk), torch.arange(200, 200 + tq)
    q, k, v = heads(device, dtype, 1, tq, tk, 2, 2, 64)
    keys = Tokens(i32(at * 0, device), i32(at, device))
    queries = Tokens(i32(new * 0, device), i32(new, device), queries_only=True)
    seen = see(new * 0, at * 0, new, at, 40, 3)
    unseen = ~seen[0].any(0)
    k2, v2 = k.clone(), v.clone()
    for n, i in enumerate(unseen.nonzero()[:, 0].tolist()):
        k2[:, i] = v2[:, i] = (float('nan'), float('inf'), float('-inf'))[n % 3]
    got = masked_attention(q, k2, v2, 0.3, keys=keys, queries=queries, window=40, sinks=3)
    check(got, q, k2, v2, 0.3, seen=seen)
    check(masked_attention(q, k, v, 0.3, keys=keys, queries=queries, window=40, sinks=3), q, k, v, 0.3, seen=seen)
    if tq > 1:      # keys that some rows see and others do not
        v2[:, 250] = float('nan')
        got = masked_attention(q, k2, v2, 0.3, keys=keys, queries=queries, window=40, sinks=3)
        sees = seen[0, :, 250]
        check(got[:, ~sees], q[:, ~sees], k2, v2, 0.3, seen=seen[:, ~sees])
        assert torch.isnan(got[:, sees]).all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('tq', [1, 90])
@pytest.mark.parametrize('huge', [1e10, 1e30, 3e38])
def test_huge_numbers_in_unseen_keys(device, huge, tq, dtype):
    # what memory that was never written may hold, beside keys that are seen: behind the queries, before the
    # window, in padding, and padded queries that would see them
    tk = 300
    at, new = torch.arange(tk), torch.arange(200, 200 + tq)
    kd = torch.where(at < 290, 0, -1)
    qd = torch.zeros(tq, dtype=torch.int64)
    qd[tq // 2 + 1:] = -1
    q, k, v = heads(device, dtype, 2, tq, tk, 2, 2, 64)
    keys = Tokens(i32(kd, device), i32(at, device))
    queries = Tokens(i32(qd, device), i32(new, device), queries_only=True)
    seen = see(qd, kd, new, at, 40, 3)
    unseen = ~seen[0].any(0)
    k[:, unseen.to(device)] *= huge
    v[:, unseen.to(device)] *= huge
    got = masked_attention(q, k, v, 0.3, keys=keys, queries=queries, window=40, sinks=3)
    check(got, q, torch.where(unseen[None, :, None, None], 0, k.cpu()), torch.where(unseen[None, :, None, None], 0, v.cpu()), 0.3,
          seen=seen)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('d', [64, 96])
def test_documents_and_keys_of_different_sizes(device, d, dtype):
    sizes, scales = [40, 70, 20, 100, 5, 65], torch.tensor([1.0, 1e12, 1e-12, 1e5, 1e-3, 1e20])
    docs = torch.repeat_interleave(torch.arange(6), torch.tensor(sizes))
    at = torch.cat([torch.arange(n) for n in sizes])
    q, k, v = heads(device, torch.float32, 1, 300, 300, 2, 1, d)
    of = scales[docs][None, :, None, None].to(device)
    q, k, v = (q / of).to(dtype), (k * of).to(dtype), (v * of).to(dtype)
    side = Tokens(i32(docs, device), i32(at, device))
    got = masked_attention(q, k, v, 0.2, keys=side, window=33, sinks=2)
    check(got, q, k, v, 0.2, seen=see(docs, docs, at, at, 33, 2))
    # one document whose values grow and shrink by 2^60 over its length
    at = torch.arange(300)
    grow = (2.0 ** (30 - (at - 150).abs() / 5).floor()).to(device)[None, :, None, None]
    q, k, v = heads(device, torch.float32, 1, 300, 300, 2, 1, d)
    k, v, q = (k * grow ** 0.1).to(dtype), (v * grow).to(dtype), q.to(dtype)
    side = Tokens(i32(at * 0, device), i32(at, device))
    got = masked_attention(q, k, v, 0.2, keys=side, window=20)
    check(got, q, k, v, 0.2, seen=see(at * 0, at * 0, at, at, 20, 0))


@pytest.mark.parametrize('tq', [1, 100])
@pytest.mark.parametrize('size', [1e-30, 1e-12, 1e15])
def test_fp32_sizes(device, size, tq):
    at = torch.arange(150)
    q, k, v = heads(device, torch.float32, 1, tq, 150, 2, 2, 64)
    q, k, v = q / size, k * size, v * size
    keys = Tokens(i32(at * 0, device), i32(at, device))
    queries = Tokens(i32(at[:tq] * 0, device), i32(at[-tq:], device), queries_only=True)
    got = masked_attention(q, k, v, 0.2, keys=keys, queries=queries, window=60, sinks=1)
    check(got, q, k, v, 0.2, seen=see(at[:tq] * 0, at * 0, at[-tq:], at, 60, 1))


def test_fp32_infinities_that_are_seen(device):
    t = 120
    q, k, v = heads(device, torch.float32, 1, t, t, 1, 1, 64)
    at = torch.arange(t)
    side = Tokens(i32(at * 0, device), i32(at, device))
    v[0, 30, 0, 5], v[0, 70, 0, 6] = float('inf'), float('nan')
    got = masked_attention(q, k, v, 0.1, keys=side, window=20)
    assert (got[0, 30:50, 0, 5] == float('inf')).all() and torch.isnan(got[0, 70:90, 0, 6]).all()
    got[0, 30:50, 0, 5] = got[0, 70:90, 0, 6] = 0
    assert torch.isfinite(got).all()
    k[0, 100, 0, 3] = float('nan')
    q[0, 10, 0, 0] = float('inf')
    got = masked_attention(q, k, v, 0.1, keys=side, window=20)
    assert torch.isnan(got[0, 100:]).all() and torch.isnan(got[0, 10]).all()
    assert torch.isfinite(got[0, 11:30]).all() and torch.isfinite(got[0, :10]).all()


@pytest.mark.parametrize('dtype', DTYPES)
def test_a_window_over_everything_is_masked_attention(device, dtype):
    t = 400
    q, k, v = heads(device, dtype, 1, t, t, 4, 2, 64)
    side = Tokens(i32(torch.arange(t) // 170, device), i32(torch.arange(t) % 170, device))
    a, b = masked_attention(q, k, v, 0.2, keys=side, window=170), masked_attention(q, k, v, 0.2, keys=side)
    # each is within its tolerance of the exact values
    seen = see(torch.arange(t) // 170, torch.arange(t) // 170, torch.arange(t) % 170, torch.arange(t) % 170, 170, 0)
    check(a, q, k, v, 0.2, seen=seen)
    check(b, q, k, v, 0.2, seen=seen)


def test_captured_with_moving_queries(device):
    tk, b = 5000, 3
    q, k, v = heads(device, torch.bfloat16, b, 1, tk, 8, 2, 64)
    keys = Tokens(i32(torch.zeros((b, tk)), device), i32(torch.arange(tk).expand(b, tk), device).contiguous())
    last = i32(torch.tensor([[100], [2000], [4000]]), device)
    queries = Tokens(torch.zeros_like(last), last, queries_only=True)
    masked_attention(q, k, v, 0.1, keys=keys, queries=queries, window=900, sinks=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = masked_attention(q, k, v, 0.1, keys=keys, queries=queries, window=900, sinks=4)
    for turn in range(4):
        last.add_(207)
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(turn)))
        eager = masked_attention(q, k, v, 0.1, keys=keys, queries=queries, window=900, sinks=4)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, eager)
        check(kept, q, k, v, 0.1, seen=see(torch.zeros((b, 1)), torch.zeros((b, tk)), last.cpu(), torch.arange(tk).expand(b, tk), 900, 4))


def test_refusals(device):
    q, k, v = heads(device, torch.float16, 1, 8, 8, 2, 2, 64)
    at = i32(torch.arange(8), device)
    side = Tokens(torch.zeros_like(at), at)
    for window, sinks in ((-1, 0), (0, 2), (4, -1), (1 << 31, 0), (4, 1 << 31)):
        with pytest.raises(ValueError, match='window'):
            masked_attention(q, k, v, 1.0, keys=side, window=window, sinks=sinks)
    with pytest.raises(TypeError):
        masked_attention(q, k, v, 1.0, keys=side, window=2.5)
    for keys in (None, Tokens(torch.zeros_like(at))):
        with pytest.raises(ValueError, match='order'):
            masked_attention(q, k, v, 1.0, keys=keys, window=4)
    with pytest.raises(ValueError, match='backward'):
        masked_attention(q.requires_grad_(), k, v, 1.0, keys=side, window=4)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('tq', [1, 40, 300])
def test_caches_past_32_bit_offsets(device, tq, dtype):
    """Heads of a wide cache, a token every 8 Ki numbers: the last keys lie more than 2^32 bytes after the first."""
    tk, h, d = (1 << 18 if dtype == torch.bfloat16 else 1 << 17) + 1037, 2, 64
    cache = torch.empty((1, tk, 1 << 13), dtype=dtype, device=device)
    q, k, v = heads(device, dtype, 1, tq, tk, h, 1, d)
    cache[..., 128:192], cache[..., 4096:4160] = k[:, :, 0], v[:, :, 0]
    at = torch.arange(tk)
    keys = Tokens(i32(torch.zeros(tk), device), i32(at, device))
    queries = Tokens(i32(torch.zeros(tq), device), i32(at[-tq:], device), queries_only=True)
    assert (tk - 300) * (1 << 13) * cache.element_size() > 1 << 32
    got = masked_attention(q, cache[:, :, None, 128:192], cache[:, :, None, 4096:4160], 0.3, keys=keys, queries=queries,
                           window=700, sinks=3)
    some = torch.cat([at[:32], at[-1100:]])
    seen = see(torch.zeros(tq), torch.zeros(len(some)), at[-tq:], some, 700, 3)
    check(got, q, k[:, some], v[:, some], 0.3, seen=seen)
