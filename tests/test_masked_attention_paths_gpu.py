"""Masked attention where a launch is chosen by its sizes: row tiles in parts of their keys for every
type and head width, sequences past the sorted tiles and the schedule's limit, and long flat tails.
Tolerances are test_masked_attention_gpu's."""
import ctypes

import pytest
import torch

from musc_hip import _masked_attention_hip, _runtime as rt
from musc_hip._masked_attention_hip import Tokens, masked_attention

from test_masked_attention_gpu import DTYPES, check, heads, i32, see

pytestmark = pytest.mark.gpu


@pytest.fixture
def workspaces(monkeypatch):
    """Workspace bytes that each call of a test asked for."""
    asked, pack = [], rt.PACK_MASKED_ATTENTION

    class Pack:
        @staticmethod
        def pack(*values):
            call, need = pack.pack(*values), ctypes.c_size_t()
            rt.check(rt.library().musc_masked_attention_workspace_bytes(call, ctypes.byref(need)), 'workspace')
            asked.append(need.value)
            return call

    monkeypatch.setattr(_masked_attention_hip.rt, 'PACK_MASKED_ATTENTION', Pack)
    return asked


def causal(device, sizes, batch=1, cuts=0):
    """Documents with an order, (T,) or (batch, T) rolled per entry with `cuts` padding tokens."""
    docs = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes))
    order = torch.arange(len(docs))
    if batch > 1:
        docs = torch.stack([docs.roll(100 * b) for b in range(batch)])
        order = order.expand(batch, -1).contiguous()
    if cuts:
        docs[..., :cuts] = -1
    return docs, order, Tokens(i32(docs, device), i32(order, device), order.float()[..., None].contiguous().to(device))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('h,hk,d', [(2, 2, 64), (4, 1, 72), (2, 2, 96), (2, 1, 104), (8, 1, 128), (2, 2, 128)])
@pytest.mark.parametrize('sizes,batch', [([2500, 30, 900], 1), ([1500, 700], 2)])
def test_row_tiles_in_parts(device, workspaces, sizes, batch, h, hk, d, dtype):
    docs, order, tokens = causal(device, sizes, batch, cuts=37)
    t = docs.shape[-1]
    q, k, v = heads(device, dtype, batch, t, t, h, hk, d)
    slopes, pos = torch.full((h, 1), 0.01), order.float()[..., None].expand(batch, t, 1)
    rows = torch.randperm(t, generator=torch.Generator().manual_seed(4))[:150]
    rows[0] = 0
    seen = see(docs[..., rows], docs, order[..., rows], order)
    got = masked_attention(q, k, v, 0.1, keys=tokens)
    check(got[:, rows], q[:, rows], k, v, 0.1, seen=seen)
    assert (got[docs.to(device).expand(batch, t) < 0] == 0).all()
    full = masked_attention(q, k, v, 0.1, keys=tokens, cap=20.0, slopes=slopes.to(device))
    check(full[:, rows], q[:, rows], k, v, 0.1, seen=seen, cap=20.0, slopes=slopes, qpos=pos[:, rows], kpos=pos)
    assert workspaces[0] > 0 and workspaces[1] > 0          # parts, and their join, ran
    assert torch.equal(full, masked_attention(q, k, v, 0.1, keys=tokens, cap=20.0, slopes=slopes.to(device)))
    # what a row does not see may hold anything
    k[:, :37], v[:, :37] = float('nan'), float('inf')       # padding
    v[:, t - 1] = float('nan')                              # seen by its own row alone
    held = masked_attention(q, k, v, 0.1, keys=tokens)
    rows = rows[rows != t - 1]
    check(held[:, rows], q[:, rows], k, v, 0.1, seen=see(docs[..., rows], docs, order[..., rows], order))
    assert torch.isnan(held[:, t - 1]).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('h,d', [(1, 64), (1, 128), (24, 64)])
def test_more_tiles_than_are_sorted_at_a_time(device, h, d, dtype):
    docs, order, tokens = causal(device, [4500, 300, 20])
    t = len(docs)
    q, k, v = heads(device, dtype, 1, t, t, h, h, d)
    rows = torch.randperm(t, generator=torch.Generator().manual_seed(5))[:60]
    got = masked_attention(q, k, v, 0.1, keys=tokens)
    check(got[:, rows], q[:, rows], k, v, 0.1, seen=see(docs[rows], docs, order[rows], order))
    got = masked_attention(q, k, v, 0.1, keys=Tokens(i32(docs, device)))
    check(got[:, rows], q[:, rows], k, v, 0.1, seen=see(docs[rows], docs))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('t,h,hk', [(16385, 1, 1), (18000, 2, 1), (900, 3, 1), (2500, 5, 1), (700, 14, 2)])
def test_without_a_schedule(device, t, h, hk, dtype):
    # more tokens than a schedule takes, or 3, 5 and 7 heads a key head
    docs = torch.arange(t) // 650
    order = torch.arange(t)
    q, k, v = heads(device, dtype, 1, t, t, h, hk, 64)
    rows = torch.randperm(t, generator=torch.Generator().manual_seed(6))[:100]
    got = masked_attention(q, k, v, 0.1, keys=Tokens(i32(docs, device)))
    check(got[:, rows], q[:, rows], k, v, 0.1, seen=see(docs[rows], docs))
    got = masked_attention(q, k, v, 0.1, keys=Tokens(i32(docs, device), i32(order, device)))
    check(got[:, rows], q[:, rows], k, v, 0.1, seen=see(docs[rows], docs, order[rows], order))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tq,tk', [(1, 2000), (1, 60000), (40, 60000), (200, 30000)])
def test_long_flat_tails(device, tq, tk, dtype):
    # one key e^15.6 = 2^22.5 above all others: each of these is below fp16's normal numbers in the product
    # with V, and they are up to 2^-6.6 of the sum together
    q, k, v = heads(device, dtype, 1, tq, tk, 1, 1, 64)
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    q[..., 0] = 1.0
    k[0, :, 0, 0] = -15.6
    k[0, tk // 3, 0, 0] = 0.0
    v = v * 0.1 + 1.0
    v[0, tk // 3] = -1.0
    check(masked_attention(q, k, v, 1.0), q, k, v, 1.0)


def test_extreme_documents_and_orders(device):
    most, least = 2 ** 31 - 1, -2 ** 31
    docs = torch.tensor([most, 0, least, most, 0, -1, most - 1, most])
    order = torch.tensor([most, least, 0, least, most, 5, 0, 0])
    q, k, v = heads(device, torch.float16, 1, 8, 8, 2, 2, 64)
    got = masked_attention(q, k, v, 0.3, keys=Tokens(i32(docs, device), i32(order, device)))
    check(got, q, k, v, 0.3, seen=see(docs, docs, order, order))


def test_two_graphs_of_one_batch(device):
    # two captured calls share Tokens (and nothing else), replayed beside one another and eager calls
    docs, order, tokens = causal(device, [1800, 500])
    t = len(docs)
    one, two = (heads(device, torch.bfloat16, 1, t, t, 2, 2, 64, seed=s) for s in (1, 2))
    want = [masked_attention(*x, 0.1, keys=tokens) for x in (one, two)]
    graphs, kept = [], []
    for x in (one, two):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            kept.append(masked_attention(*x, 0.1, keys=tokens))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = masked_attention(*one, 0.1, keys=tokens)
        torch.cuda.synchronize()
        assert torch.equal(kept[0], want[0]) and torch.equal(kept[1], want[1]) and torch.equal(eager, want[0])


@pytest.mark.parametrize('scale,cap', [(1e39, 0.0), (-1e300, 0.0), (1.0, 1e39), (float('inf'), 0.0), (1.0, float('inf')),
                                       (2.0 ** 61, 0.0), (1.0, 2.0 ** 61), (1.0, float('nan'))])
def test_refuses_scales_and_caps_past_the_range(device, scale, cap):
    q, k, v = heads(device, torch.float16, 1, 4, 4, 2, 2, 64)
    with pytest.raises(ValueError):
        masked_attention(q, k, v, scale, cap=cap)
