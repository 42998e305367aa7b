"""Head norms with rotary positions, windows with sinks and shared prefixes as the blocks of a tower use them:
a clip through pre-norm blocks whose tokens see the last frames and the first, new tokens one at a time over
a cache, and test images beside common reference images.

Tolerance: every step is compared with the float64 step on the block's own stored input, so nothing is carried
from step to step: the linear maps are torch's."""
import threading

import pytest
import torch
from torch.nn import functional as F

from musc_hip import _layers_hip
from musc_hip._masked_attention_hip import Tokens, masked_attention, prefix_attention
from musc_hip._rotary_hip import RotaryAxes, norm_rotary

from test_norm_rotary_gpu import check as check_heads
from test_packed_block_gpu import DIM, HEADS, KV, WIDTH, weights
from test_prefix_attention_gpu import check_prefix
from test_masked_attention_gpu import DTYPES, check as check_attention, i32
from test_window_attention_gpu import see

pytestmark = pytest.mark.gpu

FRAMES, SIDE = 9, 6
SECTIONS = (8, 12, 12)


def clip(device):
    pos = torch.stack(torch.meshgrid(torch.arange(FRAMES), torch.arange(SIDE), torch.arange(SIDE), indexing='ij'), -1).reshape(-1, 3).float()
    order = pos[:, 0].long()
    return pos, order, Tokens(i32(order * 0, device), i32(order, device))


def heads_of(x, w, positions, axes, head_weight):
    qkv = F.linear(_layers_hip.rms_norm(x, w['n1'], 1e-6), w['qkv']).view(*x.shape[:2], HEADS + 2 * KV, DIM)
    q, k, v = qkv.split([HEADS, KV, KV], dim=2)
    return q, k, v, *norm_rotary(q, k, positions, axes, head_weight, head_weight, 1e-6)


def finish(x, o, w):
    s, z = _layers_hip.rms_norm(x, w['n2'], 1e-6, residual=F.linear(o.flatten(2), w['out']))
    return s + F.linear(F.gelu(F.linear(z, w['up'])), w['down'])


def inputs(device, dtype, n, seed, batch=1):
    return torch.randn((batch, n, WIDTH), generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


@pytest.mark.parametrize('dtype', DTYPES)
def test_two_blocks_of_a_clip(device, dtype):
    pos, order, tokens = clip(device)
    axes = RotaryAxes(DIM, SECTIONS, base=100.0, shared=True, device=device)
    hw = 1 + 0.1 * torch.randn(DIM, generator=torch.Generator().manual_seed(1)).to(device)
    x = inputs(device, dtype, len(pos), 2)
    for seed in (3, 4):
        w = weights(device, dtype, seed)
        q, k, v, qr, kr = heads_of(x, w, pos.to(device), axes, hw)
        check_heads(qr, q, hw, 1e-6, pos, SECTIONS, 100.0, True, False)
        check_heads(kr, k, hw, 1e-6, pos, SECTIONS, 100.0, True, False)
        o = masked_attention(qr, kr, v, DIM ** -0.5, keys=tokens, window=3, sinks=1)
        check_attention(o, qr, kr, v, DIM ** -0.5, seen=see(order * 0, order * 0, order, order, 3, 1))
        x = finish(x, o, w)


@pytest.mark.parametrize('dtype', DTYPES)
def test_new_tokens_over_a_cache_give_what_the_whole_sequence_gives(device, dtype):
    # both are within their tolerance of float64 on the same keys and queries
    t, window, sinks = 70, 12, 2
    axes = RotaryAxes(DIM, (32,), base=1e4, device=device)
    w, x = weights(device, dtype, 5), inputs(device, dtype, 70, 6)
    at = torch.arange(t)
    pos = at.float()[:, None].to(device)
    side = Tokens(i32(at * 0, device), i32(at, device))
    _, _, v, qr, kr = heads_of(x, w, pos, axes, None)
    whole = masked_attention(qr, kr, v, DIM ** -0.5, keys=side, window=window, sinks=sinks)
    check_attention(whole, qr, kr, v, DIM ** -0.5, seen=see(at * 0, at * 0, at, at, window, sinks))
    cache_k, cache_v = torch.full_like(kr, float('nan')), torch.full_like(v, float('inf'))   # never written
    for i in range(t):
        step = slice(i, i + 1)
        cache_k[:, step], cache_v[:, step] = kr[:, step], v[:, step]
        last = i32(at[step], device)
        o = masked_attention(qr[:, step], cache_k, cache_v, DIM ** -0.5, keys=side, window=window, sinks=sinks,
                             queries=Tokens(torch.zeros_like(last), last, queries_only=True))
        check_attention(o, qr[:, step], kr, v, DIM ** -0.5, seen=see(at[step] * 0, at * 0, at[step], at, window, sinks))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('batch,n', [(3, 37), (2, 150)])
def test_images_beside_reference_images(device, batch, n, dtype):
    axes = RotaryAxes(DIM, (16, 16), base=100.0, device=device)
    grid = lambda m: torch.stack([torch.arange(m) // 7, torch.arange(m) % 7], -1).float()  # noqa: E731
    w, refs, x = weights(device, dtype, 7), inputs(device, dtype, 90, 8), inputs(device, dtype, n, 9, batch)
    _, _, pv, _, pk = heads_of(refs, w, grid(90).to(device), axes, None)
    _, _, v, q, k = heads_of(x, w, grid(n).to(device), axes, None)
    o = prefix_attention(q, k, v, pk[0], pv[0], DIM ** -0.5)
    check_prefix(o, q, k, v, pk[0], pv[0], DIM ** -0.5)
    finish(x, o, w)


def test_captured_step_beside_another_graph(device):
    # two graphs of the same calls, replayed in turn: each has its own workspaces
    dtype, batch, cache, p = torch.bfloat16, 5, 300, 400
    axes, w = RotaryAxes(DIM, (32,), base=1e4, device=device), weights(device, torch.bfloat16, 10)
    hw = torch.ones(DIM, device=device)
    at = torch.arange(cache)
    keys = Tokens(i32(at * 0, device), i32(at, device))
    g = torch.Generator().manual_seed(11)
    ck, cv = (torch.randn((batch, cache, KV, DIM), generator=g).to(dtype).to(device) for _ in range(2))
    pk, pv = (torch.randn((p, KV, DIM), generator=g).to(dtype).to(device) for _ in range(2))

    def program(x, last, queries):
        _, _, _, q, k = heads_of(x, w, last, axes, hw)
        a = masked_attention(q, ck, cv, 0.125, keys=keys, queries=queries, window=100, sinks=4)
        return finish(x, a, w), prefix_attention(q, ck, cv, pk, pv, 0.125, keys=keys, queries=queries)

    made = []
    for seed in (12, 13):
        x = inputs(device, dtype, 1, seed, batch)
        last = i32(torch.randint(0, 200, (batch, 1), generator=g), device)
        queries = Tokens(torch.zeros_like(last), last, queries_only=True)
        program(x, last[..., None], queries)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = program(x, last[..., None], queries)
        made.append((x, last, queries, graph, kept))
    for turn in range(3):
        for n, (x, last, queries, graph, kept) in enumerate(made):
            x.copy_(inputs(device, dtype, 1, 20 + 2 * turn + n, batch))
            last.add_(13 + n)
        for x, last, queries, graph, kept in made:
            graph.replay()
        for x, last, queries, graph, kept in made:
            eager = program(x, last[..., None], queries)
            torch.cuda.synchronize()
            assert torch.equal(kept[0], eager[0]) and torch.equal(kept[1], eager[1])


def test_threads_on_separate_streams_match_sequential(device):
    g = torch.Generator().manual_seed(14)
    make = lambda *s: torch.randn(s, generator=g).half().to(device)  # noqa: E731
    q, k, v, pk, pv = make(6, 1, 8, 64), make(6, 5000, 2, 64), make(6, 5000, 2, 64), make(3000, 2, 64), make(3000, 2, 64)
    at = torch.arange(5000)
    keys = Tokens(i32(at * 0, device), i32(at, device))
    last = i32(torch.randint(0, 5000, (6, 1), generator=g), device)
    queries = Tokens(torch.zeros_like(last), last, queries_only=True)
    axes = RotaryAxes(64, (32,), device=device)

    def work():
        qr = norm_rotary(q, None, last[..., None], axes)
        return (qr, masked_attention(qr, k, v, 0.125, keys=keys, queries=queries, window=4000, sinks=4),
                prefix_attention(qr, k, v, pk, pv, 0.125, keys=keys, queries=queries))

    want = work()
    torch.cuda.synchronize()
    got = [None] * 4

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(5):
                got[i] = work()
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for result in got:
        assert all(torch.equal(a, b) for a, b in zip(result, want))
