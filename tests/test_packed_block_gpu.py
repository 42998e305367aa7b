"""The norms, rotary positions and masked attention as a packed encoder block uses them: images of
their own sizes in one sequence, through two pre-norm blocks, against the same in float64; and an
8-bit norm in front of a scaled product, captured whole.

Tolerance: every step is compared with the float64 step on the block's own stored input, so
nothing is carried from step to step: the linear maps are torch's."""
import pytest
import torch
from torch.nn import functional as F

from musc_hip import _layers_hip
from musc_hip._masked_attention_hip import Tokens, masked_attention
from musc_hip._rotary_hip import RotaryAxes, rotary

from test_masked_attention_gpu import check as check_attention
from test_masked_attention_gpu import see
from test_rmsnorm_gpu import check_eight, check_norm, check_sum
from test_rotary_gpu import check as check_rotary

pytestmark = pytest.mark.gpu

GRIDS = [(5, 9), (13, 4), (1, 1), (7, 7), (16, 11)]
HEADS, KV, DIM = 4, 2, 64
WIDTH = HEADS * DIM


def layout(device):
    docs = torch.cat([torch.full((h * w,), i) for i, (h, w) in enumerate(GRIDS)])
    pos = torch.cat([torch.stack(torch.meshgrid(torch.arange(h), torch.arange(w), indexing='ij'), -1).reshape(-1, 2)
                     for h, w in GRIDS]).float()
    return docs, pos.to(device), Tokens(docs.int().to(device), positions=pos.to(device))


def weights(device, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: (torch.randn(s, generator=g) * s[-1] ** -0.5).to(dtype).to(device)  # noqa: E731
    return dict(qkv=make((HEADS + 2 * KV) * DIM, WIDTH), out=make(WIDTH, WIDTH), up=make(2 * WIDTH, WIDTH),
                down=make(WIDTH, 2 * WIDTH), n1=1 + 0.1 * torch.randn(WIDTH, generator=g).to(device),
                n2=1 + 0.1 * torch.randn(WIDTH, generator=g).to(device))


def block(x, w, tokens, pos, axes, slopes, seen=None):
    y = _layers_hip.rms_norm(x, w['n1'], 1e-6)
    qkv = F.linear(y, w['qkv']).view(1, -1, HEADS + 2 * KV, DIM)
    q, k, v = qkv.split([HEADS, KV, KV], dim=2)
    qr, kr = rotary(q, k, pos, axes)
    o = masked_attention(qr, kr, v, DIM ** -0.5, keys=tokens, cap=20.0, slopes=slopes)
    a = F.linear(o.view(1, -1, WIDTH), w['out'])
    s, z = _layers_hip.rms_norm(x, w['n2'], 1e-6, residual=a)
    if seen is not None:
        check_norm(y, x, w['n1'])
        check_rotary(qr, q, pos.cpu(), (16, 16), 100.0, False, False)
        check_rotary(kr, k, pos.cpu(), (16, 16), 100.0, False, False)
        check_attention(o, qr, kr, v, DIM ** -0.5, seen=seen, cap=20.0, slopes=slopes, qpos=pos[None], kpos=pos[None])
        check_sum(s, x, a)
        check_norm(z, s, w['n2'])
    return s + F.linear(F.gelu(F.linear(z, w['up'])), w['down'])


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
def test_two_blocks_of_packed_images(device, dtype):
    docs, pos, tokens = layout(device)
    axes = RotaryAxes(DIM, (16, 16), base=100.0, device=device)
    slopes = torch.tensor([[0.5, 0.25], [0.1, 0.1], [0.02, 0.0], [0.0, 0.3]], device=device)
    x = torch.randn((1, len(docs), WIDTH), generator=torch.Generator().manual_seed(1)).to(dtype).to(device)
    for seed in (2, 3):
        x = block(x, weights(device, dtype, seed), tokens, pos, axes, slopes, seen=see(docs, docs))


def test_packing_does_not_change_an_image(device):
    # each image alone gives what it gives in the batch, up to the order of the sums
    docs, pos, tokens = layout(device)
    axes = RotaryAxes(DIM, (16, 16), base=100.0, device=device)
    slopes = torch.full((HEADS, 2), 0.1, device=device)
    w = weights(device, torch.float32, 5)
    x = torch.randn((1, len(docs), WIDTH), generator=torch.Generator().manual_seed(4)).to(device)
    whole = block(x, w, tokens, pos, axes, slopes)
    for i in range(len(GRIDS)):
        at = (docs == i).nonzero()[:, 0].to(device)
        alone = block(x[:, at].contiguous(), w, Tokens(positions=pos[at].contiguous()), pos[at].contiguous(), axes, slopes)
        # differing orders of at most 200 sums of numbers of order 1, through one block: 2e-5
        assert (whole[:, at] - alone).abs().max() <= 2e-5


def test_captured_block_replays_on_new_images(device):
    docs, pos, tokens = layout(device)
    axes = RotaryAxes(DIM, (16, 16), base=100.0, device=device)
    slopes = torch.full((HEADS, 2), 0.1, device=device)
    w = weights(device, torch.float16, 6)
    x = torch.randn((1, len(docs), WIDTH), generator=torch.Generator().manual_seed(7)).half().to(device)

    def step():
        tokens.refresh()
        out = block(x, w, tokens, pos, axes, slopes)
        return out, _layers_hip.rms_norm_quantized(out, w['n1'], 1e-6, group=64)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for turn in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 + turn)))
        tokens.documents.copy_(docs.roll(17 * turn).int())
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept[0], eager[0])
        assert torch.equal(kept[1][0].view(torch.uint8), eager[1][0].view(torch.uint8))
        assert torch.equal(kept[1][1], eager[1][1])
        check_eight(kept[1][0][0], kept[1][1][0], kept[0][0], w['n1'], 64, torch.float8_e4m3fn)
