"""Caps far above the scores: cap tanh(s / cap) is then s, to fp32's precision of s itself.

The tolerance is test_masked_attention_gpu's with the cap's share taken from the capped score instead
of the cap: scale / cap, the product and the factor back are rounded four times, tanh is within two
units in the last place (four halves): 8 2^-24 |s|.  Scores here are about 2, caps up to 2^60."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention

from test_masked_attention_gpu import U, heads, i32, see

pytestmark = pytest.mark.gpu

CAPS = [129.0, 1e3, 1e5, 1e8, 2.0 ** 60]


def check(got, q, k, v, scale, cap, seen=None, slopes=None, pos=None):
    """Self-attention or one side of it, positions (T, 1) of queries and keys."""
    dtype = q.dtype
    q, k, v = (x.double().cpu().transpose(1, 2) for x in (q, k, v))
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = cap * torch.tanh(q @ k.transpose(2, 3) * scale / cap)
    d = (q.shape[3] + 8) * (q.abs() @ k.abs().transpose(2, 3)) * abs(scale) + 8 * s.abs() + 4
    if slopes is not None:
        bias = (pos[0].double()[:, None] - pos[1].double()[None]).abs().sum(-1) * slopes.double()[:, :1, None]
        s, d = s - bias, d + 6 * bias.abs()
    if seen is not None:
        s = s.masked_fill(~seen[:, None], -torch.inf)
    p = torch.softmax(s, -1)
    out, w = p @ v, p @ v.abs()
    d = d * U + 2.0 ** -22
    tol = (p * d) @ v.abs() + (p * d).sum(-1, keepdim=True) * out.abs() + 2 * s.shape[-1] * U * w
    half = torch.finfo(dtype).eps / 2
    if dtype != torch.float32:
        tol = tol + half * w
    if dtype == torch.float16:
        tol = tol + s.shape[-1] * 2.0 ** -32 * v.abs().amax() + 2.0 ** -25
    tol = tol + half * (out.abs() + tol)
    got = got.double().cpu().transpose(1, 2)
    assert torch.isfinite(got).all()
    assert ((got - out).abs() <= tol).all(), ((got - out).abs() / tol).max().item()


@pytest.mark.parametrize('cap', CAPS)
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('tq,tk,h,hk,d', [
    (1, 300, 2, 2, 64), (3, 70, 8, 2, 128),           # few rows in one workgroup
    (1, 5000, 4, 2, 64), (2, 5000, 2, 2, 128),        # few rows over long keys
    (300, 300, 2, 2, 64), (150, 260, 2, 1, 96), (129, 200, 4, 2, 128)])
def test_every_key(device, tq, tk, h, hk, d, dtype, cap):
    q, k, v = heads(device, dtype, 1, tq, tk, h, hk, d, size=2 ** 0.5)
    scale = d ** -0.5
    check(masked_attention(q, k, v, scale, cap=cap), q, k, v, scale, cap)
    check(masked_attention(q, k, v, -scale, cap=cap), q, k, v, -scale, cap)
    pos = torch.arange(tq).float()[:, None] + 0.5, torch.arange(tk).float()[:, None]
    slopes = torch.tensor([[0.01 * 2.0 ** -i] for i in range(h)])
    got = masked_attention(q, k, v, scale, keys=Tokens(positions=pos[1].to(device)),
                           queries=Tokens(positions=pos[0].to(device)), cap=cap, slopes=slopes.to(device))
    check(got, q, k, v, scale, cap, slopes=slopes, pos=pos)


@pytest.mark.parametrize('cap', [1e3, 1e8])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('d', [64, 128])
def test_documents_and_orders(device, d, dtype, cap):
    sizes = [700, 150, 1000, 350]
    docs = torch.repeat_interleave(torch.arange(4), torch.tensor(sizes))
    t, order = len(docs), torch.arange(2200)
    q, k, v = heads(device, dtype, 1, t, t, 2, 2, d, size=2 ** 0.5)
    rows = torch.randperm(t, generator=torch.Generator().manual_seed(1))[:300]
    for given in (None, order):                       # row tiles in pieces; in parts
        got = masked_attention(q, k, v, d ** -0.5, cap=cap, keys=Tokens(i32(docs, device), None if given is None else i32(given, device)))
        seen = see(docs[rows], docs) if given is None else see(docs[rows], docs, order[rows], order)
        check(got[:, rows], q[:, rows], k, v, d ** -0.5, cap, seen=seen)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
def test_scores_about_a_large_cap(device, dtype):
    q, k, v = heads(device, dtype, 1, 200, 200, 2, 2, 64, size=8.0)   # scores of about 500
    check(masked_attention(q, k, v, 1.0, cap=1000.0), q, k, v, 1.0, 1000.0)
    check(masked_attention(q, k, v, 16.0, cap=1000.0), q, k, v, 16.0, 1000.0)
