"""Copies of Tokens and RotaryAxes that outlive what they were copied from."""
import copy

import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, masked_attention
from musc_hip._rotary_hip import RotaryAxes, rotary

pytestmark = pytest.mark.gpu


def test_copies_outlive_the_original(device):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn((1, 900, 2, 64), generator=g).half().to(device) for _ in range(3))
    docs = torch.arange(3, dtype=torch.int32).repeat_interleave(300).to(device)
    pos = torch.arange(1800).float().view(900, 2).to(device)
    tokens, axes = Tokens(docs), RotaryAxes(64, (16, 16), device=device)
    want = (*rotary(q, k, pos, axes), masked_attention(q, k, v, 0.125, keys=tokens))
    tokens2, axes2 = copy.deepcopy(tokens), copy.deepcopy(axes)
    del tokens, axes
    filler = [torch.full((n,), 0x7f7f7f7f, dtype=torch.int32, device=device) for n in (128, 128, 256, 1024, 4096) * 4]
    got = (*rotary(q, k, pos, axes2), masked_attention(q, k, v, 0.125, keys=tokens2))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert filler


def test_tokens_dropped_while_another_stream_works_with_them(device):
    g = torch.Generator().manual_seed(2)
    t = 1500
    q, k, v = (torch.randn((1, t, 2, 64), generator=g).half().to(device) for _ in range(3))
    ids = torch.arange(t, dtype=torch.int32) // 400
    docs = ids.to(device)
    want = masked_attention(q, k, v, 0.125, keys=Tokens(docs))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        masked_attention(q, k, v, 0.125, keys=Tokens(docs))            # what a first call on a stream sets up
    torch.cuda.synchronize()
    tokens = Tokens(ids.to(device))
    sizes = [x.numel() for x in (tokens.summary, tokens._schedule, tokens.documents)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)                                   # tens of milliseconds
        got = masked_attention(q, k, v, 0.125, keys=tokens)
    del tokens
    filler = [torch.zeros((n,), dtype=torch.int32, device=device) for n in sizes * 8]
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert filler
