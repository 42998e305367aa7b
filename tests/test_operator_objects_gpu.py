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
