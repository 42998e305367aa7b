"""The objects that a model keeps for its packed encoder, copied and pickled with it, and strides that no
memory has (CPU only)."""
import copy
import ctypes
import pickle

import pytest
import torch

from musc_hip import _runtime
from musc_hip._masked_attention_hip import Tokens
from musc_hip._rotary_hip import RotaryAxes


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(_runtime, 'require_device_tensor', lambda t, name: None)
    monkeypatch.setattr(_runtime, 'current_stream', lambda index: 0)
    monkeypatch.setattr(Tokens, 'refresh', lambda self: None)


def numbers(x):
    """Whole numbers that an object holds, at any depth."""
    if isinstance(x, dict):
        return [n for v in x.values() for n in numbers(v)]
    if isinstance(x, (tuple, list)):
        return [n for v in x for n in numbers(v)]
    return [x] if isinstance(x, int) else []


def storages(x):
    return [(t.untyped_storage().data_ptr(), t.untyped_storage().nbytes()) for t in vars(x).values() if isinstance(t, torch.Tensor)]


def make_axes():
    return RotaryAxes(64, (16, 16), device='cpu')


def make_tokens():
    docs = torch.zeros((2, 300), dtype=torch.int32)
    return Tokens(docs, torch.zeros_like(docs), torch.zeros((2, 300, 2)))


@pytest.mark.parametrize('copied', [copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
@pytest.mark.parametrize('make', [make_axes, make_tokens])
def test_copies_hold_no_address_of_the_original(on_cpu, make, copied):
    # a copied model may outlive the first one, or be in another process
    was = make()
    other = copied(was)
    held = numbers(vars(other))
    for first, size in storages(was):
        assert not [n for n in held if first <= n < first + size]
    for name, x in vars(was).items():
        if isinstance(x, torch.Tensor):
            assert getattr(other, name).data_ptr() != x.data_ptr() and getattr(other, name).shape == x.shape


@pytest.mark.parametrize('side', ['k_st', 'v_st'])
@pytest.mark.parametrize('stride', [1 << 28, 1 << 58, 1 << 60, (1 << 63) - 64])
def test_row_strides_past_any_tile_are_refused(side, stride):
    # 63 rows of 2^58 elements wrap around 64 bits
    from test_operator_refusals import UNSUPPORTED, attention_call
    need = ctypes.c_size_t()
    call = ctypes.byref(attention_call(**{side: stride}))
    assert _runtime.library().musc_masked_attention_workspace_bytes(call, ctypes.byref(need)) == UNSUPPORTED
