"""Whether the rows of all entries pass over a shared prefix together, as the workspace tells (CPU only)."""
import ctypes

import pytest

from test_more_operator_refusals import prefix_of
from test_operator_refusals import OK, attention_call, lib  # noqa: F401


def workspace(lib, length, **call):  # noqa: F811
    need = ctypes.c_size_t()
    prefix, call = prefix_of(len=length), attention_call(**call)
    assert lib.musc_prefix_attention_workspace_bytes(ctypes.byref(call), ctypes.byref(prefix), ctypes.byref(need)) == OK
    return need.value


@pytest.mark.parametrize('dtype', [0, 1, 2])
@pytest.mark.parametrize('batch,q_len', [(1024, 40), (4096, 8), (512, 80)])
@pytest.mark.parametrize('length', [1, 64])
def test_short_prefixes_are_taken_entry_by_entry(lib, length, batch, q_len, dtype):  # noqa: F811
    # as each entry alone: no parts of its outputs are written
    assert workspace(lib, length, dtype=dtype, batch=batch, q_len=q_len, heads=16, kv_heads=16, d=64) == 0


@pytest.mark.parametrize('dtype', [0, 1, 2])
def test_long_prefixes_are_read_once(lib, dtype):  # noqa: F811
    # both parts of every row, in fp32: more than one of each would say
    rows = 512 * 4 * 8
    need = workspace(lib, 16384, dtype=dtype, batch=512, q_len=1, heads=32, kv_heads=8, d=128, k_len=100)
    assert need >= 2 * rows * 128 * 4


@pytest.mark.parametrize('length', [256, 4096, 1 << 20, 1 << 30])
def test_parts_of_many_rows_stay_within_a_gib(lib, length):  # noqa: F811
    for batch, q_len in ((1 << 14, 40), (1 << 18, 3), (1 << 20, 1)):
        assert workspace(lib, length, batch=batch, q_len=q_len, heads=8, kv_heads=8, d=128) <= (1 << 30) + (1 << 24)
