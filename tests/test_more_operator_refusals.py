"""What the C entry points of head norms, windows and shared prefixes refuse, before any launch (CPU only):
every call here returns its error code without touching a GPU."""
import ctypes

import pytest

from test_operator_refusals import INVALID, OK, UNSUPPORTED, WORKSPACE, P, attention_call, lib, rotary_call  # noqa: F401


def normed(lib, call, **kw):  # noqa: F811
    a = dict(qw=P, q_sh=0, q_type=0, kw=None, k_sh=0, k_type=0, eps=1e-6, stream=None)
    a.update(kw)
    return lib.musc_norm_rotary(call, *a.values())


@pytest.mark.parametrize('change,code', [
    (dict(q=0), INVALID), (dict(q_out=0), INVALID), (dict(positions=0), INVALID), (dict(pairs=33), INVALID),
    (dict(k_heads=1), INVALID), (dict(dtype=3), INVALID), (dict(q_st=-1), INVALID), (dict(q=4098), INVALID),
    (dict(d=520), UNSUPPORTED), (dict(q_heads=1025), UNSUPPORTED), (dict(t=0), OK), (dict(batch=0), OK)])
def test_norm_rotary_calls(lib, change, code):  # noqa: F811
    assert normed(lib, ctypes.byref(rotary_call(**change))) == code
    assert normed(lib, None) == INVALID


@pytest.mark.parametrize('change,code', [
    (dict(eps=-1.0), INVALID), (dict(eps=float('nan')), INVALID), (dict(q_type=1), INVALID), (dict(q_type=3), INVALID),
    (dict(qw=ctypes.c_void_p(4098)), INVALID), (dict(q_sh=-64), INVALID), (dict(qw=None, q_type=3), OK),
    (dict(kw=ctypes.c_void_p(4097), k_type=3), OK), (dict(q_sh=64), OK)])
def test_norm_rotary_weights(lib, change, code):  # noqa: F811
    # no tokens: what is not refused returns without a launch; k's weight is not looked at without k
    assert normed(lib, ctypes.byref(rotary_call(t=0)), **change) == code


def windowed(lib, call, window=4, sinks=0, workspace=None, size=0):  # noqa: F811
    need = ctypes.c_size_t()
    code = lib.musc_window_attention_workspace_bytes(call, window, sinks, ctypes.byref(need))
    assert lib.musc_window_attention_fwd(call, window, sinks, workspace, ctypes.c_size_t(size), None) == code
    return code


ORDERED = dict(q_documents=4096, k_documents=4096, k_summary=4096, q_order=4096, k_order=4096)


@pytest.mark.parametrize('change,code', [
    (dict(q=0), INVALID), (dict(v=0), INVALID), (dict(k_len=0), INVALID), (dict(dtype=3), INVALID), (dict(heads=3), INVALID), (dict(d=136), UNSUPPORTED),
    (dict(k_st=1 << 28), UNSUPPORTED), (dict(q_order=0), INVALID), (dict(q_order=0, k_order=0), INVALID), (dict(k_order=0), INVALID),
    (dict(cap=float('nan')), INVALID), (dict(batch=1 << 20, kv_heads=2, q_len=1 << 20), UNSUPPORTED)])
def test_window_calls(lib, change, code):  # noqa: F811
    assert windowed(lib, ctypes.byref(attention_call(**{**ORDERED, **change}))) == code


@pytest.mark.parametrize('window,sinks', [(0, 0), (-1, 0), (4, -1), (-(1 << 31), 4)])
def test_windows(lib, window, sinks):  # noqa: F811
    assert windowed(lib, ctypes.byref(attention_call(**ORDERED)), window, sinks) == INVALID
    assert windowed(lib, None) == INVALID
    assert lib.musc_window_attention_workspace_bytes(ctypes.byref(attention_call(**ORDERED)), 4, 0, None) == INVALID


def test_window_workspace(lib):  # noqa: F811
    need = ctypes.c_size_t(1)
    one = ctypes.byref(attention_call(q_len=1, k_len=1 << 15, **ORDERED))
    assert lib.musc_window_attention_workspace_bytes(one, 100, 4, ctypes.byref(need)) == OK and need.value > 0
    for workspace, size in ((None, need.value), (P, need.value - 1), (ctypes.c_void_p(4100), need.value)):
        assert lib.musc_window_attention_fwd(one, 100, 4, workspace, ctypes.c_size_t(size), None) == WORKSPACE


def prefix_of(**kw):
    from musc_hip import _runtime as rt
    p = rt.AttentionPrefix()
    p.k = p.v = 4096
    p.k_st, p.k_sh, p.v_st, p.v_sh, p.len = 128, 64, 128, 64, 100
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def prefixed(lib, call, prefix):  # noqa: F811
    need = ctypes.c_size_t()
    code = lib.musc_prefix_attention_workspace_bytes(call, prefix, ctypes.byref(need))
    assert lib.musc_prefix_attention_fwd(call, prefix, None, ctypes.c_size_t(0), None) == code
    return code


@pytest.mark.parametrize('change,code', [
    (dict(q=0), INVALID), (dict(k=0), INVALID), (dict(k_len=-1), INVALID), (dict(dtype=3), INVALID), (dict(batch=0), INVALID), (dict(heads=3), INVALID), (dict(d=136), UNSUPPORTED),
    (dict(v_st=1 << 28), UNSUPPORTED), (dict(q_documents=4096), INVALID), (dict(axes=1, q_positions=4096, k_positions=4096, slopes=4096), INVALID),
    (dict(axes=4), UNSUPPORTED), (dict(batch=1 << 20, kv_heads=2, q_len=1 << 20), UNSUPPORTED),
    (dict(k_len=0, k=0, v=0, q_order=4096), INVALID), (dict(k_len=0, k=0, v=0, axes=1, slopes=4096), INVALID)])
def test_prefix_calls(lib, change, code):  # noqa: F811
    assert prefixed(lib, ctypes.byref(attention_call(**change)), ctypes.byref(prefix_of())) == code
    assert prefixed(lib, None, ctypes.byref(prefix_of())) == INVALID


@pytest.mark.parametrize('change,code', [
    (dict(k=0), INVALID), (dict(v=0), INVALID), (dict(len=0), INVALID), (dict(len=-5), INVALID), (dict(k=4104), INVALID),
    (dict(k_st=130), INVALID), (dict(v_sh=-64), INVALID), (dict(k_st=1 << 28), UNSUPPORTED), (dict(v_st=1 << 61), UNSUPPORTED)])
def test_prefixes(lib, change, code):  # noqa: F811
    assert prefixed(lib, ctypes.byref(attention_call()), ctypes.byref(prefix_of(**change))) == code
    assert prefixed(lib, ctypes.byref(attention_call()), None) == INVALID


def test_prefix_workspace(lib):  # noqa: F811
    need = ctypes.c_size_t(1)
    prefix = ctypes.byref(prefix_of())
    full = ctypes.byref(attention_call(batch=64, q_len=1024))
    assert lib.musc_prefix_attention_workspace_bytes(full, prefix, ctypes.byref(need)) == OK and need.value == 0
    # few rows over few keys are joined by their workgroup; over many, and stacked ones, by a kernel
    assert lib.musc_prefix_attention_workspace_bytes(ctypes.byref(attention_call(q_len=1)), prefix, ctypes.byref(need)) == OK
    assert need.value == 0
    prefix = ctypes.byref(prefix_of(len=1 << 15))
    for change in (dict(q_len=1), dict(q_len=1, k_len=0, k=0, v=0), dict(q_len=40, batch=9), dict(q_len=1, batch=1)):
        call = ctypes.byref(attention_call(**change))
        assert lib.musc_prefix_attention_workspace_bytes(call, prefix, ctypes.byref(need)) == OK and need.value > 0
        for workspace, size in ((None, need.value), (P, need.value - 1), (ctypes.c_void_p(4100), need.value)):
            assert lib.musc_prefix_attention_fwd(call, prefix, workspace, ctypes.c_size_t(size), None) == WORKSPACE
    assert lib.musc_prefix_attention_workspace_bytes(full, prefix, None) == INVALID


def test_packed_prefixes_are_the_structure():
    from musc_hip import _runtime as rt
    packed = rt.AttentionPrefix.from_buffer_copy(rt.PACK_ATTENTION_PREFIX.pack(*range(1, 9)))
    assert [getattr(packed, name) for name, _ in rt.AttentionPrefix._fields_] == list(range(1, 9))
