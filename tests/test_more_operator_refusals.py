"""What the C entry points of head norms, windows and shared prefixes refuse, before any launch (CPU only):
every call here returns its error code without touching a GPU."""
import ctypes

import pytest

from test_operator_refusals import INVALID, OK, UNSUPPORTED, P, lib, rotary_call  # noqa: F401


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
