"""What the C entry points of the norms, the rotary positions and the masked attention refuse,
before any launch (CPU only): every call here returns its error code without touching a GPU."""
import ctypes

import pytest

OK, INVALID, WORKSPACE, UNSUPPORTED = 0, 1001, 1002, 1003
P = ctypes.c_void_p(4096)      # never dereferenced: validation fails first


@pytest.fixture(scope='module')
def lib():
    from musc_hip import _runtime
    return _runtime.library()


def norm_args(**kw):
    a = dict(x=P, xs=64, r=None, rs=0, s=None, w=P, wd=0, dt=1, rows=4, width=64, eps=1e-6, y=P, stream=None)
    a.update(kw)
    return list(a.values())


def eight_args(**kw):
    a = dict(x=P, xs=64, r=None, rs=0, s=None, w=P, wd=0, dt=1, rows=4, width=64, eps=1e-6, fmt=0, group=0, y=P, sc=P,
             stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize('change,code', [
    (dict(x=None), INVALID), (dict(y=None), INVALID), (dict(rows=-1), INVALID), (dict(width=0), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float('nan')), INVALID), (dict(dt=3), INVALID), (dict(wd=2), INVALID),
    (dict(r=P, rs=64), INVALID), (dict(xs=63), INVALID), (dict(r=P, rs=63, s=P), INVALID),
    (dict(x=ctypes.c_void_p(4097)), INVALID), (dict(w=ctypes.c_void_p(4098)), INVALID),
    (dict(width=32769, xs=32769), UNSUPPORTED), (dict(dt=0, width=16385, xs=16385), UNSUPPORTED), (dict(rows=0), OK)])
def test_rmsnorm(lib, change, code):
    assert lib.musc_rmsnorm_rows(*norm_args(**change)) == code
    assert lib.musc_rmsnorm_rows_8bit(*eight_args(**change)) == code


@pytest.mark.parametrize('change,code', [
    (dict(fmt=2), INVALID), (dict(sc=None), INVALID), (dict(group=-32), INVALID), (dict(group=48), UNSUPPORTED),
    (dict(group=128), INVALID), (dict(sc=ctypes.c_void_p(4098)), INVALID)])
def test_rmsnorm_eight_bits(lib, change, code):
    assert lib.musc_rmsnorm_rows_8bit(*eight_args(**change)) == code


def rotary_args(**kw):
    a = dict(q=P, qh=2, qsb=512, qst=128, qsh=64, qo=P, qob=512, qot=128, qoh=64, k=None, kh=0, ksb=0, kst=0, ksh=0,
             ko=None, kob=0, kot=0, koh=0, dt=0, batch=1, t=4, d=64, pos=P, ints=0, psb=0, axes=2, freq=P, axis=P, pairs=32,
             adjacent=0, inverse=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize('change,code', [
    (dict(q=None), INVALID), (dict(qo=None), INVALID), (dict(pos=None), INVALID), (dict(freq=None), INVALID),
    (dict(axis=None), INVALID), (dict(pairs=33), INVALID), (dict(pairs=0), INVALID), (dict(axes=0), INVALID),
    (dict(qh=0), INVALID), (dict(kh=1), INVALID), (dict(qst=-1), INVALID), (dict(dt=3), INVALID), (dict(psb=-1), INVALID),
    (dict(q=ctypes.c_void_p(4098)), INVALID), (dict(freq=ctypes.c_void_p(4100)), INVALID),
    (dict(d=520), UNSUPPORTED), (dict(qh=1025), UNSUPPORTED), (dict(batch=65536, t=65536), UNSUPPORTED),
    (dict(d=512, pairs=256, t=0), OK), (dict(batch=0), OK)])
def test_rotary(lib, change, code):
    assert lib.musc_rotary(*rotary_args(**change)) == code
