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


def rotary_call(**kw):
    from musc_hip import _runtime as rt
    c = rt.RotaryCall()
    c.q = c.q_out = c.positions = c.frequency = c.axis = 4096
    c.q_sb, c.q_st, c.q_sh, c.q_ob, c.q_ot, c.q_oh = 512, 128, 64, 512, 128, 64
    c.q_heads, c.batch, c.t, c.d, c.axes, c.pairs = 2, 1, 4, 64, 2, 32
    for name, value in kw.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize('change,code', [
    (dict(q=0), INVALID), (dict(q_out=0), INVALID), (dict(positions=0), INVALID), (dict(frequency=0), INVALID),
    (dict(axis=0), INVALID), (dict(pairs=33), INVALID), (dict(pairs=0), INVALID), (dict(axes=0), INVALID),
    (dict(q_heads=0), INVALID), (dict(k_heads=1), INVALID), (dict(q_st=-1), INVALID), (dict(dtype=3), INVALID),
    (dict(pos_sb=-1), INVALID), (dict(q=4098), INVALID), (dict(frequency=4100), INVALID),
    (dict(d=520), UNSUPPORTED), (dict(q_heads=1025), UNSUPPORTED), (dict(batch=65536, t=65536), UNSUPPORTED),
    (dict(d=512, pairs=256, t=0), OK), (dict(batch=0), OK)])
def test_rotary(lib, change, code):
    assert lib.musc_rotary(ctypes.byref(rotary_call(**change)), None) == code
    assert lib.musc_rotary(None, None) == INVALID


def attention_call(**kw):
    from musc_hip import _runtime as rt
    c = rt.MaskedAttention()
    for x in 'qkv':
        setattr(c, x, 4096)
        for s, n in (('sb', 64 * 64 * 2), ('st', 128), ('sh', 64)):
            setattr(c, f'{x}_{s}', n)
    c.out, c.o_sb, c.o_st, c.o_sh = 4096, 64 * 64 * 2, 128, 64
    c.dtype, c.batch, c.q_len, c.k_len, c.heads, c.kv_heads, c.d, c.scale = 1, 2, 64, 64, 2, 2, 64, 0.125
    for name, value in kw.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize('change,code', [
    (dict(q=0), INVALID), (dict(out=0), INVALID), (dict(dtype=3), INVALID), (dict(batch=0), INVALID),
    (dict(q_len=0), INVALID), (dict(k_len=0), INVALID), (dict(heads=3), INVALID), (dict(kv_heads=0), INVALID),
    (dict(d=136), UNSUPPORTED), (dict(d=60), UNSUPPORTED), (dict(dtype=0, d=66), UNSUPPORTED), (dict(q=4104), INVALID),
    (dict(k_st=130), INVALID), (dict(v_sh=-64), INVALID), (dict(o_st=4), INVALID), (dict(k_st=1 << 28), UNSUPPORTED),
    (dict(cap=-1.0), INVALID), (dict(cap=float('nan')), INVALID), (dict(scale=float('inf')), INVALID),
    (dict(q_documents=4096), INVALID), (dict(q_documents=4096, k_documents=4096), INVALID),
    (dict(q_documents=4096, k_documents=4096, k_summary=4100), INVALID),
    (dict(q_order=4096, k_order=4096), INVALID), (dict(q_documents=4098, k_documents=4096, k_summary=4096), INVALID),
    (dict(q_documents=4096, k_documents=4096, k_summary=4096, q_order=4096), INVALID),
    (dict(axes=4), UNSUPPORTED), (dict(axes=1), INVALID), (dict(axes=1, q_positions=4096, k_positions=4096), INVALID),
    (dict(q_tokens_sb=-1), INVALID), (dict(schedule=4098), INVALID), (dict(schedule_sb=-2), INVALID), (dict(batch=1 << 20, kv_heads=2, q_len=1 << 20), UNSUPPORTED)])
def test_masked_attention(lib, change, code):
    need = ctypes.c_size_t()
    call = ctypes.byref(attention_call(**change))
    assert lib.musc_masked_attention_workspace_bytes(call, ctypes.byref(need)) == code
    assert lib.musc_masked_attention_fwd(call, None, ctypes.c_size_t(0), None) == code


def test_masked_attention_workspace(lib):
    need = ctypes.c_size_t(1)
    assert lib.musc_masked_attention_workspace_bytes(None, ctypes.byref(need)) == INVALID
    assert lib.musc_masked_attention_workspace_bytes(ctypes.byref(attention_call()), None) == INVALID
    # a full grid is not split; one row over many keys is, and refuses to run without its parts
    assert lib.musc_masked_attention_workspace_bytes(ctypes.byref(attention_call(batch=64, q_len=1024)), ctypes.byref(need)) == OK
    assert need.value == 0
    one = ctypes.byref(attention_call(q_len=1, k_len=4096))
    assert lib.musc_masked_attention_workspace_bytes(one, ctypes.byref(need)) == OK and need.value > 0
    assert lib.musc_masked_attention_fwd(one, None, need, None) == WORKSPACE
    assert lib.musc_masked_attention_fwd(one, P, ctypes.c_size_t(need.value - 1), None) == WORKSPACE
    assert lib.musc_masked_attention_fwd(one, ctypes.c_void_p(4100), need, None) == WORKSPACE


def test_packed_calls_are_the_structures(lib):
    from musc_hip import _runtime as rt
    values = list(range(1, 24)) + [0.5, 2.0] + list(range(26, 42))
    packed = rt.MaskedAttention.from_buffer_copy(rt.PACK_MASKED_ATTENTION.pack(*values))
    assert [getattr(packed, name) for name, _ in rt.MaskedAttention._fields_] == values
    values = list(range(1, 32))
    packed = rt.RotaryCall.from_buffer_copy(rt.PACK_ROTARY.pack(*values))
    assert [getattr(packed, name) for name, _ in rt.RotaryCall._fields_] == values


@pytest.mark.parametrize('args,code', [
    ((None, None, 1, 64, P, None), INVALID), ((P, None, 1, 64, None, None), INVALID), ((P, P, -1, 64, P, None), INVALID),
    ((ctypes.c_void_p(4098), None, 1, 64, P, None), INVALID), ((P, None, 1, 64, ctypes.c_void_p(4104), None), INVALID),
    ((P, None, 0, 64, P, None), OK), ((P, None, 1 << 16, 1 << 16, P, None), UNSUPPORTED)])
def test_token_summary(lib, args, code):
    assert lib.musc_token_summary(*args) == code


@pytest.mark.parametrize('change,code', [
    (dict(documents=None), INVALID), (dict(summary=None), INVALID), (dict(schedule=None), INVALID), (dict(schedule=ctypes.c_void_p(4098)), INVALID),
    (dict(batch=-1), INVALID), (dict(t=-1), INVALID), (dict(summary=ctypes.c_void_p(4104)), INVALID),
    (dict(order=ctypes.c_void_p(4098)), INVALID), (dict(batch=0), OK), (dict(t=0), OK),
    (dict(batch=1 << 14, t=1 << 14), UNSUPPORTED), (dict(t=16385), UNSUPPORTED)])
def test_token_schedule(lib, change, code):
    a = dict(documents=P, order=None, summary=P, batch=1, t=64, schedule=P, stream=None)
    a.update(change)
    assert lib.musc_token_schedule(*a.values()) == code
