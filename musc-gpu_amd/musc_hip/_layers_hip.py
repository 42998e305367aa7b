"""Fused encoder-block layers on MI355X (libmusc_hip musc_layernorm_rows, musc_rmsnorm_rows,
musc_rmsnorm_rows_8bit, musc_activation).

Reference: models/backbone/open_clip/transformer.py:23-29 (LayerNorm that casts back
to the input dtype), :32-35 (QuickGELU), :247-248 (residual adds around ln_2),
model.py:84-87 (QuickGELU for OpenAI weights, nn.GELU otherwise).  Each call is one
pass over the activations where torch's autocast path makes three (cast, normalise,
cast back; or 1.702 x, sigmoid, product).  The root-mean-square norms serve blocks
normalised that way; the reference has none.
"""
from __future__ import annotations

import torch

from . import _runtime as rt

_DTYPES = {torch.float32: rt.DTYPE_F32, torch.float16: rt.DTYPE_F16}


def _affine(p, width: int, device):
    if p is None:
        return None
    if p.numel() != width:
        raise ValueError('LayerNorm affine parameter does not match the row width')
    return p.detach().to(device=device, dtype=torch.float32).contiguous()


def layer_norm(x: torch.Tensor, weight, bias, eps: float, residual: torch.Tensor | None = None):
    """LayerNorm over the last dimension, fp32 statistics, output in x's dtype.

    With `residual`, returns (s, layer_norm(s)) where s = x + residual rounded to x's
    dtype (one pass for the residual add and the norm); otherwise layer_norm(x)."""
    rt.require_device_tensor(x, 'x')
    if x.dtype not in _DTYPES:
        raise ValueError('x must be float32 or float16')
    if residual is not None:
        rt.require_device_tensor(residual, 'residual')
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError('residual must match x in shape and dtype')
        residual = residual.contiguous()
    x = x.contiguous()
    width = x.shape[-1]
    rows = x.numel() // width if width else 0
    w, b = _affine(weight, width, x.device), _affine(bias, width, x.device)
    with torch.cuda.device(x.device):
        y = torch.empty_like(x)
        s = torch.empty_like(x) if residual is not None else None
        rc = rt.library().musc_layernorm_rows(
            x.data_ptr(), residual.data_ptr() if residual is not None else None,
            s.data_ptr() if s is not None else None, w.data_ptr() if w is not None else None,
            b.data_ptr() if b is not None else None, _DTYPES[x.dtype], rows, width, float(eps), y.data_ptr(),
            rt.stream(x.device))
        rt.check(rc, 'musc_layernorm_rows')
    return (s, y) if residual is not None else y


def supports_layer_norm(width: int, dtype: torch.dtype) -> bool:
    per = 8 if dtype == torch.float16 else 4
    return dtype in _DTYPES and width % per == 0 and (width // per + 63) // 64 <= 4


_STORAGE = {torch.float32: rt.DTYPE_F32, torch.float16: rt.DTYPE_F16, torch.bfloat16: rt.DTYPE_BF16}
_FP8 = {torch.float8_e4m3fn: rt.FP8_E4M3, torch.float8_e5m2: rt.FP8_E5M2}


def _rows(x: torch.Tensor, width: int):
    """(tensor, row stride) of x as rows of `width`; rows that no one stride reaches are copied."""
    if x.is_contiguous():
        return x, width
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= width:
        return x, x.stride(0)
    return x.contiguous(), width


def _rms(x, weight, eps, residual, dtype, group):
    rt.require_device_tensor(x, 'x')
    if rt.elsewhere(x):
        with torch.cuda.device(x.device):
            return _rms(x, weight, eps, residual, dtype, group)
    storage, index = _STORAGE.get(x.dtype), x.get_device()
    if storage is None or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('x must be a float32, float16 or bfloat16 tensor with at least one column')
    rt.require_no_gradient(x, weight, residual)
    width = x.shape[-1]
    rows = x.numel() // width
    if rows > 0x7fffffff:
        raise ValueError('x has more than 2^31 - 1 rows')
    w_ptr, w_dtype = None, rt.DTYPE_F32
    if weight is not None:
        rt.require_device_tensor(weight, 'weight')
        if weight.get_device() != index or weight.numel() != width or weight.dtype not in (x.dtype, torch.float32):
            raise ValueError("weight must be on x's device, one value per column, in x's dtype or float32")
        weight = weight.contiguous()
        w_ptr, w_dtype = weight.data_ptr(), _STORAGE[weight.dtype]
    x2, x_stride = _rows(x, width)
    s, r_ptr, r_stride, s_ptr = None, None, 0, None
    if residual is not None:
        rt.require_device_tensor(residual, 'residual')
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.get_device() != index:
            raise ValueError('residual must match x in shape, dtype and device')
        r2, r_stride = _rows(residual, width)
        s = torch.empty_like(x, memory_format=torch.contiguous_format)
        r_ptr, s_ptr = r2.data_ptr(), s.data_ptr()
    y = torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)
    if dtype is None:
        if rows:
            rt.check(rt.library().musc_rmsnorm_rows(x2.data_ptr(), x_stride, r_ptr, r_stride, s_ptr, w_ptr, w_dtype, storage,
                                                    rows, width, eps, y.data_ptr(), rt.current_stream(index)),
                     'musc_rmsnorm_rows')
        return y if s is None else (s, y)
    scales = torch.empty((*x.shape[:-1], width // group if group else 1), dtype=torch.float32, device=x.device)
    if rows:
        rt.check(rt.library().musc_rmsnorm_rows_8bit(x2.data_ptr(), x_stride, r_ptr, r_stride, s_ptr, w_ptr, w_dtype, storage,
                                                     rows, width, eps, _FP8[dtype], group, y.data_ptr(), scales.data_ptr(),
                                                     rt.current_stream(index)), 'musc_rmsnorm_rows_8bit')
    return (y, scales) if s is None else (s, y, scales)


def rms_norm(x: torch.Tensor, weight, eps: float, residual: torch.Tensor | None = None):
    """Root-mean-square norm over the last dimension, fp32 statistics, output in x's dtype
    (float32, float16 or bfloat16).

    With `residual`, returns (s, rms_norm(s)) where s = x + residual rounded to x's dtype, in
    one pass; otherwise rms_norm(x).  weight: one value per column in x's dtype or float32, or
    None.  The sum of squares is float32: a row whose squares overflow it (bfloat16 and float32 values
    past about 1e17) comes out as zeros.  No derivative."""
    return _rms(x, weight, eps, residual, None, 0)


def rms_norm_quantized(x: torch.Tensor, weight, eps: float, residual: torch.Tensor | None = None,
                       dtype: torch.dtype = torch.float8_e4m3fn, group: int = 0):
    """rms_norm with its output in 8 bits for an 8-bit product: (y8, scales), or (s, y8, scales)
    with a residual; y8.float() * scales (each scale for its columns) is the norm's value.

    dtype: torch.float8_e4m3fn or torch.float8_e5m2.  group 0: one scale per row, shape
    (..., 1); 32, 64, 128 or 256: one for each `group` columns, shape (..., width // group)."""
    if dtype not in _FP8:
        raise ValueError('dtype must be torch.float8_e4m3fn or torch.float8_e5m2')
    if group not in (0, 32, 64, 128, 256) or (group and x.shape[-1] % group):
        raise ValueError('group must be 0, 32, 64, 128 or 256 and divide the columns')
    return _rms(x, weight, eps, residual, dtype, group)


def activation_(x: torch.Tensor, mode: int) -> torch.Tensor:
    """In place: QuickGELU (mode rt.ACT_QUICK_GELU) or erf-GELU (rt.ACT_GELU)."""
    rt.require_device_tensor(x, 'x')
    if x.dtype not in _DTYPES or not x.is_contiguous():
        raise ValueError('x must be a contiguous float32 or float16 tensor')
    with torch.cuda.device(x.device):
        rc = rt.library().musc_activation(x.data_ptr(), x.data_ptr(), _DTYPES[x.dtype], int(mode), x.numel(),
                                          rt.stream(x.device))
        rt.check(rc, 'musc_activation')
    return x
