"""Rotary positions with several axes (time, height, width) on MI355X (libmusc_hip musc_rotary).

For encoders of images and video of any size, whose blocks turn q and k by the token's place
instead of adding a position embedding of one grid (the reference's encoder does the latter).
q and k are read in place from a packed projection; all heads of a token share its angles, whose
whole turns are taken off in float64.  norm_rotary takes the root-mean-square norm of every head first, in
the same pass (musc_norm_rotary).
"""
from __future__ import annotations

import math

import torch

from . import _runtime as rt

_F32, _CONTIGUOUS = torch.float32, torch.contiguous_format
_NO_WEIGHT = (None, 0, rt.DTYPE_F32, None)
_STORAGE = {torch.float32: rt.DTYPE_F32, torch.float16: rt.DTYPE_F16, torch.bfloat16: rt.DTYPE_BF16}


class RotaryAxes:
    """Which pairs of a head's channels turn with which axis, and how fast.

    sections: pairs of each axis, in order (e.g. (0, 16, 16) for 64 channels turned by rows and
    columns of (time, height, width) positions); their sum R may leave channels from 2 R on as
    they are.  Pair i of n in its axis's section turns base ** -(i / n) radians per unit of
    position; with `shared`, pair i of all R turns base ** -(i / R).  Pairs are channels
    (i, R + i), or (2 i, 2 i + 1) with `adjacent`.  Kept by the caller, as a weight is, and used by
    any call with the same head width."""

    def __init__(self, head_dim: int, sections, base: float = 10000.0, shared: bool = False, adjacent: bool = False,
                 device='cuda'):
        sections = [int(n) for n in sections]
        pairs = sum(sections)
        if not sections or min(sections) < 0 or pairs < 1 or 2 * pairs > head_dim:
            raise ValueError('sections must be pair counts, at least one pair and at most head_dim channels in all')
        if not (base > 0 and math.isfinite(base)):
            raise ValueError('base must be a positive number')
        axis, turns = [], []
        for a, n in enumerate(sections):
            for i in range(n):
                exponent = len(axis) / pairs if shared else i / n
                turns.append(float(base) ** -exponent / (2 * math.pi))
                axis.append(a)
        self.head_dim, self.pairs, self.axes, self.adjacent = int(head_dim), pairs, len(sections), bool(adjacent)
        both = torch.zeros(2 * pairs, dtype=torch.float64)       # one copy to the device for the two
        both[:pairs] = torch.tensor(turns, dtype=torch.float64)
        both[pairs:].view(torch.int32)[:pairs] = torch.tensor(axis, dtype=torch.int32)
        both = both.to(device)
        self.frequency, self.axis = both[:pairs], both[pairs:].view(torch.int32)[:pairs]


def _refuse_heads(x, name, axes):
    rt.require_device_tensor(x, name)
    raise ValueError(f'{name} must be a (B, T, heads, {axes.head_dim}) float32, float16 or bfloat16 tensor')


def _head_weight(weight, name, h, d, dtype, index):
    """(address, elements between the weights of two heads, storage, tensor) of a head norm's weight."""
    rt.require_device_tensor(weight, name)
    w_dtype, dims, n = weight.dtype, weight.dim(), weight.numel()
    if (weight.get_device() != index or (w_dtype is not dtype and w_dtype is not _F32)
            or not (n == d if dims == 1 else dims == 2 and n == h * d and weight.shape[1] == d)):
        raise ValueError(f"{name} must be ({d},) or ({h}, {d}) on its input's device, in its dtype or float32")
    at = weight.data_ptr()
    if at % 16 or not weight.is_contiguous():
        weight = weight.clone(memory_format=_CONTIGUOUS)     # read as 16-byte vectors
        at = weight.data_ptr()
    return at, d if dims == 2 else 0, _STORAGE[w_dtype], weight


def _turn(q, k, positions, axes, inverse, out, norm):
    d = axes.head_dim
    rt.require_device_tensor(q, 'q')
    if q.dim() != 4:
        _refuse_heads(q, 'q', axes)
    b, t, h, width = q.shape
    dtype, index = q.dtype, q.get_device()
    storage = _STORAGE.get(dtype)
    if width != d or storage is None:
        _refuse_heads(q, 'q', axes)
    if rt.elsewhere(q):
        with torch.cuda.device(q.device):
            return _turn(q, k, positions, axes, inverse, out, norm)
    if out is None:
        q_out = k_out = None
        rt.require_no_gradient(q, k, positions)
    else:
        q_out, k_out = (out, None) if k is None else out if len(out) == 2 else (None, None)
        if k is not None and len(out) != 2:
            raise ValueError('out must be (q_out, k_out)')
        rt.require_no_gradient(q, k, positions, q_out, k_out)
    sb, st, sh, last = q.stride()
    if last != 1:
        q = q.contiguous()
        sb, st, sh, _ = q.stride()
    # a dimension of one element has no stride
    q_args = (q.data_ptr(), sb if b > 1 else 0, st if t > 1 else 0, sh if h > 1 else 0)
    k_heads, k_args = 0, (0, 0, 0, 0, 0, 0, 0, 0)
    if k is not None:
        if not isinstance(k, torch.Tensor) or not k.is_cuda or k.dim() != 4:
            _refuse_heads(k, 'k', axes)
        kb, kt, k_heads, width = k.shape
        if width != d:
            _refuse_heads(k, 'k', axes)
        if kb != b or kt != t or k.dtype is not dtype or k.get_device() != index:
            raise ValueError('k must match q in batch, tokens, dtype and device')
        sb, st, sh, last = k.stride()
        if last != 1:
            k = k.contiguous()
            sb, st, sh, _ = k.stride()
        k_args = (k.data_ptr(), sb if b > 1 else 0, st if t > 1 else 0, sh if k_heads > 1 else 0)
    if not isinstance(positions, torch.Tensor) or not positions.is_cuda:
        rt.require_device_tensor(positions, 'positions')
    n, p_dtype, p_shape = axes.axes, positions.dtype, positions.shape
    shared = len(p_shape) == 2
    if ((p_dtype is not _F32 and p_dtype is not torch.int32) or positions.get_device() != index
            or p_shape != ((t, n) if shared else (b, t, n))):
        raise ValueError(f"positions must be float32 or int32 of shape (T, {n}) or (B, T, {n}) on q's device")
    frequency = axes.frequency
    if frequency.get_device() != index:
        raise ValueError("axes must be on q's device")
    positions = positions.contiguous()
    if norm is not None:
        q_weight, k_weight, eps = norm
        qw = kw = _NO_WEIGHT
        if q_weight is not None:
            qw = _head_weight(q_weight, 'q_weight', h, d, dtype, index)
        if k_weight is not None and k is not None:
            kw = _head_weight(k_weight, 'k_weight', k_heads, d, dtype, index)
        rt.require_no_gradient(qw[3], kw[3])
    if k is not None:
        if k_out is None:
            ko = torch.empty_like(k, memory_format=_CONTIGUOUS)
            k_args += (ko.data_ptr(), t * k_heads * d, k_heads * d, d)
        else:
            ko = rt.output_like(k_out, k, 'k_out')
            k_args += (ko.data_ptr(), *rt.token_strides(ko))
    if q_out is None:
        qo = torch.empty_like(q, memory_format=_CONTIGUOUS)
        q_args += (qo.data_ptr(), t * h * d, h * d, d)
    else:
        qo = rt.output_like(q_out, q, 'q_out')
        q_args += (qo.data_ptr(), *rt.token_strides(qo))
    if b and t and h:
        if not k_heads:
            k_args = (0, 0, 0, 0, 0, 0, 0, 0)
        call = rt.PACK_ROTARY.pack(
            *q_args, *k_args, positions.data_ptr(), 0 if shared else t * n, frequency.data_ptr(), axes.axis.data_ptr(), h, k_heads,
            storage, b, t, d, p_dtype is not _F32, n, axes.pairs, axes.adjacent, inverse)
        if norm is None:
            rt.check(rt.library().musc_rotary(call, rt.current_stream(index)), 'musc_rotary')
        else:
            rt.check(rt.library().musc_norm_rotary(call, qw[0], qw[1], qw[2], kw[0], kw[1], kw[2], eps, rt.current_stream(index)),
                     'musc_norm_rotary')
    elif k_heads:
        _turn(k, None, positions, axes, inverse, ko, None if norm is None else (norm[1], None, norm[2]))
    return qo if k is None else (qo, ko)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, axes: RotaryAxes, inverse: bool = False,
           out=None):
    """(q, k) turned by their tokens' positions, or q alone where k is None.

    q (B, T, heads, D), k (B, T, kv_heads, D), any strides with a contiguous last dimension;
    positions (T, axes) or (B, T, axes), float32 or int32.  inverse turns back (the transpose).
    out: the tensors to write, (q_out, k_out) or q_out; they may be q and k themselves, and may
    not overlap them otherwise.  No derivative."""
    return _turn(q, k, positions, axes, inverse, out, None)


def norm_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, axes: RotaryAxes, q_weight=None,
                k_weight=None, eps: float = 1e-6, out=None):
    """(q, k), or q alone where k is None, with every head's root-mean-square norm taken and then
    turned by its token's position, in one pass and with one rounding.

    y = x * weight / sqrt(mean(x^2) + eps) over the D channels of a head, in float32; then rotary's
    rotation of y.  q_weight, k_weight: (D,) for all heads or (heads, D), in the input's dtype or
    float32; None: 1.  The sum of squares is float32: a head whose squares overflow it (bfloat16 and
    float32 values past about 1e18) comes out as zeros.  The other arguments, the outputs and what they may
    overlap are rotary's.  No derivative."""
    return _turn(q, k, positions, axes, False, out, (q_weight, k_weight, float(eps)))
