"""Rotary positions with several axes (time, height, width) on MI355X (libmusc_hip musc_rotary).

For encoders of images and video of any size, whose blocks turn q and k by the token's place
instead of adding a position embedding of one grid (the reference's encoder does the latter).
q and k are read in place from a packed projection; all heads of a token share its angles, whose
whole turns are taken off in float64.
"""
from __future__ import annotations

import math

import torch

from . import _runtime as rt

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


def _head_rows(x, name, axes):
    rt.require_device_tensor(x, name)
    if x.dim() != 4 or x.shape[-1] != axes.head_dim or x.dtype not in _STORAGE:
        raise ValueError(f'{name} must be a (B, T, heads, {axes.head_dim}) float32, float16 or bfloat16 tensor')
    return x if x.stride(-1) == 1 else x.contiguous()


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, axes: RotaryAxes, inverse: bool = False,
           out=None):
    """(q, k) turned by their tokens' positions, or q alone where k is None.

    q (B, T, heads, D), k (B, T, kv_heads, D), any strides with a contiguous last dimension;
    positions (T, axes) or (B, T, axes), float32 or int32.  inverse turns back (the transpose).
    out: the tensors to write, (q_out, k_out) or q_out; they may be q and k themselves, and may
    not overlap them otherwise.  No derivative."""
    q2 = _head_rows(q, 'q', axes)
    if rt.elsewhere(q):
        with torch.cuda.device(q.device):
            return rotary(q, k, positions, axes, inverse, out)
    rt.require_no_gradient(q, k, positions, *(out if isinstance(out, (tuple, list)) else (out,)))
    index = q.get_device()
    b, t, h, d = q2.shape
    k2, ko, k_heads, k_args = None, None, 0, (0, 0, 0, 0, 0, 0, 0, 0)
    if k is not None:
        k2 = _head_rows(k, 'k', axes)
        if k2.shape[0] != b or k2.shape[1] != t or k2.dtype != q2.dtype or k2.get_device() != index:
            raise ValueError('k must match q in batch, tokens, dtype and device')
        if out is not None and len(out) != 2:
            raise ValueError('out must be (q_out, k_out)')
    rt.require_device_tensor(positions, 'positions')
    shape = positions.shape
    if (positions.dtype not in (torch.float32, torch.int32) or positions.get_device() != index
            or (shape != (b, t, axes.axes) and shape != (t, axes.axes))):
        raise ValueError(f"positions must be float32 or int32 of shape (T, {axes.axes}) or (B, T, {axes.axes}) on q's device")
    if axes.frequency.get_device() != index:
        raise ValueError("axes must be on q's device")
    positions = positions.contiguous()
    if k2 is not None:
        ko = rt.output_like(out[1] if out is not None else None, k2, 'k_out')
        if k2.shape[2]:
            k_heads = k2.shape[2]
            k_args = (k2.data_ptr(), *rt.token_strides(k2), ko.data_ptr(), *rt.token_strides(ko))
        out = out[0] if out is not None else None
    qo = rt.output_like(out, q2, 'q_out')
    if b and t and h:
        call = rt.PACK_ROTARY.pack(
            q2.data_ptr(), *rt.token_strides(q2), qo.data_ptr(), *rt.token_strides(qo), *k_args, positions.data_ptr(),
            0 if len(shape) == 2 else t * axes.axes, axes.frequency.data_ptr(), axes.axis.data_ptr(), h, k_heads, _STORAGE[q2.dtype], b, t,
            d, positions.dtype == torch.int32, axes.axes, axes.pairs, axes.adjacent, inverse)
        rt.check(rt.library().musc_rotary(call, rt.current_stream(index)), 'musc_rotary')
    elif k_heads:
        rotary(k2, None, positions, axes, inverse, ko)
    return qo if k is None else (qo, ko)
