"""Attention over documents, prefixes and frames on MI355X (libmusc_hip musc_masked_attention_fwd).

The fused block attention of _attention_hip sees every token of one image; here a query sees
the keys of its own document (an image of a packed batch, the live part of a padded one) whose
order is not past its own (a prefix, a causal text, the frames of a clip), and the scores may
be capped by a tanh and lowered with the distance of two tokens.  The reference's blocks pass
masks to torch's math path (models/backbone/open_clip/transformer.py:228-234); nothing here
writes the logits or a mask to memory.
"""
from __future__ import annotations

import ctypes

import torch

from . import _runtime as rt

_STORAGE = {torch.float32: rt.DTYPE_F32, torch.float16: rt.DTYPE_F16, torch.bfloat16: rt.DTYPE_BF16}
SUMMARY_KEYS = 32


class Tokens:
    """Where the tokens of one side of an attention call stand; made once per batch and shared by
    all of its blocks.

    documents  int32 (T,) or (B, T): tokens see only tokens of their own document; negative ids
               are padding, which sees nothing and is not seen.  None: all tokens see one another.
    order      int32, the same shape: a query sees the keys whose order is at most its own.  The
               token's index gives causal attention, 0 for all tokens of a prefix and the index
               after it a prefix that sees itself whole, the frame's number attention to this and
               earlier frames.  None: no such limit.
    positions  float32 (T, axes) or (B, T, axes), up to 3 axes, for the bias by distance.

    The tensors are kept, not copied.  As keys they are also summarised (32 at a time) when the
    object is made; call refresh() after changing them in place.  queries_only leaves that out."""

    def __init__(self, documents=None, order=None, positions=None, queries_only: bool = False):
        for name, x, dtype in (('documents', documents, torch.int32), ('order', order, torch.int32),
                               ('positions', positions, torch.float32)):
            if x is None:
                continue
            rt.require_device_tensor(x, name)
            if x.dtype != dtype or not x.is_contiguous():
                raise ValueError(f'{name} must be a contiguous {dtype} tensor')
        if documents is None and order is not None:
            raise ValueError('order needs documents (zeros for one document)')
        if documents is not None and documents.dim() not in (1, 2):
            raise ValueError('documents must be (T,) or (B, T)')
        if order is not None and (order.shape != documents.shape or order.device != documents.device):
            raise ValueError("order must match documents")
        if positions is not None:
            if positions.dim() not in (2, 3) or not 1 <= positions.shape[-1] <= 3:
                raise ValueError('positions must be (T, axes) or (B, T, axes) with 1 to 3 axes')
            if documents is not None and (positions.shape[-2] != documents.shape[-1]
                                          or positions.device != documents.device):
                raise ValueError('positions must have the tokens of documents')
        self.documents, self.order, self.positions, self.summary = documents, order, positions, None
        if documents is not None and not queries_only:
            b, t = documents.shape if documents.dim() == 2 else (1, documents.shape[0])
            self.summary = torch.empty((b, -(-t // SUMMARY_KEYS), 4), dtype=torch.int32, device=documents.device)
            self.refresh()

    def refresh(self) -> None:
        """Summarises the keys again, on the current stream, after a change of documents or order."""
        if self.summary is None:
            return
        docs = self.documents
        with torch.cuda.device(docs.device):
            rt.check(rt.library().musc_token_summary(
                docs.data_ptr(), None if self.order is None else self.order.data_ptr(), self.summary.shape[0],
                docs.shape[-1], self.summary.data_ptr(), rt.stream(docs.device)), 'musc_token_summary')

    def rows(self, name: str, x: torch.Tensor, batch: int, tokens: int, device) -> int:
        """Batch stride of one of the tensors, 0 where the batch shares one row."""
        token_dim = 1 if x.is_floating_point() else 0
        dims = x.dim() - token_dim
        if x.shape[dims - 1] != tokens or (dims == 2 and x.shape[0] not in (1, batch)) or x.device != device:
            raise ValueError(f'{name} has {tuple(x.shape)}: {tokens} tokens of {batch} batch entries (or 1) on {device} needed')
        return 0 if dims == 1 or x.shape[0] == 1 else x.stride(0)


_EVERY = Tokens()


def _heads(x, name, like):
    rt.require_device_tensor(x, name)
    if x.dim() != 4 or x.dtype not in _STORAGE:
        raise ValueError(f'{name} must be a (B, T, heads, D) float32, float16 or bfloat16 tensor')
    if like is not None and (x.dtype != like.dtype or x.device != like.device or x.shape[0] != like.shape[0]
                             or x.shape[3] != like.shape[3]):
        raise ValueError(f'{name} must match q in batch, head width, dtype and device')
    per = 16 // x.element_size()
    if x.stride(3) == 1 and x.data_ptr() % 16 == 0:
        strides = rt.token_strides(x)
        if not any(s % per for s in strides):
            return x, strides
    x = x.contiguous()
    return x, rt.token_strides(x)


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, keys: Tokens | None = None,
                     queries: Tokens | None = None, cap: float = 0.0, slopes: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax over the keys each query sees of c(scale q k^T) - sum_a slopes[h, a] |distance_a|,
    times v; (B, Tq, heads, D).

    q (B, Tq, heads, D), k and v (B, Tk, kv_heads, D), heads a multiple of kv_heads, float32,
    float16 or bfloat16, D up to 128 in steps of 16 bytes; views of a packed projection are read
    in place where each row starts on 16 bytes, and copied otherwise.
    keys, queries: the Tokens of both sides; queries defaults to keys (self-attention), no keys at
    all lets every query see every key.  A query that sees no key gets zeros.
    cap > 0: scores become cap tanh(score / cap) before the bias.  slopes: float32 (heads, axes),
    needs positions on both sides.  No backward pass."""
    rt.require_no_gradient(q, k, v, slopes)
    q, qs = _heads(q, 'q', None)
    k, ks = _heads(k, 'k', q)
    v, vs = _heads(v, 'v', q)
    b, tq, h, d = q.shape
    tk, hk = k.shape[1:3]
    if v.shape != k.shape:
        raise ValueError('v must match k in shape')
    if hk < 1 or h % hk:
        raise ValueError('heads of q must be a multiple of the heads of k')
    per = 16 // q.element_size()
    if d < per or d > 128 or d % per:
        raise ValueError(f'head width {d}: multiples of {per} up to 128 are supported for {q.dtype}')
    keys = _EVERY if keys is None else keys
    queries = keys if queries is None else queries
    device = q.device
    if (keys.documents is None) != (queries.documents is None) or (keys.order is None) != (queries.order is None):
        raise ValueError('keys and queries must both have documents, and both an order, or neither')
    docs, orders, q_sb, k_sb, sum_sb = (None, None), (None, None), 0, 0, 0
    summary = None
    if keys.documents is not None:
        if keys.summary is None:
            raise ValueError('keys were made with queries_only')
        q_sb = queries.rows('queries.documents', queries.documents, b, tq, device)
        k_sb = keys.rows('keys.documents', keys.documents, b, tk, device)
        docs = queries.documents.data_ptr(), keys.documents.data_ptr()
        if keys.order is not None:
            orders = queries.order.data_ptr(), keys.order.data_ptr()
        summary, sum_sb = keys.summary.data_ptr(), (keys.summary.shape[1] if k_sb else 0)
    axes, pos, qp_sb, kp_sb, slope_ptr = 0, (None, None), 0, 0, None
    if slopes is not None:
        if keys.positions is None or queries.positions is None:
            raise ValueError('slopes need positions of keys and queries')
        axes = keys.positions.shape[-1]
        rt.require_device_tensor(slopes, 'slopes')
        if (slopes.dtype != torch.float32 or slopes.shape not in ((h, axes), (h,) if axes == 1 else (h, axes))
                or queries.positions.shape[-1] != axes or slopes.device != device):
            raise ValueError(f"slopes must be float32 ({h}, {axes}) on q's device, positions of both sides have as many axes")
        slopes = slopes.contiguous()
        qp_sb = queries.rows('queries.positions', queries.positions, b, tq, device)
        kp_sb = keys.rows('keys.positions', keys.positions, b, tk, device)
        pos, slope_ptr = (queries.positions.data_ptr(), keys.positions.data_ptr()), slopes.data_ptr()
    with torch.cuda.device(device):
        o = rt.output_like(out, q, 'out')
        os_ = rt.token_strides(o)
        if o.data_ptr() % 16 or any(s % per for s in os_):
            raise ValueError('rows of out must start on 16 bytes')
        if not (b and tq and h):
            return o
        if not tk:
            return o.zero_()
        call = rt.MaskedAttention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), *qs, *ks, *vs, *os_,
                                  _STORAGE[q.dtype], b, tq, tk, h, hk, d, float(scale), float(cap), docs[0], orders[0],
                                  docs[1], orders[1], q_sb, k_sb, summary, sum_sb, pos[0], pos[1], qp_sb, kp_sb,
                                  slope_ptr, axes)
        lib, need = rt.library(), ctypes.c_size_t()
        rt.check(lib.musc_masked_attention_workspace_bytes(call, ctypes.byref(need)),
                 'musc_masked_attention_workspace_bytes')
        ws = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
        rt.check(lib.musc_masked_attention_fwd(call, None if ws is None else ws.data_ptr(), need.value,
                                               rt.stream(device)), 'musc_masked_attention_fwd')
    return o
