"""Attention over documents, prefixes and frames on MI355X (libmusc_hip musc_masked_attention_fwd).

The fused block attention of _attention_hip sees every token of one image; here a query sees
the keys of its own document (an image of a packed batch, the live part of a padded one) whose
order is not past its own (a prefix, a causal text, the frames of a clip), and the scores may
be capped by a tanh and lowered with the distance of two tokens.  The reference's blocks pass
masks to torch's math path (models/backbone/open_clip/transformer.py:232-234); nothing here
writes the logits or a mask to memory.
"""
from __future__ import annotations

import ctypes

import torch

from . import _runtime as rt

_STORAGE = {torch.float32: rt.DTYPE_F32, torch.float16: rt.DTYPE_F16, torch.bfloat16: rt.DTYPE_BF16}
SUMMARY_KEYS = 32
ROW_TILE = 128
SCHEDULE_GROUPS = (1, 2, 4, 8)
SCHEDULE_MAX_TOKENS = 16384
SCHEDULE_MAX_TILES = 1 << 22   # of all batch entries; more run unscheduled


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
    object is made, on the current stream, and self-attention over them is scheduled (its longest
    rows first, in parts where there are few); call refresh() after changing them in place.  queries_only leaves
    that out.  Calls on another stream than the one it was made on keep its memory until they are done, also
    where the object goes before; that stream waits for what made it as the caller says, as with any tensor."""

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
        self._schedule = self._made_on = None
        for x in (documents, positions):
            if x is not None:
                self._made_on = rt.current_stream(x.get_device())
        if documents is not None and not queries_only:
            b, t = documents.shape if documents.dim() == 2 else (1, documents.shape[0])
            self.summary = torch.empty((b, -(-t // SUMMARY_KEYS), 4), dtype=torch.int32, device=documents.device)
            # blocks for 1, 2, 4 and 8 query heads per key head, of n row groups each
            tiles = [-(-t * group // ROW_TILE) for group in SCHEDULE_GROUPS]
            if 0 < t <= SCHEDULE_MAX_TOKENS and b * sum(tiles) < SCHEDULE_MAX_TILES:
                blocks = [4 + 5 * n + (9 * n + 4) // 5 + n // 4 for n in tiles]
                self._schedule = torch.empty((b * sum(blocks),), dtype=torch.int32, device=documents.device)
                # bytes before a group's blocks (no address: copies have their own), ints of a block
                self._schedule_of = {group: (4 * b * sum(blocks[:i]), blocks[i]) for i, group in enumerate(SCHEDULE_GROUPS)}
            self.refresh()

    def __getstate__(self):
        return {**self.__dict__, '_made_on': None}      # a copy's tensors may be of any stream

    def used_on(self, stream: int, device: torch.device) -> None:
        """Keeps the tensors' memory for work just begun on `stream`, the device's current one."""
        if stream != self._made_on:
            for x in (self.documents, self.order, self.positions, self.summary, self._schedule):
                if x is not None:
                    x.record_stream(torch.cuda.current_stream(device))

    def refresh(self) -> None:
        """Summarises the keys again, on the current stream, after a change of documents or order."""
        if self.summary is None or not self.summary.numel():
            return
        docs = self.documents
        self.used_on(rt.current_stream(docs.get_device()), docs.device)
        with torch.cuda.device(docs.device):
            rt.check(rt.library().musc_token_summary(
                docs.data_ptr(), None if self.order is None else self.order.data_ptr(), self.summary.shape[0],
                docs.shape[-1], self.summary.data_ptr(), rt.stream(docs.device)), 'musc_token_summary')
            if self._schedule is not None:
                rt.check(rt.library().musc_token_schedule(
                    docs.data_ptr(), None if self.order is None else self.order.data_ptr(), self.summary.data_ptr(),
                    self.summary.shape[0], docs.shape[-1], self._schedule.data_ptr(), rt.stream(docs.device)),
                    'musc_token_schedule')


def _batch_stride(name: str, x: torch.Tensor, leading, batch: int, tokens: int, index: int) -> int:
    """Batch stride of documents or positions, `leading` their (T,) or (B, T); 0 where the batch
    shares one row."""
    if leading[-1] == tokens and x.get_device() == index:
        if len(leading) == 1 or leading[0] == 1:
            return 0
        if leading[0] == batch:
            return x.stride(0)
    raise ValueError(f'{name} has {tuple(x.shape)}: {tokens} tokens of {batch} batch entries (or 1) on device {index} needed')


_EVERY = Tokens()


def _heads(x, per):
    """x, copied where its rows do not start on 16 bytes (per elements), and its strides."""
    strides = rt.token_strides(x)
    if x.stride(3) == 1 and not x.data_ptr() % 16 and not (strides[0] | strides[1] | strides[2]) % per:
        return x, strides
    x = x.clone(memory_format=torch.contiguous_format)  # also where it is contiguous and starts off 16 bytes
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
    all lets every query see every key.  A query that sees no key gets zeros, as does one whose seen
    scores are all minus infinity.
    cap > 0 (up to 2^60; 16-bit types are quickest up to 128): scores become cap tanh(score / cap) before the bias.  slopes: float32 (heads, axes),
    needs positions on both sides.  out: the tensor to write, rows on 16 bytes; it may not overlap q, k
    or v.  No derivative."""
    for name, x in (('q', q), ('k', k), ('v', v)):
        rt.require_device_tensor(x, name)
        if x.dim() != 4:
            raise ValueError(f'{name} must be a (B, T, heads, D) tensor')
    if rt.elsewhere(q):
        with torch.cuda.device(q.device):
            return masked_attention(q, k, v, scale, keys, queries, cap, slopes, out)
    rt.require_no_gradient(q, k, v, slopes, out)
    dtype, index = q.dtype, q.get_device()
    if dtype not in _STORAGE:
        raise ValueError('q must be float32, float16 or bfloat16')
    b, tq, h, d = q.shape
    kb, tk, hk, kd = k.shape
    if kb != b or kd != d or k.dtype != dtype or v.dtype != dtype or k.get_device() != index or v.get_device() != index:
        raise ValueError('k and v must match q in batch, head width, dtype and device')
    if v.shape != k.shape:
        raise ValueError('v must match k in shape')
    if hk < 1 or h % hk:
        raise ValueError('heads of q must be a multiple of the heads of k')
    per = 16 // q.element_size()
    if d < per or d > 128 or d % per:
        raise ValueError(f'head width {d}: multiples of {per} up to 128 are supported for {dtype}')
    q, qs = _heads(q, per)
    k, ks = _heads(k, per)
    v, vs = _heads(v, per)
    keys = _EVERY if keys is None else keys
    queries = keys if queries is None else queries
    kdocs, qdocs, kord, qord = keys.documents, queries.documents, keys.order, queries.order
    if (kdocs is None) != (qdocs is None) or (kord is None) != (qord is None):
        raise ValueError('keys and queries must both have documents, and both an order, or neither')
    q_sb = k_sb = sum_sb = qd_ptr = kd_ptr = qo_ptr = ko_ptr = sum_ptr = 0
    if kdocs is not None:
        if keys.summary is None:
            raise ValueError('keys were made with queries_only')
        q_sb = _batch_stride('queries.documents', qdocs, qdocs.shape, b, tq, index)
        k_sb = _batch_stride('keys.documents', kdocs, kdocs.shape, b, tk, index)
        qd_ptr, kd_ptr, sum_ptr = qdocs.data_ptr(), kdocs.data_ptr(), keys.summary.data_ptr()
        sum_sb = keys.summary.shape[1] if k_sb else 0
        if kord is not None:
            qo_ptr, ko_ptr = qord.data_ptr(), kord.data_ptr()
    axes = qp_ptr = kp_ptr = qp_sb = kp_sb = slope_ptr = 0
    if slopes is not None:
        kpos, qpos = keys.positions, queries.positions
        if kpos is None or qpos is None:
            raise ValueError('slopes need positions of keys and queries')
        rt.require_no_gradient(kpos, qpos)
        axes = kpos.shape[-1]
        rt.require_device_tensor(slopes, 'slopes')
        if (slopes.dtype != torch.float32 or slopes.get_device() != index or qpos.shape[-1] != axes
                or not (slopes.shape == (h, axes) or (axes == 1 and slopes.shape == (h,)))):
            raise ValueError(f"slopes must be float32 ({h}, {axes}) on q's device, positions of both sides have as many axes")
        slopes = slopes.contiguous()
        qp_sb = _batch_stride('queries.positions', qpos, qpos.shape[:-1], b, tq, index)
        kp_sb = _batch_stride('keys.positions', kpos, kpos.shape[:-1], b, tk, index)
        qp_ptr, kp_ptr, slope_ptr = qpos.data_ptr(), kpos.data_ptr(), slopes.data_ptr()
    o = rt.output_like(out, q, 'out')
    os_ = rt.token_strides(o)
    if o.data_ptr() % 16 or (os_[0] | os_[1] | os_[2]) % per:
        raise ValueError('rows of out must start on 16 bytes')
    if not (b and tq and h):
        return o
    if not tk:
        return o.zero_()
    schedule = schedule_sb = 0
    if queries is keys and keys._schedule is not None and h // hk in keys._schedule_of:
        before, block = keys._schedule_of[h // hk]
        schedule, schedule_sb = keys._schedule.data_ptr() + before, block if k_sb else 0
    call = rt.PACK_MASKED_ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), *qs, *ks, *vs, *os_, _STORAGE[dtype], b, tq, tk, h, hk, d,
        scale, cap, qd_ptr, qo_ptr, kd_ptr, ko_ptr, q_sb, k_sb, sum_ptr, sum_sb, qp_ptr, kp_ptr, qp_sb, kp_sb, slope_ptr,
        axes, schedule, schedule_sb)
    lib, need, ws = rt.library(), ctypes.c_size_t(), None
    rt.check(lib.musc_masked_attention_workspace_bytes(call, ctypes.byref(need)), 'musc_masked_attention_workspace_bytes')
    if need.value:
        ws = torch.empty(need.value, dtype=torch.uint8, device=q.device)
    stream = rt.current_stream(index)
    rt.check(lib.musc_masked_attention_fwd(call, None if ws is None else ws.data_ptr(), need.value, stream),
             'musc_masked_attention_fwd')
    if keys is not _EVERY:
        keys.used_on(stream, q.device)
    if queries is not keys:
        queries.used_on(stream, q.device)
    return o
