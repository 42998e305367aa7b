"""The operators of packed and masked encoders, as cases that can be timed and compared.

`run()` computes each of them in elementary torch operations in 32 bits (64 for angles),
or, with `own` set, through musc_hip's public entry points.  `exact()` gives the same
outputs from the definitions in float64.

  attention   softmax attention whose keys are limited by documents and an order, with an
              optional tanh cap on the scores and an optional bias by distance:
              score(i, j) = c(scale q_i . k_j) - sum_a slope[h, a] |p_a(i) - p_a(j)|,
              c(s) = cap tanh(s / cap) or s; key j is seen by query i when both are of the
              same document (ids >= 0) and order(j) <= order(i); a query that sees no key
              gets zeros
  rotary      rotation of q and k by angles position[axis(i)] * base^(-exponent(i)),
              pairs of channels (i, i + R) or (2 i, 2 i + 1), the rest left as it is
  norm        s = x + residual rounded to the type, y = s / sqrt(mean(s^2) + eps) * weight,
              as it is or in 8 bits with one scale per row or per group of columns
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = 'cuda'
DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
E4M3_MAX = 448.0
EPS = 1e-6


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one latent query pools one 518 px image (37 x 37 patches + class token): a single-token call
        dict(name='attend_pool_1', op='attention', layout='pool', images=1, low=37, high=37, shapes=1, latents=1,
             heads=16, kv_heads=16, dim=64, cap=0.0, bias=False, dtype='f16'),
        # twelve images of their own aspect ratios packed into one sequence, distance bias over rows and columns
        dict(name='attend_packed_f16', op='attention', layout='packed', images=12, low=13, high=40, shapes=2, heads=16,
             kv_heads=16, dim=64, cap=0.0, bias=True, dtype='f16'),
        # the same without autocast, no bias: four images
        dict(name='attend_packed_f32', op='attention', layout='packed', images=4, low=20, high=37, shapes=3, heads=16,
             kv_heads=16, dim=64, cap=0.0, bias=False, dtype='f32'),
        # a caption after each image: the 1369 patches see one another, the text sees what is before it; padded batch
        dict(name='attend_prefix_bf16', op='attention', layout='prefix', batch=4, image=1369, text=700, shapes=4,
             heads=16, kv_heads=4, dim=128, cap=50.0, bias=False, dtype='bf16'),
        # a clip of 16 frames of 32 x 32 patches, each frame sees itself and the earlier ones
        dict(name='attend_frames_bf16', op='attention', layout='frames', clips=1, frames=16, side=32, heads=16,
             kv_heads=16, dim=128, cap=0.0, bias=False, dtype='bf16'),
        # one new token for each of eight requests, over keys and values of up to 32768 tokens
        dict(name='attend_step_bf16', op='attention', layout='step', batch=8, cache=32768, shapes=5, heads=32,
             kv_heads=8, dim=128, cap=30.0, bias=True, dtype='bf16'),
        # q and k of one encoder batch (four 518 px images, packed projection), angles by row and column
        dict(name='rotary_images_f16', op='rotary', batch=4, grid='1,37,37', cls=True, heads=16, kv_heads=16, dim=64,
             sections='0,16,16', shared=False, adjacent=False, base=100.0, far=0, dtype='f16'),
        # a clip of 64 frames of 16 x 16 patches, grouped heads, one row of frequencies over time, height and width
        dict(name='rotary_video_bf16', op='rotary', batch=1, grid='64,16,16', cls=False, heads=32, kv_heads=8, dim=128,
             sections='16,24,24', shared=True, adjacent=False, base=1e6, far=0, dtype='bf16'),
        # one new token for each of eight requests, far into their sequences
        dict(name='rotary_step_bf16', op='rotary', batch=8, grid='1,1,1', cls=False, heads=32, kv_heads=8, dim=128,
             sections='16,24,24', shared=True, adjacent=False, base=1e6, far=200000, dtype='bf16'),
        # the norm of eight single tokens, 8-bit output with a scale per row
        dict(name='norm_step_bf16', op='norm', rows=8, width=4096, residual=True, group=0, eight=True, dtype='bf16'),
        # the tokens of one encoder batch, residual and norm in one pass
        dict(name='norm_images_f16', op='norm', rows=5480, width=1024, residual=True, group=0, eight=False, dtype='f16'),
        # many wide rows, 8-bit output with a scale for each 128 columns
        dict(name='norm_wide_bf16', op='norm', rows=16384, width=8192, residual=True, group=128, eight=True,
             dtype='bf16'),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['attention', 'attention', 'rotary', 'norm'])
    dtype = rng.choice(['f16', 'bf16', 'f32'])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    if op == 'attention':
        case = dict(op=op, layout=rng.choice(['packed', 'pool', 'prefix', 'frames', 'step']), heads=heads,
                    kv_heads=kv_heads, dim=rng.choice([32, 64, 72, 80, 96, 128]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                    bias=rng.random() < 0.5, dtype=dtype, shapes=rng.randrange(1 << 20))
        if case['layout'] in ('packed', 'pool'):
            low = rng.randint(1, 24)
            case.update(images=_log(rng, 1, 12), low=low, high=low + rng.randint(0, 16))
            if case['layout'] == 'pool':
                case.update(latents=rng.choice([1, 1, 2, 5, 32]))
        elif case['layout'] == 'prefix':
            case.update(batch=rng.randint(1, 4), image=_log(rng, 1, 1600), text=_log(rng, 1, 1000))
        elif case['layout'] == 'frames':
            case.update(clips=rng.randint(1, 2), frames=_log(rng, 1, 16), side=rng.randint(3, 22))
        else:
            case.update(batch=_log(rng, 1, 16), cache=_log(rng, 16, 16384))
        return case
    if op == 'rotary':
        dim = rng.choice([32, 64, 72, 80, 96, 128])
        pairs = dim // 2 - rng.choice([0, 0, 4])
        t = rng.choice([0, 0, pairs // 4])
        h = (pairs - t) // 2
        frames, rows, columns = (1 if t == 0 else _log(rng, 1, 32)), _log(rng, 1, 40), _log(rng, 1, 40)
        return dict(op=op, batch=rng.randint(1, 4), grid=f'{frames},{rows},{columns}', cls=rng.random() < 0.5,
                    heads=heads, kv_heads=kv_heads, dim=dim, sections=f'{t},{h},{pairs - t - h}',
                    shared=rng.random() < 0.5, adjacent=rng.random() < 0.5, base=rng.choice([100.0, 1e4, 1e6]),
                    far=rng.choice([0, 0, rng.randrange(1 << 18)]), dtype=dtype)
    group = rng.choice([0, 0, 32, 64, 128])
    width = (group * _log(rng, 1, 64)) if group else _log(rng, 8, 8192)
    return dict(op='norm', rows=_log(rng, 1, 16384), width=width, residual=rng.random() < 0.7, group=group,
                eight=bool(group) or rng.random() < 0.5, dtype=dtype)


# --------------------------------------------------------------------------- layouts of tokens
def _grids(case):
    rng = random.Random(case['shapes'])
    return [(rng.randint(case['low'], case['high']), rng.randint(case['low'], case['high'])) for _ in range(case['images'])]


def _prompts(case):
    rng = random.Random(case['shapes'])
    return [case['image'] + rng.randint(1, case['text']) for _ in range(case['batch'])]


def _filled(case):
    rng = random.Random(case['shapes'])
    return [rng.randint(max(1, case['cache'] // 4), case['cache']) for _ in range(case['batch'])]


def _grid_positions(frames, rows, columns):
    axes = torch.meshgrid(torch.arange(frames), torch.arange(rows), torch.arange(columns), indexing='ij')
    return torch.stack([a.reshape(-1) for a in axes], dim=-1).float()


def _tokens(case):
    """The two sides of an attention call: dicts of documents (B, T) int32, order (B, T) int32 or
    None, positions (B, T, A) float32 or None, on the host."""
    layout = case['layout']
    if layout in ('packed', 'pool'):
        grids = _grids(case)
        docs = torch.cat([torch.full((h * w,), i, dtype=torch.int32) for i, (h, w) in enumerate(grids)])[None]
        pos = torch.cat([_grid_positions(1, h, w)[:, 1:] for h, w in grids])[None]
        keys = dict(documents=docs, order=None, positions=pos)
        if layout == 'packed':
            return keys, keys
        latents = case['latents']
        qdocs = torch.arange(len(grids), dtype=torch.int32).repeat_interleave(latents)[None]
        centre = torch.tensor([[(h // 2, w // 2)] * latents for h, w in grids], dtype=torch.float32).reshape(1, -1, 2)
        return dict(documents=qdocs, order=None, positions=centre), keys
    if layout == 'prefix':
        t, at = case['image'] + case['text'], torch.arange(case['image'] + case['text'], dtype=torch.int32)
        lengths = torch.tensor(_prompts(case), dtype=torch.int32)[:, None]
        docs = torch.where(at[None] < lengths, 0, -1).to(torch.int32)
        order = torch.where(at < case['image'], 0, at)[None].expand(case['batch'], t).contiguous().to(torch.int32)
        side = dict(documents=docs, order=order, positions=at.float()[None, :, None].expand(case['batch'], t, 1).contiguous())
        return side, side
    if layout == 'frames':
        per, n = case['side'] ** 2, case['clips']
        docs = torch.arange(n, dtype=torch.int32).repeat_interleave(case['frames'] * per)[None]
        order = torch.arange(case['frames'], dtype=torch.int32).repeat_interleave(per).repeat(n)[None]
        pos = _grid_positions(case['frames'], case['side'], case['side']).repeat(n, 1)[None]
        side = dict(documents=docs, order=order, positions=pos)
        return side, side
    b, cache = case['batch'], case['cache']
    at = torch.arange(cache, dtype=torch.int32)[None].expand(b, cache).contiguous()
    last = torch.tensor(_filled(case), dtype=torch.int32)[:, None] - 1
    keys = dict(documents=torch.zeros_like(at), order=at, positions=at.float()[..., None].contiguous())
    return dict(documents=torch.zeros_like(last), order=last, positions=last.float()[..., None].contiguous()), keys


def _axes_of(case):
    return {'packed': 2, 'pool': 2, 'prefix': 1, 'frames': 3, 'step': 1}[case['layout']]


def _pairs(case):
    """(pairs of query and key that see one another, keys that a query sees)"""
    layout = case['layout']
    if layout in ('packed', 'pool'):
        sizes = [h * w for h, w in _grids(case)]
        return (sum(n * n for n in sizes) if layout == 'packed' else case['latents'] * sum(sizes)), sum(sizes)
    if layout == 'prefix':
        p = case['image']
        return sum(p * p + (n * (n + 1) - p * (p + 1)) // 2 for n in _prompts(case)), sum(_prompts(case))
    if layout == 'frames':
        per, f = case['side'] ** 2, case['frames']
        return case['clips'] * per * per * f * (f + 1) // 2, case['clips'] * f * per
    return sum(_filled(case)), sum(_filled(case))


# --------------------------------------------------------------------------- inputs
def _package():
    pkg = os.path.abspath('musc-gpu_amd')
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case['dtype']]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)

    if case['op'] == 'attention':
        return _prepare_attention(case, g, normal)
    if case['op'] == 'rotary':
        return _prepare_rotary(case, g, normal)
    rows, width = case['rows'], case['width']
    scale = torch.exp(torch.randn((rows, 1), generator=g, device=DEV) * 0.5)
    return dict(case=case, x=(normal(rows, width).float() * scale).to(dtype),
                residual=normal(rows, width, scale=0.5) if case['residual'] else None,
                weight=1.0 + 0.2 * torch.randn((width,), generator=g, device=DEV))


def _prepare_attention(case, g, normal):
    queries, keys = _tokens(case)
    on = lambda side: {k: v if v is None else v.to(DEV) for k, v in side.items()}  # noqa: E731
    q_side, k_side = on(queries), on(keys)
    if not case['bias']:
        q_side['positions'] = k_side['positions'] = None
    h, hk, d = case['heads'], case['kv_heads'], case['dim']
    b, t = keys['documents'].shape
    if queries is keys:  # views of one packed projection, as an encoder block has them
        qkv = normal(b, t, h + 2 * hk, d)
        q, k, v = qkv[:, :, :h], qkv[:, :, h:h + hk], qkv[:, :, h + hk:]
    else:
        q, k, v = normal(b, queries['documents'].shape[1], h, d), normal(b, t, hk, d), normal(b, t, hk, d)
    slopes = None
    if case['bias']:
        slopes = (2.0 ** (-8.0 * torch.arange(1, h + 1, device=DEV) / h))[:, None].expand(h, _axes_of(case)).contiguous()
    state = dict(case=case, q=q, k=k, v=v, q_side=q_side, k_side=k_side, slopes=slopes, scale=2.0 / math.sqrt(d))
    if own:
        _package()
        from musc_hip._masked_attention_hip import Tokens
        state['keys'] = Tokens(**k_side)
        state['queries'] = state['keys'] if queries is keys else Tokens(**q_side, queries_only=True)
    return state


def _sections(case):
    """(axis of each pair, exponent of each pair's frequency)"""
    sizes = [int(x) for x in case['sections'].split(',')]
    total = sum(sizes)
    axis, exponent = [], []
    for a, n in enumerate(sizes):
        for i in range(n):
            exponent.append(len(axis) / total if case['shared'] else i / n)
            axis.append(a)
    return axis, exponent


def _prepare_rotary(case, g, normal):
    frames, rows, columns = (int(x) for x in case['grid'].split(','))
    pos = _grid_positions(frames, rows, columns).to(DEV) + float(case['far'])
    if case['cls']:
        pos = torch.cat([torch.zeros((1, 3), device=DEV), pos])
    h, hk, d, b, t = case['heads'], case['kv_heads'], case['dim'], case['batch'], pos.shape[0]
    # each request or image of the batch is somewhere else
    pos = pos[None] + torch.randint(0, 16, (b, 1, 1), generator=g, device=DEV).float()
    qkv = normal(b, t, h + 2 * hk, d)
    axis, exponent = _sections(case)
    state = dict(case=case, q=qkv[:, :, :h], k=qkv[:, :, h:h + hk], positions=pos,
                 axis=torch.tensor(axis, device=DEV), exponent=torch.tensor(exponent, dtype=torch.float64, device=DEV))
    if own:
        _package()
        from musc_hip._rotary_hip import RotaryAxes
        state['axes'] = RotaryAxes(d, [int(x) for x in case['sections'].split(',')], base=case['base'],
                                   shared=case['shared'], adjacent=case['adjacent'], device=DEV)
    return state


# --------------------------------------------------------------------------- one pass
def run(state):
    return {'attention': _attention, 'rotary': _rotary, 'norm': _norm}[state['case']['op']](state)


def _visible(q_side, k_side):
    seen = (q_side['documents'][:, :, None] == k_side['documents'][:, None, :]) & (k_side['documents'] >= 0)[:, None, :]
    if k_side['order'] is not None:
        seen = seen & (k_side['order'][:, None, :] <= q_side['order'][:, :, None])
    return seen


def _attention(state):
    case, q, k, v = state['case'], state['q'], state['k'], state['v']
    if own:
        from musc_hip._masked_attention_hip import masked_attention
        return masked_attention(q, k, v, state['scale'], keys=state['keys'], queries=state['queries'], cap=case['cap'],
                                slopes=state['slopes'])
    b, tq, h, d = q.shape
    tk, hk = k.shape[1:3]
    q32 = q.float().permute(0, 2, 1, 3).reshape(b, hk, (h // hk) * tq, d)
    k32 = k.float().permute(0, 2, 3, 1).contiguous()
    v32 = v.float().permute(0, 2, 1, 3).contiguous()
    s = (q32 @ k32).view(b, h, tq, tk) * state['scale']
    if case['cap']:
        s = case['cap'] * torch.tanh(s / case['cap'])
    if state['slopes'] is not None:
        apart = (state['q_side']['positions'][:, :, None] - state['k_side']['positions'][:, None]).abs()
        s = s - sum(w[:, None, None] * x[:, None] for w, x in zip(state['slopes'].unbind(1), apart.unbind(-1)))
    s = s.masked_fill(~_visible(state['q_side'], state['k_side'])[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, -1, tk) @ v32).view(b, h, tq, d)
    return torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3).to(q.dtype)


def _rotary(state):
    case = state['case']
    if own:
        from musc_hip._rotary_hip import rotary
        return rotary(state['q'], state['k'], state['positions'], state['axes'])
    frequency = case['base'] ** -state['exponent']
    angle = state['positions'].double()[..., state['axis']] * frequency  # (B, T, pairs)
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    return (_rotated(state['q'], cos, sin, case['adjacent']), _rotated(state['k'], cos, sin, case['adjacent']))


def _rotated(x, cos, sin, adjacent):
    n = cos.shape[-1]
    x32 = x.float()
    if adjacent:
        a, b = x32[..., 0:2 * n:2], x32[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x32[..., :n], x32[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x32[..., 2 * n:]], dim=-1).to(x.dtype)


def _norm(state):
    case, x, r, w = state['case'], state['x'], state['residual'], state['weight']
    if own:
        _package()
        from musc_hip import _layers_hip
        if case['eight']:
            return _layers_hip.rms_norm_quantized(x, w, EPS, residual=r, group=case['group'])
        return _layers_hip.rms_norm(x, w, EPS, residual=r)
    s = x if r is None else (x.float() + r.float()).to(x.dtype)
    s32 = s.float()
    y = s32 * torch.rsqrt(s32.square().mean(-1, keepdim=True) + EPS) * w
    if not case['eight']:
        return y.to(x.dtype) if r is None else (s, y.to(x.dtype))
    # 8-bit values stay what the next product takes: float8 numbers beside their scales
    groups = y.view(y.shape[0], -1, case['group'] or y.shape[1])
    top = groups.abs().amax(-1)
    scales = torch.where(top > 0, top / E4M3_MAX, 1.0)
    y8 = (groups / scales[..., None]).view_as(y).to(torch.float8_e4m3fn)
    return (y8, scales) if r is None else (s, y8, scales)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = {'f32': 4, 'f16': 2, 'bf16': 2}[case['dtype']]
    if case['op'] == 'attention':
        pairs, seen = _pairs(case)
        queries, _ = _tokens(case)
        tq = queries['documents'].numel()
        bytes_ = size * case['dim'] * (2 * tq * case['heads'] + 2 * seen * case['kv_heads'])
        return dict(bytes=bytes_, flops=4 * pairs * case['heads'] * case['dim'])
    if case['op'] == 'rotary':
        frames, rows, columns = (int(x) for x in case['grid'].split(','))
        tokens = case['batch'] * (frames * rows * columns + case['cls'])
        values = tokens * (case['heads'] + case['kv_heads']) * case['dim']
        return dict(bytes=2 * size * values + 12 * tokens, flops=3 * values)
    values = case['rows'] * case['width']
    moved = size * (1 + 2 * case['residual']) + (1 if case['eight'] else size)
    scales = 4 * case['rows'] * (case['width'] // case['group'] if case['group'] else 1) if case['eight'] else 0
    return dict(bytes=values * moved + scales + 4 * case['width'], flops=5 * values)


# --------------------------------------------------------------------------- the definitions in float64
def exact(case, seed):
    state = prepare(case, seed)
    return {'attention': _exact_attention, 'rotary': _exact_rotary, 'norm': _exact_norm}[case['op']](state)


def _exact_attention(state):
    case, q, k, v = state['case'], state['q'], state['k'], state['v']
    qs, ks, group = state['q_side'], state['k_side'], case['heads'] // case['kv_heads']
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b in range(q.shape[0]):
        for first in range(0, q.shape[1], 4096):
            rows = slice(first, first + 4096)
            hidden = qs['documents'][b, rows, None] != ks['documents'][b, None]
            hidden |= ks['documents'][b, None] < 0
            if ks['order'] is not None:
                hidden |= ks['order'][b, None] > qs['order'][b, rows, None]
            live = ~hidden.all(1)
            for h in range(case['heads']):
                logits = torch.mm(q[b, rows, h].double(), k[b, :, h // group].double().T) * state['scale']
                if case['cap']:
                    logits = (logits / case['cap']).tanh() * case['cap']
                if state['slopes'] is not None:
                    for a in range(state['slopes'].shape[1]):
                        gap = torch.sub(qs['positions'][b, rows, a, None].double(), ks['positions'][b, None, :, a].double())
                        logits -= state['slopes'][h, a].double() * gap.abs()
                logits[hidden] = -math.inf
                weights = torch.softmax(logits[live], dim=1)
                out[b, first:first + live.numel(), h][live] = torch.mm(weights, v[b, :, h // group].double())
    return out


def _exact_rotary(state):
    case = state['case']
    place = state['positions'].double()
    radians = torch.stack([place[..., a] * case['base'] ** -e for a, e in zip(*_sections(case))], dim=-1)
    turn = torch.polar(torch.ones_like(radians), radians)[:, :, None]
    n = turn.shape[-1]
    outs = []
    for x in (state['q'].double(), state['k'].double()):
        if case['adjacent']:
            z = torch.view_as_real(torch.complex(x[..., 0:2 * n:2], x[..., 1:2 * n:2]) * turn).flatten(-2)
        else:
            z = torch.complex(x[..., :n], x[..., n:2 * n]) * turn
            z = torch.cat([z.real, z.imag], dim=-1)
        outs.append(torch.cat([z, x[..., 2 * n:]], dim=-1))
    return tuple(outs)


def _exact_norm(state):
    case, x, r = state['case'], state['x'], state['residual']
    total = x.double() if r is None else x.double() + r.double()
    s = total if r is None else total.to(x.dtype).double()
    y = s / (s.pow(2).sum(-1, keepdim=True) / s.shape[-1] + EPS).sqrt() * state['weight'].double()
    head = () if r is None else (total,)
    if not case['eight']:
        return (*head, y) if head else y
    blocks = y.unflatten(-1, (-1, case['group'] or y.shape[-1]))
    scales = blocks.abs().max(-1).values / E4M3_MAX
    return (*head, (blocks / scales.unsqueeze(-1)).flatten(-2), scales)
