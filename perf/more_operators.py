"""More operators of packed and masked encoders, as cases that can be timed and compared.

`run()` computes each of them in elementary torch operations in 32 bits (64 for angles),
or, with `own` set, through musc_hip's public entry points.  `exact()` gives the same
outputs from the definitions in float64.

  window      attention in which query i sees key j of its document when
              order(j) <= order(i) and (order(j) > order(i) - window or order(j) < sinks):
              the last `window` places and the first `sinks` ones; an optional tanh cap on the
              scores and an optional bias by distance; a query that sees no key gets zeros
  prefix      attention of a batch in which every query sees all keys of one shared prefix and
              the keys of its own batch entry that its document and order let it see; queries
              without a document (padding) get zeros
  heads       y = x / sqrt(mean(x^2) + eps) * weight for every head of q and k, then rotation by
              angles position[axis(i)] * base^(-exponent(i)), rounded once
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
EPS = 1e-6


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token for each of eight streams, over a window of a long cache and its first tokens
        dict(name='window_step_bf16', op='window', layout='step', batch=8, cache=32768, shapes=3, window=4096, sinks=4,
             heads=32, kv_heads=8, dim=128, cap=0.0, bias=False, dtype='bf16'),
        # a clip of 24 frames of 16 x 16 patches: each frame sees itself, the three before it and the first one
        dict(name='window_frames_f16', op='window', layout='frames', clips=1, frames=24, side=16, window=4, sinks=1,
             heads=16, kv_heads=16, dim=64, cap=0.0, bias=True, dtype='f16'),
        # one long sequence
        dict(name='window_long_bf16', op='window', layout='text', batch=1, length=8192, shapes=0, window=1024, sinks=4,
             heads=32, kv_heads=8, dim=128, cap=0.0, bias=False, dtype='bf16'),
        # a padded batch of sequences of their own lengths without autocast, scores capped
        dict(name='window_batch_f32', op='window', layout='text', batch=3, length=1500, shapes=7, window=250, sinks=17,
             heads=8, kv_heads=4, dim=80, cap=30.0, bias=False, dtype='f32'),
        # two short requests after a short common beginning: the smallest call
        dict(name='prefix_few_f16', op='prefix', layout='step', prefix=300, batch=2, cache=40, shapes=1, heads=16,
             kv_heads=16, dim=64, cap=0.0, bias=False, dtype='f16'),
        # one new token for each of 32 requests that begin with the same 16384 tokens
        dict(name='prefix_step_bf16', op='prefix', layout='step', prefix=16384, batch=32, cache=700, shapes=2, heads=32,
             kv_heads=8, dim=128, cap=0.0, bias=False, dtype='bf16'),
        # 16 test images of 518 px (37 x 37 patches + class token), each beside the same four reference images
        dict(name='prefix_images_f16', op='prefix', layout='images', prefix=5480, batch=16, length=1370, heads=16,
             kv_heads=16, dim=64, cap=0.0, bias=False, dtype='f16'),
        # the same question asked of a few images in words, without autocast, distance bias and cap
        dict(name='prefix_text_f32', op='prefix', layout='text', prefix=1000, batch=4, length=130, shapes=4, heads=8,
             kv_heads=2, dim=96, cap=20.0, bias=True, dtype='f32'),
        # one new token for each of eight requests, far into their sequences
        dict(name='heads_step_bf16', op='heads', batch=8, grid='1,1,1', cls=False, heads=32, kv_heads=8, dim=128,
             sections='16,24,24', shared=True, adjacent=False, base=1e6, far=200000, each=False, dtype='bf16'),
        # q and k of one encoder batch (four 518 px images, packed projection), angles by row and column
        dict(name='heads_images_f16', op='heads', batch=4, grid='1,37,37', cls=True, heads=16, kv_heads=16, dim=64,
             sections='0,16,16', shared=False, adjacent=False, base=100.0, far=0, each=False, dtype='f16'),
        # a clip of 64 frames of 16 x 16 patches, grouped heads, one row of frequencies over time, height and width
        dict(name='heads_video_bf16', op='heads', batch=1, grid='64,16,16', cls=False, heads=32, kv_heads=8, dim=128,
             sections='16,24,24', shared=True, adjacent=False, base=1e6, far=0, each=False, dtype='bf16'),
        # heads of 72 channels of which 64 turn, a weight for each head, neighbouring channels in pairs, no autocast
        dict(name='heads_odd_f32', op='heads', batch=3, grid='1,29,31', cls=True, heads=12, kv_heads=4, dim=72,
             sections='0,16,16', shared=True, adjacent=True, base=1e4, far=0, each=True, dtype='f32'),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['window', 'prefix', 'heads'])
    dtype = rng.choice(['f16', 'bf16', 'f32'])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    if op == 'heads':
        dim = rng.choice([32, 64, 72, 80, 96, 128])
        pairs = dim // 2 - rng.choice([0, 0, 4])
        t = rng.choice([0, 0, pairs // 4])
        h = (pairs - t) // 2
        frames, rows, columns = (1 if t == 0 else _log(rng, 1, 32)), _log(rng, 1, 40), _log(rng, 1, 40)
        return dict(op=op, batch=rng.randint(1, 4), grid=f'{frames},{rows},{columns}', cls=rng.random() < 0.5,
                    heads=heads, kv_heads=kv_heads, dim=dim, sections=f'{t},{h},{pairs - t - h}',
                    shared=rng.random() < 0.5, adjacent=rng.random() < 0.5, base=rng.choice([100.0, 1e4, 1e6]),
                    far=rng.choice([0, 0, rng.randrange(1 << 18)]), each=rng.random() < 0.3, dtype=dtype)
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=rng.choice([32, 64, 72, 80, 96, 128]),
                cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.4, dtype=dtype,
                shapes=rng.randrange(1 << 20))
    if op == 'window':
        case['layout'] = rng.choice(['text', 'text', 'packed', 'frames', 'step'])
        if case['layout'] == 'frames':
            case.update(clips=rng.randint(1, 2), frames=_log(rng, 1, 24), side=rng.randint(3, 18),
                        window=rng.randint(1, 8), sinks=rng.randint(0, 2))
        else:
            if case['layout'] == 'step':
                case.update(batch=_log(rng, 1, 16), cache=_log(rng, 16, 32768))
            else:
                case.update(batch=rng.randint(1, 4), length=_log(rng, 1, 3000))
            case.update(window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, _log(rng, 1, 200)]))
        return case
    case['layout'] = rng.choice(['step', 'step', 'text', 'images'])
    case['prefix'] = _log(rng, 1, 16384 if case['layout'] == 'step' else 5000)
    if case['layout'] == 'step':
        case.update(batch=_log(rng, 1, 48), cache=_log(rng, 1, 1000))
    else:
        case.update(batch=rng.randint(1, 8), length=_log(rng, 1, 1400))
    return case


# --------------------------------------------------------------------------- layouts of tokens
def _lengths(case):
    """Lengths of a batch's (or packed) sequences, or how far each cache is filled."""
    rng = random.Random(case['shapes'])
    most = case['cache'] if case['layout'] == 'step' else case['length']
    if case['layout'] == 'text' and case['batch'] == 1:
        return [most]
    return [rng.randint(max(1, most // 4), most) for _ in range(case['batch'])]


def _grid_positions(frames, rows, columns):
    axes = torch.meshgrid(torch.arange(frames), torch.arange(rows), torch.arange(columns), indexing='ij')
    return torch.stack([a.reshape(-1) for a in axes], dim=-1).float()


def _tokens(case):
    """The two sides of an attention call (of its own keys): dicts of documents (B, T) int32 or
    None, order (B, T) int32 or None, positions (B or 1, T, A) float32, on the host."""
    layout, start = case['layout'], float(case.get('prefix', 0))
    if layout == 'frames':
        per, n = case['side'] ** 2, case['clips']
        docs = torch.arange(n, dtype=torch.int32).repeat_interleave(case['frames'] * per)[None]
        order = torch.arange(case['frames'], dtype=torch.int32).repeat_interleave(per).repeat(n)[None]
        side = dict(documents=docs, order=order, positions=_grid_positions(case['frames'], case['side'], case['side']).repeat(n, 1)[None])
        return side, side
    if layout == 'images':
        at = torch.arange(case['length']).float()[None, :, None] + start
        side = dict(documents=None, order=None, positions=at)
        return side, side
    lengths = _lengths(case)
    if layout == 'packed':
        order = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths])[None]
        docs = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(lengths)])[None]
        side = dict(documents=docs, order=order, positions=order.float()[..., None])
        return side, side
    b, t = case['batch'], case['cache'] if layout == 'step' else case['length']
    at = torch.arange(t, dtype=torch.int32)[None].expand(b, t).contiguous()
    if layout == 'text':
        docs = torch.where(at < torch.tensor(lengths, dtype=torch.int32)[:, None], 0, -1).to(torch.int32)
        side = dict(documents=docs, order=at, positions=at.float()[..., None] + start)
        return side, side
    last = torch.tensor(lengths, dtype=torch.int32)[:, None] - 1
    keys = dict(documents=torch.zeros_like(at), order=at, positions=at.float()[..., None] + start)
    return dict(documents=torch.zeros_like(last), order=last, positions=last.float()[..., None] + start), keys


def _axes_of(case):
    return 3 if case['layout'] == 'frames' else 1


def _seen_counts(case):
    """(pairs of query and own key that see one another, own keys that some query sees, live queries)"""
    if case['layout'] == 'images':
        n = case['batch'] * case['length']
        return n * case['length'], n, n
    if case['op'] == 'prefix':
        lengths = _lengths(case)
        if case['layout'] == 'step':
            return sum(lengths), sum(lengths), len(lengths)
        return sum(n * (n + 1) // 2 for n in lengths), sum(lengths), sum(lengths)
    w, s = case['window'], case['sinks']

    def places(i):  # that place i sees
        return torch.clamp(i + 1, max=w) + torch.clamp(torch.clamp(i + 1 - w, max=s), min=0)

    if case['layout'] == 'frames':
        per, n = case['side'] ** 2, case['clips']
        tokens = n * case['frames'] * per
        return int(places(torch.arange(case['frames'])).sum()) * per * per * n, tokens, tokens
    lengths = _lengths(case)
    if case['layout'] == 'step':
        seen = sum(int(places(torch.tensor(n - 1))) for n in lengths)
        return seen, seen, len(lengths)
    return sum(int(places(torch.arange(n)).sum()) for n in lengths), sum(lengths), sum(lengths)


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

    return _prepare_heads(case, g, normal) if case['op'] == 'heads' else _prepare_attention(case, g, normal)


def _prepare_attention(case, g, normal):
    queries, keys = _tokens(case)
    q_side, k_side = ({k: v if v is None else v.to(DEV) for k, v in side.items()} for side in (queries, keys))
    if not case['bias']:
        q_side['positions'] = k_side['positions'] = None
    h, hk, d = case['heads'], case['kv_heads'], case['dim']
    b, t = (case['batch'], case['length']) if keys['documents'] is None else keys['documents'].shape
    if queries is keys:  # views of one packed projection, as an encoder block has them
        qkv = normal(b, t, h + 2 * hk, d)
        q, k, v = qkv[:, :, :h], qkv[:, :, h:h + hk], qkv[:, :, h + hk:]
    else:
        q, k, v = normal(b, queries['documents'].shape[1], h, d), normal(b, t, hk, d), normal(b, t, hk, d)
    slopes = None
    if case['bias']:
        slopes = (2.0 ** (-8.0 * torch.arange(1, h + 1, device=DEV) / h))[:, None].expand(h, _axes_of(case)).contiguous()
    state = dict(case=case, q=q, k=k, v=v, q_side=q_side, k_side=k_side, slopes=slopes, scale=2.0 / math.sqrt(d))
    if case['op'] == 'prefix':
        p = case['prefix']
        state.update(prefix_k=normal(p, hk, d), prefix_v=normal(p, hk, d), prefix_positions=None)
        if case['bias']:
            state['prefix_positions'] = torch.arange(p, device=DEV).float()[:, None]
    if own:
        _package()
        from musc_hip._masked_attention_hip import Tokens
        plain = keys['documents'] is None and not case['bias']
        state['keys'] = None if plain else Tokens(**k_side)
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


def _prepare_heads(case, g, normal):
    frames, rows, columns = (int(x) for x in case['grid'].split(','))
    pos = _grid_positions(frames, rows, columns).to(DEV) + float(case['far'])
    if case['cls']:
        pos = torch.cat([torch.zeros((1, 3), device=DEV), pos])
    h, hk, d, b, t = case['heads'], case['kv_heads'], case['dim'], case['batch'], pos.shape[0]
    # each request or image of the batch is somewhere else
    pos = pos[None] + torch.randint(0, 16, (b, 1, 1), generator=g, device=DEV).float()
    # heads of their own sizes, as projections have them before such a norm
    size = torch.exp(torch.randn((1, 1, h + 2 * hk, 1), generator=g, device=DEV))
    qkv = (torch.randn((b, t, h + 2 * hk, d), generator=g, device=DEV) * size).to(DTYPES[case['dtype']])
    axis, exponent = _sections(case)
    weight = lambda n: 1.0 + 0.2 * torch.randn((n, d) if case['each'] else (d,), generator=g, device=DEV)  # noqa: E731
    state = dict(case=case, q=qkv[:, :, :h], k=qkv[:, :, h:h + hk], positions=pos, q_weight=weight(h), k_weight=weight(hk),
                 axis=torch.tensor(axis, device=DEV), exponent=torch.tensor(exponent, dtype=torch.float64, device=DEV))
    if own:
        _package()
        from musc_hip._rotary_hip import RotaryAxes
        state['axes'] = RotaryAxes(d, [int(x) for x in case['sections'].split(',')], base=case['base'],
                                   shared=case['shared'], adjacent=case['adjacent'], device=DEV)
    return state


# --------------------------------------------------------------------------- one pass
def run(state):
    return {'window': _window, 'prefix': _prefix, 'heads': _heads}[state['case']['op']](state)


def _seen(case, q_side, k_side):
    """(B or 1, Tq, Tk) truth values of a call's own keys, or None where all are seen"""
    if k_side['documents'] is None:
        return None
    seen = (q_side['documents'][:, :, None] == k_side['documents'][:, None, :]) & (k_side['documents'] >= 0)[:, None, :]
    if k_side['order'] is not None:
        back = q_side['order'][:, :, None] - k_side['order'][:, None, :]
        seen = seen & (back >= 0)
        if case['op'] == 'window':
            seen = seen & ((back < case['window']) | (k_side['order'] < case['sinks'])[:, None, :])
    return seen


def _softmax_product(case, q, k, v, scale, seen, slopes, q_pos, k_pos):
    """float32 q (B, Tq, H, D), k and v (B, Tk, Hk, D): softmax over the seen keys times v"""
    b, tq, h, d = q.shape
    tk, hk = k.shape[1:3]
    q = q.permute(0, 2, 1, 3).reshape(b, hk, (h // hk) * tq, d)
    s = (q @ k.permute(0, 2, 3, 1).contiguous()).view(b, h, tq, tk) * scale
    if case['cap']:
        s = case['cap'] * torch.tanh(s / case['cap'])
    if slopes is not None:
        apart = (q_pos[:, :, None] - k_pos[:, None]).abs()
        s = s - sum(w[:, None, None] * x[:, None] for w, x in zip(slopes.unbind(1), apart.unbind(-1)))
    if seen is not None:
        s = s.masked_fill(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, -1, tk) @ v.permute(0, 2, 1, 3).contiguous()).view(b, h, tq, d)
    return torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3)


def _window(state):
    case, q, k, v = state['case'], state['q'], state['k'], state['v']
    if own:
        from musc_hip._masked_attention_hip import masked_attention
        return masked_attention(q, k, v, state['scale'], keys=state['keys'], queries=state['queries'], cap=case['cap'],
                                slopes=state['slopes'], window=case['window'], sinks=case['sinks'])
    q_side, k_side = state['q_side'], state['k_side']
    return _softmax_product(case, q.float(), k.float(), v.float(), state['scale'], _seen(case, q_side, k_side),
                            state['slopes'], q_side['positions'], k_side['positions']).to(q.dtype)


def _prefix(state):
    case, q, k, v = state['case'], state['q'], state['k'], state['v']
    pk, pv, pos = state['prefix_k'], state['prefix_v'], state['prefix_positions']
    if own:
        from musc_hip._masked_attention_hip import prefix_attention
        return prefix_attention(q, k, v, pk, pv, state['scale'], keys=state['keys'], queries=state['queries'],
                                cap=case['cap'], slopes=state['slopes'], prefix_positions=pos)
    b, p = k.shape[0], pk.shape[0]
    q_side, k_side = state['q_side'], state['k_side']
    k_all = torch.cat([pk.float()[None].expand(b, -1, -1, -1), k.float()], dim=1)
    v_all = torch.cat([pv.float()[None].expand(b, -1, -1, -1), v.float()], dim=1)
    seen, q_pos, k_pos = _seen(case, q_side, k_side), q_side['positions'], k_side['positions']
    if seen is not None:
        seen = torch.cat([(q_side['documents'] >= 0)[:, :, None].expand(-1, -1, p), seen], dim=2)
    if pos is not None:
        k_pos = torch.cat([pos[None].expand(k_pos.shape[0], -1, -1), k_pos], dim=1)
    return _softmax_product(case, q.float(), k_all, v_all, state['scale'], seen, state['slopes'], q_pos, k_pos).to(q.dtype)


def _heads(state):
    case = state['case']
    if own:
        from musc_hip._rotary_hip import norm_rotary
        return norm_rotary(state['q'], state['k'], state['positions'], state['axes'], state['q_weight'],
                           state['k_weight'], EPS)
    frequency = case['base'] ** -state['exponent']
    angle = state['positions'].double()[..., state['axis']] * frequency  # (B, T, pairs)
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    return tuple(_normed_and_rotated(state[x], state[x + '_weight'], cos, sin, case['adjacent']) for x in 'qk')


def _normed_and_rotated(x, weight, cos, sin, adjacent):
    n = cos.shape[-1]
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight
    if adjacent:
        a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., :n], y[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, y[..., 2 * n:]], dim=-1).to(x.dtype)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = {'f32': 4, 'f16': 2, 'bf16': 2}[case['dtype']]
    if case['op'] == 'heads':
        frames, rows, columns = (int(x) for x in case['grid'].split(','))
        tokens = case['batch'] * (frames * rows * columns + case['cls'])
        values = tokens * (case['heads'] + case['kv_heads']) * case['dim']
        return dict(bytes=2 * size * values + 12 * tokens, flops=7 * values)
    pairs, seen, live = _seen_counts(case)
    if case['op'] == 'prefix':
        pairs, seen = pairs + live * case['prefix'], seen + case['prefix']
    bytes_ = size * case['dim'] * (2 * live * case['heads'] + 2 * seen * case['kv_heads'])
    return dict(bytes=bytes_, flops=4 * pairs * case['heads'] * case['dim'])


# --------------------------------------------------------------------------- the definitions in float64
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_heads(state) if case['op'] == 'heads' else _exact_attention(state)


def _exact_attention(state):
    case, q, slopes = state['case'], state['q'], state['slopes']
    qs, ks, group = state['q_side'], state['k_side'], case['heads'] // case['kv_heads']
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b in range(q.shape[0]):
        of = lambda x: x[b if x.shape[0] > 1 else 0]  # noqa: E731
        for first in range(0, q.shape[1], 4096):
            rows = slice(first, min(first + 4096, q.shape[1]))
            n = rows.stop - first
            hidden = torch.zeros((n, state['k'].shape[1]), dtype=torch.bool, device=q.device)
            live = torch.ones((n,), dtype=torch.bool, device=q.device)
            if ks['documents'] is not None:
                kd, qd = of(ks['documents']), of(qs['documents'])[rows]
                hidden |= (qd[:, None] != kd) | (kd < 0)
                live = qd >= 0
            if ks['order'] is not None:
                ko, qo = of(ks['order']).long(), of(qs['order'])[rows].long()[:, None]
                hidden |= ko > qo
                if case['op'] == 'window':
                    hidden |= (ko <= qo - case['window']) & (ko >= case['sinks'])
            if case['op'] == 'prefix':
                hidden = torch.cat([(~live)[:, None].expand(n, case['prefix']), hidden], dim=1)
            live = ~hidden.all(1)
            for h in range(case['heads']):
                kv = h // group
                kk, vv = state['k'][b, :, kv].double(), state['v'][b, :, kv].double()
                if case['op'] == 'prefix':
                    kk = torch.cat([state['prefix_k'][:, kv].double(), kk])
                    vv = torch.cat([state['prefix_v'][:, kv].double(), vv])
                logits = torch.mm(q[b, rows, h].double(), kk.T) * state['scale']
                if case['cap']:
                    logits = (logits / case['cap']).tanh() * case['cap']
                if slopes is not None:
                    for a in range(slopes.shape[1]):
                        there = of(ks['positions'])[:, a].double()
                        if case['op'] == 'prefix':
                            there = torch.cat([state['prefix_positions'][:, a].double(), there])
                        gap = torch.sub(of(qs['positions'])[rows, a, None].double(), there[None])
                        logits -= slopes[h, a].double() * gap.abs()
                logits[hidden] = -math.inf
                weights = torch.softmax(logits[live], dim=1)
                out[b, rows, h][live] = torch.mm(weights, vv)
    return out


def _exact_heads(state):
    case = state['case']
    place = state['positions'].double()
    radians = torch.stack([place[..., a] * case['base'] ** -e for a, e in zip(*_sections(case))], dim=-1)
    turn = torch.polar(torch.ones_like(radians), radians)[:, :, None]
    n = turn.shape[-1]
    outs = []
    for name in 'qk':
        x = state[name].double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * state[name + '_weight'].double()
        if case['adjacent']:
            z = torch.view_as_real(torch.complex(x[..., 0:2 * n:2], x[..., 1:2 * n:2]) * turn).flatten(-2)
        else:
            z = torch.complex(x[..., :n], x[..., n:2 * n]) * turn
            z = torch.cat([z.real, z.imag], dim=-1)
        outs.append(torch.cat([z, x[..., 2 * n:]], dim=-1))
    return tuple(outs)
