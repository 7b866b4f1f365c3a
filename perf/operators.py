"""The sequence operators of gast_hip.temporal at the sizes they are used with, beside their plain forms in elementary torch operations.

    rotary                 rotation of q and k by their position (half / interleaved pairs, part of the head)
    decay                  causal linear attention with a decay for each head: forward, or forward and gradients
    decay_step             the same for ONE new token of every stream, on a state that stays on the device
    norm                   layer norm, alone or of residual + dropout(branch): forward, or forward and gradients

A sequence belongs to one joint of one clip, as everywhere in this framework: tensors are (B, T, J, H, D), J = 1 for plain token sequences."""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


def listed():
    return [
        # one frame of a causal stream: q and k of 17 joints, 4 heads of 32 channels (128 channels): latency
        dict(name='rotary, one frame', op='rotary', dtype='fp32', B=1, T=1, J=17, Hq=4, Hk=4, D=32, R=32, layout='half', far=100000, train=False),
        # a long prompt with shared key heads, half of each head rotated, trained at far positions
        dict(name='rotary, long, gradients', op='rotary', dtype='bf16', B=1, T=16384, J=1, Hq=32, Hk=8, D=128, R=64, layout='interleaved',
             far=1000000, train=True),
        # inference over one clip of 243 frames
        dict(name='decay, one clip', op='decay', dtype='fp32', B=1, T=243, J=17, H=4, Dk=32, Dv=32, ragged=False, state=False, train=False),
        # training on the default windows: 128 windows of 27 frames, 17 joints, 128 channels
        dict(name='decay, windows, gradients', op='decay', dtype='fp32', B=128, T=27, J=17, H=4, Dk=32, Dv=32, ragged=False, state=False, train=True),
        # training on long sequences
        dict(name='decay, long, gradients', op='decay', dtype='bf16', B=2, T=4096, J=1, H=16, Dk=64, Dv=64, ragged=False, state=False, train=True),
        # a batch of clips of different lengths (an empty one among them), uneven heads, going on from a state and returning the next one
        dict(name='decay, ragged, gradients', op='decay', dtype='fp16', B=6, T=1003, J=5, H=3, Dk=48, Dv=80, ragged=True, state=True, train=True),
        # one very long prompt: few sequences, so the time axis has to be split
        dict(name='decay, prompt', op='decay', dtype='bf16', B=1, T=32768, J=1, H=16, Dk=128, Dv=128, ragged=False, state=True, train=False),
        # one frame of one causal stream
        dict(name='decay step, one frame', op='decay_step', dtype='fp32', B=1, J=17, H=4, Dk=32, Dv=32, ragged=False),
        # a full serving batch, some of whose streams have no new token
        dict(name='decay step, full batch', op='decay_step', dtype='bf16', B=256, J=1, H=32, Dk=128, Dv=128, ragged=True),
        # the norm of one frame
        dict(name='norm, one frame', op='norm', dtype='fp32', rows=17, C=128, p=0.0, add=False, train=False),
        # the norm of a training batch of windows (128 x 27 x 17 rows)
        dict(name='norm, windows, gradients', op='norm', dtype='fp32', rows=58752, C=128, p=0.0, add=False, train=True),
        # a wide residual stream with dropout on the branch
        dict(name='add + norm, wide, gradients', op='norm', dtype='bf16', rows=8192, C=4096, p=0.1, add=True, train=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['rotary', 'decay', 'decay', 'decay_step', 'norm', 'norm'])
    dtype = rng.choice(['fp32', 'bf16', 'fp16'])
    if op == 'rotary':
        J = rng.choice([1, 1, 15, 17])
        Hk = rng.choice([1, 2, 4, 8])
        Hq = Hk * rng.choice([1, 1, 2, 4])
        D = 2 * _log(rng, 4, 64)
        R = D if rng.random() < 0.5 else 2 * rng.randint(1, D // 2)
        rows = _log(rng, 1, max(1, (64 << 20) // (D * (Hq + Hk) * J)))
        B = _log(rng, 1, min(rows, 64))
        return dict(op=op, dtype=dtype, B=B, T=max(1, rows // B), J=J, Hq=Hq, Hk=Hk, D=D, R=R, layout=rng.choice(['half', 'interleaved']),
                    far=_log(rng, 1, 2000000), train=rng.random() < 0.5)
    if op == 'decay':
        J = rng.choice([1, 1, 15, 17])
        H = rng.choice([1, 2, 4, 8, 16])
        Dk = rng.choice([16, 32, 64, 128, rng.randint(8, 128)])
        Dv = Dk if rng.random() < 0.6 else rng.choice([32, 64, 128, rng.randint(8, 128)])
        train = rng.random() < 0.5
        tokens = _log(rng, 64, (32 << 20) // (H * max(Dk, Dv)) // (4 if train else 1) // J)
        B = _log(rng, 1, min(tokens, 64, max(1, (12 << 20) // (J * H * Dk * Dv))))          # (bounds the states: they are held in 32 bits)
        return dict(op=op, dtype=dtype, B=B, T=max(1, tokens // B), J=J, H=H, Dk=Dk, Dv=Dv, ragged=rng.random() < 0.4, state=rng.random() < 0.5, train=train)
    if op == 'decay_step':
        J = rng.choice([1, 1, 15, 17])
        H = rng.choice([1, 2, 4, 8, 32])
        Dk = rng.choice([16, 32, 64, 128, rng.randint(8, 128)])
        Dv = Dk if rng.random() < 0.6 else rng.choice([32, 64, 128, rng.randint(8, 128)])
        return dict(op=op, dtype=dtype, B=_log(rng, 1, max(1, (120 << 20) // (J * H * Dk * Dv))), J=J, H=H, Dk=Dk, Dv=Dv, ragged=rng.random() < 0.4)
    C = _log(rng, 8, 8192)
    add = rng.random() < 0.5
    return dict(op=op, dtype=dtype, rows=_log(rng, 1, (30 << 20) // C), C=C, p=rng.choice([0.0, 0.1, 0.25]) if add else 0.0, add=add, train=rng.random() < 0.6)


# ------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """What the case works on, as a dict of tensors on the GPU, made from the seed alone."""
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case['dtype']]

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    s = {}
    if case['op'] == 'rotary':
        B, T, J, D, R = (case[k] for k in ('B', 'T', 'J', 'D', 'R'))
        s['q'], s['k'] = normal(B, T, J, case['Hq'], D), normal(B, T, J, case['Hk'], D)
        # every clip goes on from a place of its own
        first = torch.randint(0, case['far'], (B, 1), generator=g, device=dev)
        s['positions'] = first + torch.arange(T, device=dev)
        s['freqs'] = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=dev) / R)
        if case['train']:
            s['dq'], s['dk'] = normal(B, T, J, case['Hq'], D), normal(B, T, J, case['Hk'], D)
    elif case['op'] in ('decay', 'decay_step'):
        B, J, H, Dk, Dv = (case[k] for k in ('B', 'J', 'H', 'Dk', 'Dv'))
        lead = (B, case['T'], J, H) if case['op'] == 'decay' else (B, J, H)
        s['q'], s['k'], s['v'] = normal(*lead, Dk), normal(*lead, Dk), normal(*lead, Dv)
        # the decays that a stack of heads is given: from 31 / 32 to 1 - 2^-12 a token
        s['log_decay'] = torch.log1p(-torch.exp2(-5.0 - 7.0 * torch.arange(H, device=dev, dtype=torch.float64) / max(1, H - 1))).float()
        s['lengths'] = None
        if case['ragged']:
            most = case.get('T', 1)
            s['lengths'] = torch.randint(0, most + 1, (B,), generator=g, device=dev, dtype=torch.int32)
            s['lengths'][0] = most
            if B > 1:
                s['lengths'][1] = 0
        s['state'] = normal(B, J, H, Dk, Dv, dtype=torch.float32, scale=4.0) if case.get('state', True) else None
        if case.get('train'):
            s['do'] = normal(*lead, Dv)
            s['dstate'] = normal(B, J, H, Dk, Dv, dtype=torch.float32) if case['state'] else None
    else:
        rows, C = case['rows'], case['C']
        s['x'] = normal(rows, C)
        s['residual'] = normal(rows, C, scale=2.0) if case['add'] else None
        s['weight'] = normal(C, dtype=torch.float32, scale=0.1) + 1.0
        s['bias'] = normal(C, dtype=torch.float32, scale=0.1)
        s['seed'] = torch.randint(1, 2 ** 31 - 1, (1,), generator=g, device=dev, dtype=torch.int32)
        if case['train']:
            s['dy'] = normal(rows, C)
            s['ds'] = normal(rows, C) if case['add'] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s['case'] = case
    if case.get('train'):
        for name in ('q', 'k', 'v', 'state', 'x', 'residual', 'weight', 'bias'):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _rotated(x, positions, freqs, layout):
    R = 2 * freqs.numel()
    angle = positions.double().unsqueeze(-1) * freqs              # (B, T, R / 2), in 64 bits: positions go far
    cos, sin = (f(angle).float()[:, :, None, None] for f in (torch.cos, torch.sin))
    xf = x.float()
    if layout == 'half':
        a, b = xf[..., :R // 2], xf[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    else:
        a, b = xf[..., 0:R:2], xf[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([turned, xf[..., R:]], dim=-1).to(x.dtype)


def _decay_plain(q, k, v, log_decay, state, lengths):
    """o_t = scale q_t S_t, S_t = exp(log_decay) S_(t-1) + k_t v_t, by chunks of C tokens: inside a chunk as a product of matrices,
    from chunk to chunk by the sums of k v of each.  Tokens from `lengths` on are not there."""
    B, T, J, H, Dk = q.shape
    Dv = v.shape[-1]
    dev = q.device
    C = min(T, 128)
    n = -(-T // C)
    length = torch.full((B,), T, device=dev) if lengths is None else lengths.long()
    there = (torch.arange(T, device=dev) < length[:, None]).float()                            # (B, T)

    def chunks(x):                                                                             # -> (B, J, H, n, C, D)
        x = torch.nn.functional.pad(x.float() * there[:, :, None, None, None], (0, 0, 0, 0, 0, 0, 0, n * C - T))
        return x.view(B, n, C, J, H, -1).permute(0, 3, 4, 1, 2, 5).contiguous()

    Q, K, V = chunks(q) * Dk ** -0.5, chunks(k), chunks(v)
    g = log_decay.double()
    i = torch.arange(C, device=dev)
    gap = i[:, None] - i
    inside = torch.where(gap >= 0, torch.exp(g[:, None, None] * gap.clamp(min=0)), 0.0).float()[:, None]     # (H, 1, C, C)
    o = torch.matmul(torch.matmul(Q, K.transpose(-1, -2).contiguous()) * inside, V)
    later = torch.exp(g[:, None] * (C - 1 - i)).float()[:, None, :, None]                                    # (H, 1, C, 1)
    sums = torch.matmul((K * later).transpose(-1, -2).contiguous(), V)                                       # (B, J, H, n, Dk, Dv)
    c = torch.arange(n, device=dev)
    gap = c[:, None] - 1 - c
    carry = torch.where(gap >= 0, torch.exp(g[:, None, None] * C * gap.clamp(min=0)), 0.0).float()           # (H, n, n)
    before = torch.matmul(carry, sums.flatten(-2)).unflatten(-1, (Dk, Dv))
    if state is not None:
        before = before + torch.exp(g[:, None] * C * c).float()[:, :, None, None] * state[:, :, :, None]
    o = o + torch.matmul(Q * torch.exp(g[:, None] * (i + 1)).float()[:, None, :, None], before)
    o = o.permute(0, 3, 4, 1, 2, 5).reshape(B, n * C, J, H, Dv)[:, :T]
    # the state behind each sequence's last token
    t = torch.arange(n * C, device=dev)
    left = (length[:, None] - 1 - t).clamp(min=0)                                                            # (B, n C)
    w = torch.exp(g[None, :, None] * left[:, None]).float()[:, None, :, :, None]                             # (B, 1, H, n C, 1)
    new = torch.matmul((K.flatten(3, 4) * w).transpose(-1, -2).contiguous(), V.flatten(3, 4))
    if state is not None:
        new = new + torch.exp(g * length[:, None]).float()[:, None, :, None, None] * state
    return o.to(q.dtype), new


def _hash32(x):
    m = 0xffffffff
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & m
    x = x ^ (x >> 15)
    x = (x * 0x846ca68b) & m
    return x ^ (x >> 16)


def _keep(case, seed):
    """(rows, C) multipliers of the library's dropout stream: 0, or 1 / (1 - p) with p in 65536ths"""
    thresh = int(round(case['p'] * 65536))
    e = torch.arange(case['rows'] * case['C'], device=seed.device).view(case['rows'], case['C'])
    key = (seed.long() * 0x9E3779B9) & 0xffffffff
    h = _hash32(((e >> 1) ^ key) & 0xffffffff)
    bits = torch.where((e & 1) == 1, h >> 16, h & 0xffff)
    return torch.where(bits >= thresh, 65536.0 / (65536 - thresh), 0.0).float()


def _norm_plain(s):
    case, x = s['case'], s['x']
    stream = x
    if case['add']:
        branch = x.double()                                            # (64 bits: a sum next to the border of two 16-bit values)
        if case['p'] > 0:
            branch = branch * _keep(case, s['seed'])
        total = s['residual'].double() + branch
        # what the next layer reads, and the norm is of these stored values; the rounding passes gradients on unchanged
        stream = total + (total.detach().to(x.dtype).double() - total.detach())
    f = stream.float()
    mean = f.mean(dim=-1, keepdim=True)
    centred = f - mean
    rstd = torch.rsqrt((centred * centred).mean(dim=-1, keepdim=True) + 1e-5)
    y = (centred * rstd * s['weight'] + s['bias']).to(x.dtype)
    return y, stream.to(x.dtype)


# ------------------------------------------------------------------------------------------------ one pass
def _temporal():
    """gast_hip.temporal, the package's folder put on the path as its users do"""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'gast-net-3dposeestimation_amd')
    if at not in sys.path:
        sys.path.insert(0, at)
    import gast_hip.temporal
    return gast_hip.temporal


def _own_norm(s):
    ops, case = _temporal(), s['case']
    if not case['add']:
        return ops.layer_norm(s['x'], s['weight'], s['bias'], eps=1e-5), None
    from gast_hip.binding import Dropout, dropout_params
    drop = Dropout(s['seed'], *dropout_params(case['p'])) if case['p'] > 0 else None
    return ops.add_layer_norm(s['x'], s['residual'], s['weight'], s['bias'], eps=1e-5, drop=drop)


def run(state):
    s, case = state, state['case']
    if case['op'] == 'rotary':
        if own:
            q, k = _temporal().rotary((s['q'], s['k']), s['positions'], s['freqs'], interleaved=case['layout'] == 'interleaved')
        else:
            q, k = (_rotated(s[n], s['positions'], s['freqs'], case['layout']) for n in ('q', 'k'))
        out = {'q': q, 'k': k}
        if case['train']:
            out['dq'], out['dk'] = torch.autograd.grad([q, k], [s['q'], s['k']], [s['dq'], s['dk']])
        return _detached(out)
    if case['op'] == 'decay':
        if own:
            got = _temporal().decay_attention(s['q'], s['k'], s['v'], s['log_decay'], state=s['state'], lengths=s['lengths'],
                                              return_state=case['state'])
            o, new = got if case['state'] else (got, None)
        else:
            o, new = _decay_plain(s['q'], s['k'], s['v'], s['log_decay'], s['state'], s['lengths'])
        out = {'o': o}
        if case['state']:
            out['state'] = new
        if case['train']:
            leaves, outs, grads = ['q', 'k', 'v'], [o], [s['do']]
            if case['state']:
                leaves, outs, grads = leaves + ['state'], outs + [new], grads + [s['dstate']]
            for name, d in zip(leaves, torch.autograd.grad(outs, [s[n] for n in leaves], grads)):
                out['d' + name] = d
        return _detached(out)
    if case['op'] == 'decay_step':
        if own:
            return {'o': _temporal().decay_attention_step(s['q'], s['k'], s['v'], s['log_decay'], s['state'], lengths=s['lengths']), 'state': s['state']}
        there = torch.ones_like(s['q'][:, 0, 0, 0], dtype=torch.float32) if s['lengths'] is None else s['lengths'].clamp(0, 1).float()
        there = there[:, None, None, None, None]
        new = torch.exp(s['log_decay'])[:, None, None] * s['state'] + s['k'].float().unsqueeze(-1) * s['v'].float().unsqueeze(-2)
        s['state'].copy_(torch.where(there > 0, new, s['state']))
        o = torch.matmul((s['q'].float() * case['Dk'] ** -0.5).unsqueeze(-2), s['state']) * there
        return {'o': o.squeeze(-2).to(s['q'].dtype), 'state': s['state']}
    y, stream = _own_norm(s) if own else _norm_plain(s)
    out = {'y': y}
    if case['add']:
        out['stream'] = stream
    if case['train']:
        leaves, outs, grads = ['x', 'weight', 'bias'], [y], [s['dy']]
        if case['add']:
            leaves, outs, grads = leaves + ['residual'], outs + [stream], grads + [s['ds']]
        for name, d in zip(leaves, torch.autograd.grad(outs, [s[n] for n in leaves], grads)):
            out['d' + name] = d
    return _detached(out)


def _detached(out):
    return {k: v.detach() for k, v in out.items()}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    es = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'rotary':
        rows = case['B'] * case['T'] * case['J']
        values = rows * (case['Hq'] + case['Hk']) * case['D']
        part = case['R'] / case['D']
        times = 2 if case['train'] else 1
        return {'bytes': 2.0 * values * es * times + 8 * case['B'] * case['T'], 'flops': 3.0 * values * part * times}
    if case['op'] == 'decay':
        heads = case['B'] * case['J'] * case['H']
        rows = heads * case['T']
        Dk, Dv = case['Dk'], case['Dv']
        once = (2 * Dk + 2 * Dv) * es
        states = 2.0 * heads * Dk * Dv * 4 if case['state'] else 0.0
        if not case['train']:      # S and q S of the recurrence
            return {'bytes': rows * once + states, 'flops': 4.0 * rows * Dk * Dv}
        # + dq of S, the recurrence of dS, and dk, dv of it; q, k, v, do are read, o, dq, dk, dv written
        return {'bytes': 2.0 * rows * once + 2 * states, 'flops': 12.0 * rows * Dk * Dv}
    if case['op'] == 'decay_step':
        heads = case['B'] * case['J'] * case['H']
        Dk, Dv = case['Dk'], case['Dv']
        return {'bytes': heads * (8.0 * Dk * Dv + (2 * Dk + 2 * Dv) * es), 'flops': 5.0 * heads * Dk * Dv}
    values = case['rows'] * case['C']
    tensors = 4 if case['add'] else 2                                        # x, y (+ residual, stream)
    flops = 8.0 * values
    if case['train']:
        tensors += 4 if case['add'] else 2                                   # dy, dx (+ d stream, d residual)
        flops += 14.0 * values
    return {'bytes': float(tensors) * values * es + 8.0 * case['C'] * (2 if case['train'] else 1), 'flops': flops}


# ------------------------------------------------------------------------------------------------ in 64 bits, from the definitions
def _exact_rotary(case, s):
    def turn(x, sign):
        x = x.detach().double()
        R = case['R']
        angle = sign * s['positions'].double()[..., None] * s['freqs']
        z = torch.polar(torch.ones_like(angle), angle)[:, :, None, None]
        head = x[..., :R]
        pair = head.unflatten(-1, (2, R // 2)).transpose(-1, -2) if case['layout'] == 'half' else head.unflatten(-1, (R // 2, 2))
        w = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
        w = (w.transpose(-1, -2) if case['layout'] == 'half' else w).flatten(-2)
        return torch.cat([w, x[..., R:]], dim=-1)
    out = {'q': turn(s['q'], 1), 'k': turn(s['k'], 1)}
    if case['train']:        # a rotation's transpose is the rotation back
        out['dq'], out['dk'] = turn(s['dq'], -1), turn(s['dk'], -1)
    return out


def _exact_decay(case, s):
    """Row blocks of the T x T matrix of scores, head by head: o = (scale q k' o W) v with W_ts = exp(log_decay (t - s)) for s <= t, and
    the derivatives of that, written out."""
    B, T, J, H, Dk, Dv = (case[k] for k in ('B', 'T', 'J', 'H', 'Dk', 'Dv'))
    dev = s['q'].device
    scale = Dk ** -0.5
    train = case['train']
    names = ['q', 'k', 'v'] + (['do'] if train else [])
    x = {n: s[n].detach().double().permute(3, 0, 2, 1, 4).reshape(H, B * J, T, -1) for n in names}          # (H, B J, T, D)
    length = torch.full((B,), T, device=dev) if s['lengths'] is None else s['lengths'].long()
    length = length[:, None].expand(B, J).reshape(-1)
    t = torch.arange(T, device=dev)
    there = (t < length[:, None]).double()[..., None]                                                       # (B J, T, 1)
    S0 = s['state'].detach().double().permute(2, 0, 1, 3, 4).reshape(H, B * J, Dk, Dv) if case['state'] else None
    dS = s['dstate'].double().permute(2, 0, 1, 3, 4).reshape(H, B * J, Dk, Dv) if case['state'] and train else None
    res = {n: torch.zeros(H, B * J, T, d, dtype=torch.float64, device=dev) for n, d in (('o', Dv),) + ((('dq', Dk), ('dk', Dk), ('dv', Dv)) if train else ())}
    new = torch.zeros(H, B * J, Dk, Dv, dtype=torch.float64, device=dev)
    dS0 = torch.zeros_like(new)
    block = max(1, min(T, (1 << 28) // T))
    group = max(1, (1 << 28) // (block * T))
    for h in range(H):
        g = s['log_decay'][h].double()
        for n0 in range(0, B * J, group):
            at = slice(n0, n0 + group)
            q, k, v = (x[n][h, at] * there[at] for n in ('q', 'k', 'v'))
            do = x['do'][h, at] * there[at] if train else None
            for r in range(0, T, block):
                rows, cols = slice(r, min(T, r + block)), slice(0, min(T, r + block))
                gap = t[rows, None] - t[cols]
                W = torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), 0.0) * scale
                P = torch.matmul(q[:, rows], k[:, cols].transpose(-1, -2).contiguous()) * W
                res['o'][h, at, rows] = torch.matmul(P, v[:, cols])
                if train:
                    res['dv'][h, at, cols] += torch.matmul(P.transpose(-1, -2).contiguous(), do[:, rows])
                    dP = torch.matmul(do[:, rows], v[:, cols].transpose(-1, -2).contiguous()) * W
                    res['dq'][h, at, rows] = torch.matmul(dP, k[:, cols])
                    res['dk'][h, at, cols] += torch.matmul(dP.transpose(-1, -2).contiguous(), q[:, rows])
            left = torch.exp(g * (length[at, None] - 1 - t).clamp(min=0))[..., None] * there[at]             # to the last token
            new[h, at] = torch.matmul((k * left).transpose(-1, -2).contiguous(), v)
            if S0 is not None:
                gone = torch.exp(g * (t + 1))[:, None] * there[at]
                whole = torch.exp(g * length[at])[:, None, None]
                new[h, at] += whole * S0[h, at]
                res['o'][h, at] += scale * torch.matmul(q * gone, S0[h, at])
                if train:
                    res['dq'][h, at] += scale * torch.matmul(do * gone, S0[h, at].transpose(-1, -2).contiguous())
                    res['dk'][h, at] += torch.matmul(v * left, dS[h, at].transpose(-1, -2).contiguous())
                    res['dv'][h, at] += torch.matmul(k * left, dS[h, at])
                    dS0[h, at] = scale * torch.matmul((q * gone).transpose(-1, -2).contiguous(), do) + whole * dS[h, at]

    def back(y):
        return y.view(H, B, J, T, -1).permute(1, 3, 2, 0, 4).contiguous()

    def back_state(y):
        return y.view(H, B, J, Dk, Dv).permute(1, 2, 0, 3, 4).contiguous()

    out = {'o': back(res['o'])}
    if case['state']:
        out['state'] = back_state(new)
    if train:
        out.update({n: back(res[n]) for n in ('dq', 'dk', 'dv')})
        if case['state']:
            out['dstate'] = back_state(dS0)
    return out


def _exact_step(case, s):
    q, k, v = (s[n].double() for n in ('q', 'k', 'v'))
    S = s['state'].double()
    moved = S * torch.exp(s['log_decay'].double()).view(1, 1, -1, 1, 1) + torch.einsum('bjhd,bjhe->bjhde', k, v)
    o = torch.einsum('bjhd,bjhde->bjhe', q, moved) * case['Dk'] ** -0.5
    if s['lengths'] is not None:
        on = (s['lengths'] >= 1).view(-1, 1, 1, 1)
        o, moved = o * on, torch.where(on.unsqueeze(-1), moved, S)
    return {'o': o, 'state': moved}


def _exact_keep(case, seed):
    """The dropout stream on the host, in unsigned 32-bit words: two elements share a word, the even one has its low half."""
    u = np.uint32
    n = case['rows'] * case['C']
    thresh = round(case['p'] * 65536)
    key = u(int(seed.item()) * 0x9E3779B9 % 2 ** 32)
    h = np.arange((n + 1) // 2, dtype=u) ^ key
    for shift, factor in ((16, 0x7feb352d), (15, 0x846ca68b)):
        h ^= h >> u(shift)
        h *= u(factor)
    h ^= h >> u(16)
    kept = h.view(np.uint16)[:n] >= thresh
    factor = np.float32(65536.0 / (65536 - thresh))
    return torch.from_numpy(kept).to(seed.device).view(case['rows'], case['C']).double() * float(factor)


def _exact_norm(case, s):
    x, w, b = s['x'].detach(), s['weight'].detach().double(), s['bias'].detach().double()
    keep = None
    stream = x
    if case['add']:
        keep = _exact_keep(case, s['seed']) if case['p'] > 0 else torch.ones_like(x, dtype=torch.float64)
        stream = (s['residual'].detach().double() + x.double() * keep).to(x.dtype)
    f = stream.double()
    var, mean = torch.var_mean(f, dim=-1, keepdim=True, correction=0)
    rstd = 1.0 / torch.sqrt(var + 1e-5)
    xhat = (f - mean) * rstd
    out = {'y': xhat * w + b}
    if case['add']:
        out['stream'] = stream.double()
    if case['train']:
        dy = s['dy'].double()
        out['dweight'], out['dbias'] = (dy * xhat).sum(0), dy.sum(0)
        gr = dy * w
        df = rstd * (gr - gr.mean(-1, keepdim=True) - xhat * (gr * xhat).mean(-1, keepdim=True))
        if case['add']:
            df = df + s['ds'].double()
            out['dresidual'] = df
            df = df * keep
        out['dx'] = df
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    with torch.no_grad():
        return {'rotary': _exact_rotary, 'decay': _exact_decay, 'decay_step': _exact_step, 'norm': _exact_norm}[case['op']](case, s)
