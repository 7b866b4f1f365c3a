"""Sequence operators along the frame axis: rotary positions, causal linear attention with a decay for each head (whole sequences, and
one frame at a time on a state), layer norm with an optional dropped-out branch.

They stand beside the path's own attention over joints, BatchNorm and dropout for models that look further back than the receptive
field of the dilated convolutions: `model/temporal_attention.py` builds its block of them, and its frame-at-a-time form.  The kernels are
csrc/rotary.hip, csrc/decay_attn.hip and csrc/layer_norm.hip.

Tensors are (B, T, J, H, D) -- a sequence belongs to one joint of one clip, H heads of D channels -- or (B, T, H, D) for plain token
sequences; any strides, as long as a head's D values are contiguous (other tensors are copied first).  fp32, bfloat16 and float16; all of a
call's activations have one type.  Everything is enqueued on the current stream of the tensors' device; there is no CPU fallback.
"""
import torch

from gast_hip.binding import DECAY_MAX_D, ROTARY_MAX_BATCH, ROTARY_MAX_D

_OPS = None
_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _ops():
    global _OPS
    if _OPS is None:
        from gast_hip.binding import HipOps
        _OPS = HipOps()
    return _OPS


def _on_device(what, t, *others):
    """the checks that need the tensors themselves; every tensor on one HIP device"""
    if t.dtype not in _TYPES:
        raise ValueError('%s: float32, bfloat16 or float16 tensors, got %s' % (what, t.dtype))
    if not t.is_cuda:
        raise RuntimeError('%s: tensors are on %s; the HIP path needs device tensors (no CPU fallback)' % (what, t.device))
    for o in others:
        if o is not None and o.device != t.device:
            raise RuntimeError('%s: tensors on %s and %s' % (what, t.device, o.device))


def _heads(what, name, t):
    """(B, T, J, H, D) view of a (B, T, J, H, D) or (B, T, H, D) tensor with contiguous channels"""
    if t.dim() == 4:
        t = t.unsqueeze(2)
    elif t.dim() != 5:
        raise ValueError('%s: %s has to be (B, T, J, H, D) or (B, T, H, D), got %s' % (what, name, tuple(t.shape)))
    if 0 in t.shape[2:]:
        raise ValueError('%s: %s has an empty axis: %s' % (what, name, tuple(t.shape)))
    return t if t.stride(4) == 1 or t.shape[4] == 1 else t.contiguous()


# ------------------------------------------------------------------------------------------------ rotary positions
def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, low=1.0, high=32.0, length=None, device=None):
    """Angles per position of the dim / 2 channel pairs, float64: base ** (-2 f / dim), for longer contexts stretched by `factor`:
      scaling 'linear'   every frequency / factor (positions are interpolated)
      scaling 'base'     base * factor ** (dim / (dim - 2)): the slowest pair is stretched by `factor`, the fastest not at all
      scaling 'bands'    pairs that turn fewer than `low` times over `length` positions are stretched, those that turn more than `high`
                         times are kept, between them a straight blend over the number of turns
    """
    if dim < 2 or dim % 2:
        raise ValueError('rotary_frequencies: dim has to be even and positive, got %r' % (dim,))
    if scaling not in (None, 'linear', 'base', 'bands'):
        raise ValueError("rotary_frequencies: scaling is None, 'linear', 'base' or 'bands', got %r" % (scaling,))
    if not base > 0 or not factor > 0:
        raise ValueError('rotary_frequencies: base and factor have to be positive, got %r and %r' % (base, factor))
    if scaling == 'base' and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == 'linear':
        f = f / factor
    elif scaling == 'bands':
        if length is None or not high > low:
            raise ValueError("rotary_frequencies: scaling 'bands' needs length and low < high")
        turns = f * (length / 6.283185307179586)
        kept = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        f = f * kept + f / factor * (1.0 - kept)
    return f.to(device) if device is not None else f


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, freqs, interleaved, scale, *xs):
        ys = tuple(torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs)
        _rotate(xs, ys, positions, freqs, interleaved, scale, False)
        ctx.save_for_backward(positions, freqs)
        ctx.how = interleaved, scale
        return ys

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *dys):
        positions, freqs = ctx.saved_tensors
        interleaved, scale = ctx.how
        want = [i for i in range(len(dys)) if ctx.needs_input_grad[4 + i]]
        dxs = [None] * len(dys)
        if want:
            src = [dys[i] if dys[i].stride(4) == 1 else dys[i].contiguous() for i in want]
            out = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in src]
            _rotate(src, out, positions, freqs, interleaved, scale, True)
            for i, o in zip(want, out):
                dxs[i] = o
        return (None, None, None, None) + tuple(dxs)


def _rotate(xs, ys, positions, freqs, interleaved, scale, backward):
    if xs[0].numel() == 0:
        return
    with torch.cuda.device(xs[0].device):
        _ops().rotary_multi(list(zip(xs, ys)), positions, freqs, 2 * freqs.shape[0], interleaved, scale, backward)


def rotary(x, positions, freqs, interleaved=False, scale=1.0):
    """x with the first 2 * len(freqs) channels of every head turned by positions * freqs and multiplied by `scale`, the others as they
    are.  x: one tensor, or a tuple of up to four (q and k, say, with heads of their own) that are turned in one launch.  Pairs are
    channels (f, f + len(freqs)), or (2 f, 2 f + 1) with interleaved=True.  positions: (T,) for all clips or (B, T), int32 or int64, any
    values (angles are reduced in 64 bits).  Differentiable in x."""
    xs = tuple(x) if isinstance(x, (tuple, list)) else (x,)
    if not 1 <= len(xs) <= ROTARY_MAX_BATCH:
        raise ValueError('rotary: 1 to %d tensors in a call, got %d' % (ROTARY_MAX_BATCH, len(xs)))
    shapes = [t.shape for t in xs]
    xs = tuple(_heads('rotary', 'x', t) for t in xs)
    B, T, J, _, D = xs[0].shape
    for t in xs[1:]:
        if t.shape[:3] != xs[0].shape[:3] or t.shape[4] != D or t.dtype != xs[0].dtype:
            raise ValueError('rotary: tensors of one call differ in their heads alone, got %s %s and %s %s'
                             % (tuple(xs[0].shape), xs[0].dtype, tuple(t.shape), t.dtype))
    if freqs.dim() != 1 or freqs.dtype != torch.float64 or not 1 <= freqs.shape[0] <= D // 2:
        raise ValueError('rotary: freqs is a float64 vector of 1 to %d frequencies, got %s %s' % (D // 2, freqs.dtype, tuple(freqs.shape)))
    if D > ROTARY_MAX_D:
        raise ValueError('rotary: at most %d channels a head, got %d' % (ROTARY_MAX_D, D))
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError('rotary: positions are int32 or int64, got %s' % positions.dtype)
    if tuple(positions.shape) == (T,):
        positions = positions.unsqueeze(0)
    elif tuple(positions.shape) not in ((B, T), (1, T)):
        raise ValueError('rotary: positions have to be (%d,) or (%d, %d), got %s' % (T, B, T, tuple(positions.shape)))
    _on_device('rotary', xs[0], *xs[1:], positions, freqs)
    ys = _Rotary.apply(positions, freqs.contiguous(), bool(interleaved), float(scale), *xs)
    ys = tuple(y.view(s) for y, s in zip(ys, shapes))
    return ys if isinstance(x, (tuple, list)) else ys[0]


# ------------------------------------------------------------------------------------------------ linear attention with a decay
class _Decay(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale, want_state):
        B, T, J, H, Dk = q.shape
        Dv = v.shape[4]
        o = torch.empty(B, T, J, H, Dv, dtype=q.dtype, device=q.device)
        new = torch.empty(B, J, H, Dk, Dv, dtype=torch.float32, device=q.device) if want_state else None
        if B * T > 0:
            with torch.cuda.device(q.device):
                _ops().decay_fwd(q, k, v, log_decay, lengths, scale, state, o, new)
        elif new is not None:
            new.zero_() if state is None else new.copy_(state)
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, new

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dnew):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        B, T, J, H, Dk = q.shape
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        dstate = torch.empty_like(state) if ctx.needs_input_grad[4] else None
        if dnew is not None:
            dnew = dnew.contiguous()
        if B * T > 0:
            if do is None:
                do = torch.zeros(B, T, J, H, v.shape[4], dtype=q.dtype, device=q.device)
            elif do.stride(4) != 1:
                do = do.contiguous()
            with torch.cuda.device(q.device):
                _ops().decay_bwd(q, k, v, log_decay, lengths, ctx.scale, state, do, dnew, dq, dk, dv, dstate)
        elif dstate is not None:
            dstate.zero_() if dnew is None else dstate.copy_(dnew)
        return dq, dk, dv, None, dstate, None, None, None


def _decay_check(what, q, k, v, log_decay, state, lengths, scale):
    """(scale, log_decay, state, lengths) as the kernels take them; q, k, v are (B, T, J, H, D) views"""
    B, T, J, H, Dk = q.shape
    Dv = v.shape[4]
    if k.shape != q.shape or v.shape[:4] != q.shape[:4]:
        raise ValueError('%s: q, k and v differ: %s, %s, %s (shared heads: expand them)' % (what, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if not q.dtype == k.dtype == v.dtype:
        raise ValueError('%s: q, k and v have types %s, %s, %s' % (what, q.dtype, k.dtype, v.dtype))
    if max(Dk, Dv) > DECAY_MAX_D:
        raise ValueError('%s: at most %d channels a head, got %d and %d' % (what, DECAY_MAX_D, Dk, Dv))
    if tuple(log_decay.shape) != (H,) or not log_decay.is_floating_point():
        raise ValueError('%s: log_decay holds one number for each of the %d heads, got %s %s' % (what, H, log_decay.dtype, tuple(log_decay.shape)))
    if log_decay.requires_grad:
        raise ValueError('%s: the decays are fixed: there is no gradient for log_decay (pass log_decay.detach())' % what)
    if state is not None and (tuple(state.shape) != (B, J, H, Dk, Dv) or state.dtype != torch.float32):
        raise ValueError('%s: the state has to be float32 %s, got %s %s' % (what, (B, J, H, Dk, Dv), state.dtype, tuple(state.shape)))
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError('%s: lengths holds %d integers, got %s %s' % (what, B, lengths.dtype, tuple(lengths.shape)))
    _on_device(what, q, k, v, log_decay, state, lengths)
    if lengths is not None:
        lengths = (lengths if lengths.dtype == torch.int32 else lengths.clamp(0, T).int()).contiguous()
    return float(Dk ** -0.5 if scale is None else scale), log_decay.float().contiguous(), lengths


def decay_attention(q, k, v, log_decay, state=None, lengths=None, scale=None, return_state=False):
    """Causal linear attention with a decay for each head:  S_t = exp(log_decay[h]) S_(t-1) + k_t v_t',  o_t = scale q_t' S_t.

    q, k: (B, T, J, H, Dk), v: (B, T, J, H, Dv), or without J; at most 128 channels a head.  Heads shared by several query heads are
    passed expanded (a stride of 0 is read as it is).  log_decay: (H,), normally <= 0 (minus infinity: no memory), not trained.  state:
    S before the first token, (B, J, H, Dk, Dv) float32 (J = 1 for plain sequences; None: zero).  lengths: (B,) tokens of each clip,
    clamped to 0 .. T (None: T); outputs and gradients behind a clip's end are zero, whatever stands there in the inputs.  scale: Dk ** -0.5.
    Returns o, or (o, state behind the last token of each clip) with return_state=True.  Differentiable in q, k, v and state; S is held in
    fp32 throughout."""
    plain = q.dim() == 4
    qs, ks, vs = (_heads('decay_attention', n, t) for n, t in (('q', q), ('k', k), ('v', v)))
    scale, log_decay, lengths = _decay_check('decay_attention', qs, ks, vs, log_decay, state, lengths, scale)
    if state is not None:
        state = state.contiguous()
    o, new = _Decay.apply(qs, ks, vs, log_decay, state, lengths, scale, bool(return_state))
    o = o.squeeze(2) if plain else o
    return (o, new) if return_state else o


def decay_attention_step(q, k, v, log_decay, state, lengths=None, scale=None):
    """decay_attention for ONE token of every stream: q, k (B, J, H, Dk), v (B, J, H, Dv), or without J; `state` (B, J, H, Dk, Dv) float32,
    contiguous, is updated in place.  A stream whose lengths[b] is below 1 has no token: its state stays, its output is zero.
    Inference only: raises where autograd would have to record the call."""
    what = 'decay_attention_step'
    plain = q.dim() == 3
    if not (q.dim() == k.dim() == v.dim() and q.dim() in (3, 4)):
        raise ValueError('%s: q, k and v have to be (B, J, H, D) or (B, H, D), got %s, %s, %s' % (what, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    qs, ks, vs = (_heads(what, n, t.unsqueeze(1)) for n, t in (('q', q), ('k', k), ('v', v)))
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state)):
        raise RuntimeError('%s updates the state in place and has no gradient: call it under torch.no_grad(), or use decay_attention' % what)
    scale, log_decay, lengths = _decay_check(what, qs, ks, vs, log_decay, state, lengths, scale)
    if not state.is_contiguous():
        raise ValueError('%s: the state has to be contiguous' % what)
    B, _, J, H, _ = qs.shape
    o = torch.empty(B, 1, J, H, vs.shape[4], dtype=q.dtype, device=q.device)
    if B:
        with torch.cuda.device(q.device):
            _ops().decay_step(qs, ks, vs, log_decay, lengths, scale, state, o)
    return o.view(B, H, -1) if plain else o.squeeze(1)


# ------------------------------------------------------------------------------------------------ layer norm
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, drop, salt):
        C = x.shape[-1]
        X = _rows(x)
        rows = X.shape[0]
        Y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        train = any(ctx.needs_input_grad)
        mean, rstd = (torch.empty(rows, dtype=torch.float32, device=x.device) for _ in range(2)) if train else (None, None)
        R = S = None
        if residual is not None:
            R = _rows(residual)
            S = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if rows:
            with torch.cuda.device(x.device):
                _ops().layer_norm_fwd(X, R, weight, bias, eps, drop, salt, None if S is None else S.view(rows, C), Y.view(rows, C), mean, rstd)
        if train:
            ctx.save_for_backward(X if S is None else S, weight, mean, rstd, None if drop is None else drop.seed)
        ctx.drop, ctx.salt, ctx.added = drop, salt, S is not None
        ctx.set_materialize_grads(False)
        return Y, S

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dY, dStream):
        S, weight, mean, rstd, seed = ctx.saved_tensors
        shape = (dY if dY is not None else dStream).shape
        C = shape[-1]
        S = S.view(-1, C) if ctx.added else S
        rows = S.shape[0]
        want_x, want_r, want_w, want_b = ctx.needs_input_grad[:4]
        empty = lambda *s, dtype=S.dtype: torch.empty(*s, dtype=dtype, device=S.device)  # noqa: E731
        drop = None if seed is None else ctx.drop._replace(seed=seed)
        # without dropout the branch and the stream have the same gradient
        shared = drop is None
        dS = empty(rows, C) if want_r or (want_x and shared) else None
        dX = empty(rows, C) if want_x and not shared else None
        dw = empty(C, dtype=torch.float32) if want_w else None
        db = empty(C, dtype=torch.float32) if want_b else None
        if rows:
            with torch.cuda.device(S.device):
                _ops().layer_norm_bwd(None if dY is None else _rows(dY), None if dStream is None else _rows(dStream), S, weight, mean, rstd, drop,
                                      ctx.salt, dX, dS, dw, db)
        else:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        dx = (dS if shared else dX).view(shape) if want_x else None
        return dx, dS.view(shape) if want_r else None, dw, db, None, None, None


def _rows(t):
    """(rows, C) view with contiguous channels and one stride between rows; a copy where there is none"""
    C = t.shape[-1]
    if t.dim() == 2 and (t.stride(1) == 1 or C == 1):
        return t
    if t.dim() != 2 and not t.is_contiguous():
        try:
            r = t.view(-1, C)
            if r.stride(1) == 1:
                return r
        except RuntimeError:
            pass
    return t.contiguous().view(-1, C)


def _norm(what, x, residual, weight, bias, eps, drop, salt):
    C = x.shape[-1] if x.dim() else 0
    if not C:
        raise ValueError('%s: x needs a last axis to normalise, got %s' % (what, tuple(x.shape)))
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError('%s: x and residual differ: %s %s and %s %s' % (what, tuple(x.shape), x.dtype, tuple(residual.shape), residual.dtype))
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None and (tuple(t.shape) != (C,) or not t.is_floating_point()):
            raise ValueError('%s: %s holds %d numbers, got %s %s' % (what, name, C, t.dtype, tuple(t.shape)))
    if not eps >= 0:
        raise ValueError('%s: eps has to be at least 0, got %r' % (what, eps))
    if drop is not None and (drop.seed is None or drop.seed.numel() != 1 or drop.seed.element_size() != 4 or drop.seed.is_floating_point()):
        raise ValueError('%s: the dropout seed is a one-element int32 tensor' % what)
    _on_device(what, x, residual, weight, bias, None if drop is None else drop.seed)
    if drop is not None and drop.thresh == 0:
        drop = None
    weight, bias = (None if t is None else t.float().contiguous() for t in (weight, bias))
    return _LayerNorm.apply(x, residual, weight, bias, float(eps), drop, int(salt))


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis.  Statistics in fp32; weight and bias (C,) in fp32 (other types are
    converted).  Differentiable in all three; the weight's and bias' gradients are summed in a fixed order."""
    return _norm('layer_norm', x, None, weight, bias, eps, None, 0)[0]


def add_layer_norm(x, residual, weight=None, bias=None, eps=1e-5, drop=None, salt=0):
    """s = residual + dropout(x), y = layer_norm(s), in one pass: returns (y, s).  s is rounded to the tensors' type and y is the norm of
    the rounded values, so both match what the next layer reads.  drop: gast_hip.binding.Dropout(seed, *dropout_params(p)) -- the library's
    counter stream at tensor `salt`, element by element in the order of x's axes; its mask is not stored but made again in the backward
    pass from the seed tensor, which must not change in between -- or None.  Differentiable in x, residual, weight and bias."""
    return _norm('add_layer_norm', x, residual, weight, bias, eps, drop, salt)
