"""Sequence operators along the frame axis: rotary positions, causal linear attention with a decay for each head (whole sequences, and
one frame at a time on a state), layer norm with an optional dropped-out branch.

They stand beside the path's own attention over joints, BatchNorm and dropout for models that look further back than the receptive
field of the dilated convolutions: `model/temporal_attention.py` builds its block of them, and its frame-at-a-time form.  The kernels are
csrc/rotary.hip, csrc/decay_attn.hip and csrc/layer_norm.hip.

Tensors are (B, T, J, H, D) -- a sequence belongs to one joint of one clip, H heads of D channels -- or (B, T, H, D) for plain token
sequences; any strides, as long as a head's D values are contiguous (other tensors are copied first).  fp32, bfloat16 and float16; all of a
call's activations have one type.  Everything is enqueued on the current stream of the tensors' device; there is no CPU fallback.  The
checks, autograd nodes and kernel calls are csrc/temporal_nodes.cpp (gast_hip/_temporal.so).

Every call can be captured into a HIP graph (workspaces come from torch's allocator, so every graph has its own), a backward pass together
with its forward pass, on leaves made for the capture: no graph of the same leaves that was recorded outside the capture may be alive then,
because autograd would make the capture wait for the stream of the older one.
There is no second derivative and no forward-mode one: asking for one raises.
"""
import os

import torch

from gast_hip import binding

_HERE = os.path.dirname(os.path.abspath(__file__))
if not os.path.exists(os.path.join(_HERE, '_temporal.so')):
    raise RuntimeError('gast_hip: %s not found -- build it with `python -c "import __graft_entry__ as g; g.build()"`. There is no CPU/PyTorch fallback.'
                       % os.path.join(_HERE, '_temporal.so'))
from gast_hip import _temporal  # noqa: E402

_temporal.libraries(binding.library_path(torch.bfloat16), binding.library_path(torch.float16))


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


def rotary(x, positions, freqs, interleaved=False, scale=1.0):
    """x with the first 2 * len(freqs) channels of every head turned by positions * freqs and multiplied by `scale`, the others as they
    are.  x: one tensor, or a tuple of up to four (q and k, say, with heads of their own) that are turned in one launch.  Pairs are
    channels (f, f + len(freqs)), or (2 f, 2 f + 1) with interleaved=True.  positions: (T,) for all clips or (B, T), int32 or int64, any
    values (angles are reduced in 64 bits).  Differentiable in x; freqs that require grad
    are refused where autograd records."""
    if isinstance(x, (tuple, list)):
        return tuple(_temporal.rotary(x, positions, freqs, interleaved, scale))
    return _temporal.rotary((x,), positions, freqs, interleaved, scale)[0]


# ------------------------------------------------------------------------------------------------ linear attention with a decay
def decay_attention(q, k, v, log_decay, state=None, lengths=None, scale=None, return_state=False):
    """Causal linear attention with a decay for each head:  S_t = exp(log_decay[h]) S_(t-1) + k_t v_t',  o_t = scale q_t' S_t.

    q, k: (B, T, J, H, Dk), v: (B, T, J, H, Dv), or without J; at most 128 channels a head.  Heads shared by several query heads are
    passed expanded (a stride of 0 is read as it is).  log_decay: (H,), normally <= 0 (minus infinity: no memory; above 0
    exp(log_decay * min(tokens, 32)) has to be a finite fp32 number), not trained: one that requires grad is refused where autograd records.
    state: S before the first token, (B, J, H, Dk, Dv) float32 (J = 1 for plain sequences; None: zero).  lengths: (B,) tokens of each clip,
    clamped to 0 .. T (None: T); outputs and gradients behind a clip's end are zero, whatever stands there in the inputs.  scale: Dk ** -0.5.
    Returns o, or (o, state behind the last token of each clip) with return_state=True.  Differentiable in q, k, v and state.  Whatever the
    type, scores, sums and S are fp32 and enter products with all their bits; o and the gradients are rounded to the type at the end."""
    out = _temporal.decay_attention(q, k, v, log_decay, state, lengths, scale, return_state)
    return tuple(out) if return_state else out[0]


def decay_attention_step(q, k, v, log_decay, state, lengths=None, scale=None):
    """decay_attention for ONE token of every stream: q, k (B, J, H, Dk), v (B, J, H, Dv), or without J; `state` (B, J, H, Dk, Dv) float32,
    contiguous, is updated in place.  A stream whose lengths[b] is below 1 has no token: its state stays, its output is zero.
    Inference only: raises where autograd would have to record the call."""
    return _temporal.decay_attention_step(q, k, v, log_decay, state, lengths, scale)


# ------------------------------------------------------------------------------------------------ layer norm
def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis.  Statistics in fp32; weight and bias (C,) in fp32 (other types are
    converted).  Differentiable in all three; the weight's and bias' gradients are summed in a fixed order."""
    return _temporal.norm('layer_norm', x, None, weight, bias, eps, False, None, 0, 1.0, 0)[0]


def add_layer_norm(x, residual, weight=None, bias=None, eps=1e-5, drop=None, salt=0):
    """s = residual + dropout(x), y = layer_norm(s), in one pass: returns (y, s).  s is made in fp32 and rounded to the tensors' type,
    and y is the norm of the rounded values, so both match what the next layer reads.  drop: gast_hip.binding.Dropout(seed, *dropout_params(p)) -- the library's
    counter stream at tensor `salt`, element by element in the order of x's axes; its mask is not stored but made again in the backward
    pass from the seed tensor, which must not change in between -- or None.  Differentiable in x, residual, weight and bias."""
    if drop is None:
        return tuple(_temporal.norm('add_layer_norm', x, residual, weight, bias, eps, False, None, 0, 1.0, 0))
    return tuple(_temporal.norm('add_layer_norm', x, residual, weight, bias, eps, True, drop.seed, drop.thresh, drop.inv_keep, salt))
