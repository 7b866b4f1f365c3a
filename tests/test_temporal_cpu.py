"""gast_hip.temporal without a GPU: what the entry points refuse, the frequencies, and the 64-bit oracle against itself."""
import ctypes
import math

import pytest
import torch

from gast_hip import binding
from gast_hip import temporal as tp
from gast_hip.binding import Dropout
from oracle import temporal_oracle as to


def z(*s, dtype=torch.float32, **k):
    return torch.zeros(s, dtype=dtype, **k)


def test_cpu_tensors_are_refused():
    f = tp.rotary_frequencies(4)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        tp.rotary(z(1, 2, 1, 1, 4), torch.arange(2), f)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        tp.decay_attention(z(1, 2, 1, 4), z(1, 2, 1, 4), z(1, 2, 1, 4), z(1))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        tp.decay_attention_step(z(1, 1, 4), z(1, 1, 4), z(1, 1, 4), z(1), z(1, 1, 1, 4, 4))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        tp.layer_norm(z(2, 4))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        tp.add_layer_norm(z(2, 4), z(2, 4))


def rotary_args(**k):
    a = dict(x=z(2, 3, 1, 2, 8), positions=torch.arange(3), freqs=tp.rotary_frequencies(8))
    a.update(k)
    return a


@pytest.mark.parametrize('bad', [
    dict(x=z(2, 3, 8)), dict(x=z(2, 3, 1, 2, 0)), dict(x=()), dict(x=(z(2, 3, 1, 2, 8),) * 5), dict(x=(z(2, 3, 1, 2, 8), z(2, 3, 1, 2, 6))),
    dict(x=(z(2, 3, 1, 2, 8), z(2, 4, 1, 2, 8))), dict(x=(z(2, 3, 1, 2, 8), z(2, 3, 1, 2, 8, dtype=torch.bfloat16))), dict(x=z(2, 3, 1, 2, 6)),
    dict(x=z(2, 3, 1, 2, 1026)), dict(x=z(2, 3, 1, 2, 8, dtype=torch.float64)), dict(positions=torch.arange(4)), dict(positions=z(3)),
    dict(positions=torch.zeros(3, 3, dtype=torch.int64)), dict(freqs=z(4)), dict(freqs=z(2, 2, dtype=torch.float64)), dict(freqs=z(0, dtype=torch.float64)),
    dict(freqs=z(5, dtype=torch.float64))])
def test_rotary_refuses(bad):
    with pytest.raises(ValueError, match='rotary'):
        tp.rotary(**rotary_args(**bad))


def decay_args(**k):
    a = dict(q=z(2, 3, 2, 4), k=z(2, 3, 2, 4), v=z(2, 3, 2, 5), log_decay=z(2))
    a.update(k)
    return a


DECAY_BAD = [
    dict(k=z(2, 3, 1, 4)), dict(v=z(2, 4, 2, 5)), dict(k=z(2, 3, 2, 4, dtype=torch.bfloat16)), dict(log_decay=z(3)), dict(log_decay=z(2, dtype=torch.int32)),
    dict(log_decay=z(2, requires_grad=True)), dict(state=z(2, 2, 4, 5)), dict(state=z(2, 1, 2, 5, 4)), dict(state=z(2, 1, 2, 4, 5, dtype=torch.bfloat16)),
    dict(lengths=torch.ones(3, dtype=torch.int32)), dict(lengths=z(2)), dict(q=z(2, 3, 2, 0), k=z(2, 3, 2, 0)),
    dict(q=z(2, 3, 2, 129), k=z(2, 3, 2, 129)), dict(v=z(2, 3, 2, 129)),
    dict(q=z(2, 3, 2, 4, dtype=torch.float64), k=z(2, 3, 2, 4, dtype=torch.float64), v=z(2, 3, 2, 5, dtype=torch.float64))]


@pytest.mark.parametrize('bad', DECAY_BAD + [dict(q=z(3, 2, 4))])
def test_decay_attention_refuses(bad):
    with pytest.raises(ValueError, match='decay_attention'):
        tp.decay_attention(**decay_args(**bad))


@pytest.mark.parametrize('bad', DECAY_BAD[:1] + DECAY_BAD[2:])          # (the second differs in its frames alone)
def test_decay_attention_step_refuses(bad):
    a = decay_args(**dict(dict(state=z(2, 1, 2, 4, 5)), **bad))
    for n in 'qkv':
        a[n] = a[n][:, 0]
    with pytest.raises(ValueError, match='decay_attention_step'):
        tp.decay_attention_step(**a)


def test_decay_attention_step_refuses_gradients_and_strided_states():
    a = dict(q=z(2, 2, 4), k=z(2, 2, 4), v=z(2, 2, 5), log_decay=z(2), state=z(2, 1, 2, 4, 5))
    with pytest.raises(RuntimeError, match='no gradient'):
        tp.decay_attention_step(**dict(a, k=z(2, 2, 4, requires_grad=True)))
    with pytest.raises(ValueError):
        tp.decay_attention_step(**dict(a, q=z(2, 4)))


@pytest.mark.parametrize('bad', [
    dict(x=z()), dict(x=z(3, 0)), dict(residual=z(2, 5)), dict(residual=z(2, 4, dtype=torch.bfloat16)), dict(weight=z(5)), dict(bias=z(2, 4)),
    dict(weight=z(4, dtype=torch.int32)), dict(eps=-1.0), dict(eps=float('nan')), dict(x=z(2, 4, dtype=torch.float64), residual=z(2, 4, dtype=torch.float64)),
    dict(drop=Dropout(None, 100, 1.0)), dict(drop=Dropout(z(1), 100, 1.0)), dict(drop=Dropout(torch.ones(2, dtype=torch.int32), 100, 1.0))])
def test_add_layer_norm_refuses(bad):
    a = dict(x=z(2, 4), residual=z(2, 4))
    if 'x' in bad and 'residual' not in bad:
        a['residual'] = bad['x']
    with pytest.raises(ValueError, match='add_layer_norm'):
        tp.add_layer_norm(**dict(a, **bad))


def test_rotary_frequencies():
    f = tp.rotary_frequencies(8)
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-12)
    assert torch.equal(tp.rotary_frequencies(8, scaling='linear', factor=4.0), f / 4.0)
    g = tp.rotary_frequencies(8, scaling='base', factor=4.0)
    assert g[0] == f[0] and abs(float(g[3] / f[3]) - 0.25) < 1e-12 and torch.all(g <= f)
    b = tp.rotary_frequencies(64, scaling='bands', factor=8.0, low=1.0, high=32.0, length=2048)
    f = tp.rotary_frequencies(64)
    turns = f * 2048 / (2 * math.pi)
    assert torch.equal(b[turns >= 32], f[turns >= 32]) and torch.allclose(b[turns <= 1], f[turns <= 1] / 8, rtol=1e-12)
    between = (turns > 1) & (turns < 32)
    assert between.any() and torch.all(b[between] < f[between]) and torch.all(b[between] > f[between] / 8)
    assert tp.rotary_frequencies(2, scaling='base', factor=2.0).tolist() == [1.0]
    for bad in (dict(dim=3), dict(dim=0), dict(dim=4, scaling='x'), dict(dim=4, base=0.0), dict(dim=4, factor=-1.0), dict(dim=4, scaling='bands'),
                dict(dim=4, scaling='bands', length=8, low=2.0, high=2.0)):
        with pytest.raises(ValueError, match='rotary_frequencies'):
            tp.rotary_frequencies(**bad)


def test_the_oracles_recurrence_is_the_sum_over_earlier_tokens():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 9, 1, 3, d, generator=g, dtype=torch.float64) for d in (4, 4, 5))
    ld = torch.tensor([0.0, -0.3, -5.0], dtype=torch.float64)
    o, S = to.decay(q, k, v, ld, scale=0.5)
    t = torch.arange(9)
    w = torch.where(t[:, None] >= t, torch.exp(ld[:, None, None] * (t[:, None] - t).clamp(min=0)), 0.0)
    a = torch.einsum('bthd,bshd->bhts', q[:, :, 0], k[:, :, 0]) * w * 0.5
    assert torch.allclose(o[:, :, 0], torch.einsum('bhts,bshe->bthe', a, v[:, :, 0]), rtol=1e-12, atol=1e-12)
    assert torch.allclose(S[:, 0], torch.einsum('bshd,hs,bshe->bhde', k[:, :, 0], torch.exp(ld[:, None] * (8 - t)), v[:, :, 0]), rtol=1e-12, atol=1e-12)



def test_axes_that_an_int_cannot_count_are_refused():
    """sizes reach the kernels as C ints: views of 2^32 + 5 tokens (of one stored token) must not come out as 5"""
    T = 2 ** 32 + 5
    x = z(1, 1, 1, 4).expand(1, T, 1, 4)
    with pytest.raises(ValueError, match='longer than'):
        tp.decay_attention(x, x, x, z(1))
    with pytest.raises(ValueError, match='longer than'):
        tp.rotary(x, torch.zeros(1, dtype=torch.int64).expand(T), tp.rotary_frequencies(4))
    with pytest.raises(ValueError, match='longer than'):
        tp.decay_attention_step(z(1, 1, 4).expand(T, 1, 4), z(1, 1, 4).expand(T, 1, 4), z(1, 1, 4).expand(T, 1, 4), z(1), z(1, 1, 1, 4, 4).expand(T, 1, 1, 4, 4))
    with pytest.raises(ValueError, match='last axis'):
        tp.layer_norm(z(1, 1).expand(1, T))


class Seq(ctypes.Structure):
    _fields_ = [('p', ctypes.c_void_p), ('b', ctypes.c_long), ('t', ctypes.c_long), ('j', ctypes.c_long), ('h', ctypes.c_long)]


class DecayArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ('dtype', 'B', 'T', 'J', 'H', 'Dk', 'Dv')] + [
        ('scale', ctypes.c_float), ('log_decay', ctypes.c_void_p), ('lengths', ctypes.c_void_p)] + [(n, Seq) for n in ('q', 'k', 'v', 'o')] + [
        ('state', ctypes.c_void_p), ('state_out', ctypes.c_void_p)] + [(n, Seq) for n in ('d_o', 'dq', 'dk', 'dv')] + [
        (n, ctypes.c_void_p) for n in ('dstate_out', 'dstate', 'ws', 'ws_fwd')]


def test_the_c_entries_refuse_what_is_missing():
    """gast_decay_*: GAST_EINVAL (-1) or GAST_ERANGE before anything is launched"""
    lib = ctypes.CDLL(binding.library_path(torch.bfloat16))
    lib.gast_decay_ws_floats.restype = ctypes.c_long
    some = ctypes.create_string_buffer(64)
    at = ctypes.cast(some, ctypes.c_void_p).value

    def args(**k):
        a = DecayArgs(dtype=0, B=1, T=4096, J=1, H=1, Dk=32, Dv=32, scale=1.0, log_decay=at)
        for n in ('q', 'k', 'v', 'o', 'd_o', 'dq', 'dk', 'dv'):
            setattr(a, n, Seq(at, 0, 32, 0, 32))
        a.ws = a.ws_fwd = at
        for n, v in k.items():
            setattr(a, n, v)
        return a

    assert lib.gast_decay_ws_floats(0, 1, 4096, 1, 1, 32, 32) > 0 and lib.gast_decay_ws_floats(0, 1, 32, 1, 1, 32, 32) == 0
    assert lib.gast_decay_ws_floats(0, 0, 4096, 1, 1, 32, 32) == 0
    for entry in ('fwd', 'bwd', 'step'):
        call = getattr(lib, 'gast_decay_' + entry)
        T = 1 if entry == 'step' else 4096
        bad = [dict(B=0), dict(T=0), dict(J=-1), dict(H=0), dict(Dk=0), dict(Dv=0), dict(Dk=129), dict(Dv=129), dict(dtype=7), dict(log_decay=None), dict(q=Seq()),
               dict(k=Seq()), dict(v=Seq()), dict(T=2 ** 30 + 1)]
        bad += dict(fwd=[dict(o=Seq()), dict(ws=None)], bwd=[dict(d_o=Seq()), dict(dq=Seq()), dict(dk=Seq()), dict(dv=Seq()), dict(ws=None), dict(ws_fwd=None)],
                    step=[dict(o=Seq()), dict(state=None), dict(state=at, T=2)])[entry]
        for b in bad:
            assert call(ctypes.byref(args(**dict(dict(T=T, state=at), **b))), None) < 0, (entry, b)
        assert call(None, None) < 0
