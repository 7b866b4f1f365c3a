"""What the entry points of gast_hip.temporal refuse, beyond sizes and types."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from gast_hip import temporal as tp


def z(*s, **k):
    return torch.zeros(s, **k)


CALLS = dict(
    rotary=(lambda t: tp.rotary((t['q'], t['k']), torch.arange(3), t['freqs']), 'q k freqs'),
    decay_attention=(lambda t: tp.decay_attention(t['q'], t['k'], t['v'], t['log_decay'], state=t['state']), 'q k v log_decay state'),
    decay_attention_step=(lambda t: tp.decay_attention_step(t['q'][:, 0], t['k'][:, 0], t['v'][:, 0], t['log_decay'], t['state']), 'q k v log_decay state'),
    layer_norm=(lambda t: tp.layer_norm(t['q'], t['weight'], t['bias']), 'q weight bias'),
    add_layer_norm=(lambda t: tp.add_layer_norm(t['q'], t['k'], t['weight'], t['bias']), 'q k weight bias'))


def inputs():
    return dict(q=z(2, 3, 1, 2, 4), k=z(2, 3, 1, 2, 4), v=z(2, 3, 1, 2, 5), log_decay=z(2), state=z(2, 1, 2, 4, 5), freqs=tp.rotary_frequencies(4),
                weight=z(4), bias=z(4))


@pytest.mark.parametrize('grad', [False, True], ids=['no grad', 'grad'])
@pytest.mark.parametrize('name', list(CALLS))
def test_tangents_are_refused(name, grad):
    """a dual tensor came back without its tangent, as if the derivative were zero"""
    call, which = CALLS[name]
    for n in which.split():
        with torch.set_grad_enabled(grad), fwAD.dual_level():
            t = inputs()
            t[n] = fwAD.make_dual(t[n], torch.ones_like(t[n]))
            with pytest.raises(NotImplementedError, match='%s: there is no forward-mode derivative' % name):
                call(t)
            t[n] = fwAD.unpack_dual(t[n]).primal
            with pytest.raises(RuntimeError, match='no CPU fallback'):          # (and goes on without one)
                call(t)


@pytest.mark.parametrize('name', ['decay_attention', 'decay_attention_step'])
def test_a_trained_decay_is_refused_only_where_autograd_records(name):
    """inference of a model that holds its decays as a parameter"""
    t = inputs()
    t['log_decay'].requires_grad_(True)
    with pytest.raises(ValueError, match='no gradient for log_decay'):
        CALLS[name][0](t)
    with torch.no_grad(), pytest.raises(RuntimeError, match='no CPU fallback'):
        CALLS[name][0](t)


def test_trained_frequencies_are_refused_where_autograd_records():
    """they got no gradient, without a word"""
    t = inputs()
    t['freqs'].requires_grad_(True)
    with pytest.raises(ValueError, match='no gradient for freqs'):
        CALLS['rotary'][0](t)
    with torch.no_grad(), pytest.raises(RuntimeError, match='no CPU fallback'):
        CALLS['rotary'][0](t)


def strided_states():
    """states of the right size whose numbers do not lie one after the other"""
    return [z(2, 1, 2, 5, 4).transpose(3, 4), z(2, 1, 2, 4, 10)[..., ::2], z(1, 1, 2, 4, 5).expand(2, 1, 2, 4, 5), z(4, 1, 2, 4, 5)[::2]]


@pytest.mark.parametrize('i', range(4))
def test_a_step_refuses_a_state_that_is_not_contiguous(i):
    t = dict(inputs(), state=strided_states()[i])
    assert t['state'].shape == (2, 1, 2, 4, 5)
    with pytest.raises(ValueError, match='has to be contiguous'):
        CALLS['decay_attention_step'][0](t)


def test_add_layer_norm_needs_a_residual():
    """it returned one output instead of two"""
    with pytest.raises(ValueError, match='add_layer_norm: a residual is needed'):
        tp.add_layer_norm(z(2, 4), None)
