"""Derivatives that gast_hip.temporal does not have are refused, not taken for zero."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def tp():
    from gast_hip import temporal
    return temporal


def leaf(*shape, on=True):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape))).cuda().requires_grad_(on)


def twice(out, leaves, asked, depends):
    """a penalty on the gradient of out.sum(): its incoming gradient is a constant, the gradient is none where `depends`"""
    g, = torch.autograd.grad(out.sum(), [leaves[asked]], create_graph=True)
    assert g.requires_grad == depends, asked
    if depends:
        other = torch.ones(3, device='cuda', requires_grad=True)
        with pytest.raises(RuntimeError, match='differentiate twice'):
            ((other * 2).sum() + g.pow(2).sum()).backward()


@pytest.mark.parametrize('asked', ['x', 'weight', 'bias'])
def test_penalties_on_layer_norms_gradients(tp, asked):
    t = dict(x=leaf(5, 32), weight=leaf(32), bias=leaf(32))
    twice(tp.layer_norm(t['x'], t['weight'], t['bias']), t, asked, asked != 'bias')
    # made from nothing that is trained: a constant, as it should be
    t = {n: leaf(*v.shape, on=n == asked) for n, v in t.items()}
    twice(tp.layer_norm(t['x'], t['weight'], t['bias']), t, asked, asked == 'x')


@pytest.mark.parametrize('asked', ['x', 'residual', 'weight', 'bias'])
@pytest.mark.parametrize('p', [0.0, 0.5])
def test_penalties_on_add_layer_norms_gradients(tp, asked, p):
    from gast_hip.binding import Dropout, dropout_params
    drop = Dropout(torch.tensor([3], dtype=torch.int32).cuda(), *dropout_params(p)) if p else None
    t = dict(x=leaf(5, 32), residual=leaf(5, 32), weight=leaf(32), bias=leaf(32))
    twice(tp.add_layer_norm(t['x'], t['residual'], t['weight'], t['bias'], drop=drop)[0], t, asked, asked != 'bias')
    if asked in ('weight', 'bias'):
        t = dict(t, x=leaf(5, 32, on=False))           # the stream depends on the residual all the same
        twice(tp.add_layer_norm(t['x'], t['residual'], t['weight'], t['bias'], drop=drop)[0], t, asked, asked == 'weight')


@pytest.mark.parametrize('T', [7, 40])
def test_penalties_on_the_attentions_gradients(tp, T):
    ld = torch.full((2,), -0.1, device='cuda')
    shapes = dict(q=(2, T, 1, 2, 8), k=(2, T, 1, 2, 8), v=(2, T, 1, 2, 16), state=(2, 1, 2, 8, 16))
    partners = dict(q='k v state', k='q v', v='q k', state='q')              # what a gradient is made from

    def out(t):
        o, s = tp.decay_attention(t['q'], t['k'], t['v'], ld, state=t['state'], return_state=True)
        return o.sum() + s.sum()

    for asked, others in partners.items():
        for trained in shapes:
            t = {n: leaf(*s, on=n in (asked, trained)) for n, s in shapes.items()}
            twice(out(t), t, asked, trained in others.split())


def test_a_rotation_is_linear(tp):
    """its gradient is made from the incoming one alone"""
    x = leaf(2, 7, 1, 2, 8)
    y = tp.rotary(x, torch.arange(7).cuda(), tp.rotary_frequencies(8).cuda())
    twice(y, dict(x=x), 'x', False)
