"""Gradients that are not there: a node of gast_hip.temporal whose outputs nobody differentiates is called without one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def tp():
    from gast_hip import temporal
    return temporal


class Mute(torch.autograd.Function):
    """passes its inputs on and has no gradient for them"""

    @staticmethod
    def forward(ctx, *xs):
        return sum(x.float().sum() for x in xs)

    @staticmethod
    def backward(ctx, d):
        return (None,) * len(ctx.needs_input_grad)


def leaf(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape))).cuda().requires_grad_(True)


def nothing(out, leaves):
    got = torch.autograd.grad(Mute.apply(*out), leaves, allow_unused=True)
    assert all(g is None or not g.any() for g in got), got


def test_layer_norm_without_a_gradient(tp):
    x, w, b = leaf(5, 32), leaf(32), leaf(32)
    nothing((tp.layer_norm(x, w, b),), [x, w, b])
    nothing((tp.layer_norm(x),), [x])


@pytest.mark.parametrize('p', [0.0, 0.5])
def test_add_layer_norm_without_a_gradient(tp, p):
    from gast_hip.binding import Dropout, dropout_params
    drop = Dropout(torch.tensor([3], dtype=torch.int32).cuda(), *dropout_params(p)) if p else None
    x, r, w, b = leaf(5, 3, 32), leaf(5, 3, 32), leaf(32), leaf(32)
    y, s = tp.add_layer_norm(x, r, w, b, drop=drop)
    nothing((y, s), [x, r, w, b])
    # one of the outputs alone: the other's gradient counts
    y, s = tp.add_layer_norm(x, r, w, b, drop=drop)
    got = torch.autograd.grad(Mute.apply(y) + s.sum(), [x, r, w, b], allow_unused=True)
    assert torch.equal(got[1], torch.ones_like(r)) and not got[2].any() and not got[3].any()


def test_the_other_operators_without_a_gradient(tp):
    q, k, v, s = leaf(2, 40, 1, 2, 8), leaf(2, 40, 1, 2, 8), leaf(2, 40, 1, 2, 16), leaf(2, 1, 2, 8, 16)
    ld = torch.full((2,), -0.1, device='cuda')
    nothing((tp.decay_attention(q, k, v, ld),), [q, k, v])
    nothing(tp.decay_attention(q, k, v, ld, state=s, return_state=True), [q, k, v, s])
    f = tp.rotary_frequencies(8).cuda()
    nothing((tp.rotary(q, torch.arange(40).cuda(), f),), [q])
    nothing(tp.rotary((q, k), torch.arange(40).cuda(), f), [q, k])


@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16, torch.float16], ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('C', [7, 32, 130, 4096, 20000])
@pytest.mark.parametrize('p', [0.0, 0.5])
def test_the_streams_gradient_alone_passes_rows_with_infinities(tp, dt, C, p):
    """where nobody differentiates y, the norm of such a row (NaN) has no part in anything"""
    from gast_hip.binding import Dropout, dropout_params
    drop = Dropout(torch.tensor([3], dtype=torch.int32).cuda(), *dropout_params(p)) if p else None
    x, r, w, b = (t.detach().to(d).requires_grad_(True) for t, d in ((leaf(9, C), dt), (leaf(9, C), dt), (leaf(C), torch.float32), (leaf(C), torch.float32)))
    with torch.no_grad():
        r[2, C // 2], r[8, 0], r[5, C - 1] = float('inf'), float('nan'), -float('inf')
    y, s = tp.add_layer_norm(x, r, w, b, drop=drop)
    ds = leaf(9, C + 1)[:, :C].detach().to(dt)
    dx, dr, dw, db = torch.autograd.grad(Mute.apply(y) + (s * ds).sum(), [x, r, w, b], allow_unused=True)
    assert torch.equal(dr, ds)
    assert torch.isfinite(dx).all() and (p or torch.equal(dx, ds))
    assert not dw.any() and not db.any()


@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16, torch.float16], ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('T,Dk,Dv', [(1, 8, 8), (20, 3, 40), (40, 32, 16), (70, 100, 128), (2000, 16, 24)])
def test_the_states_gradient_alone_does_not_see_the_queries(tp, dt, T, Dk, Dv):
    q, k, v = (t.detach().to(dt) for t in (leaf(2, T, 1, 2, Dk), leaf(2, T + 1, 1, 2, Dk)[:, :T], leaf(2, T, 1, 2, Dv)))
    s, dn = leaf(2, 1, 2, Dk, Dv).detach(), leaf(2, 1, 2, Dk, Dv).detach()
    ld = torch.tensor([-0.1, -0.01], device='cuda')
    wild = q.clone()
    wild[0, T // 2, 0, 1, 0], wild[1, 0, 0, 0, Dk - 1] = float('nan'), float('inf')
    got = []
    for queries, zero in ((q, True), (q, False), (wild, False)):
        t = [x.clone().requires_grad_(True) for x in (queries, k, v, s)]
        o, new = tp.decay_attention(*t[:3], ld, state=t[3], return_state=True)
        outs, grads = ([o, new], [torch.zeros_like(o), dn]) if zero else ([new], [dn])
        got.append(torch.autograd.grad(outs, t, grads, allow_unused=True))
    for name, a, b, c in zip(('dk', 'dv', 'dstate'), *(g[1:] for g in got)):
        assert torch.equal(a, b) and torch.equal(b, c), name
    assert all(g[0] is None or not g[0].any() for g in got)
