"""16-bit linear attention computes in fp32: sums that nearly cancel show how many bits of a score and of a state enter a product.

Two terms of size m, generic in all of fp32's bits, are left with 2^-12 of m.  The terms come from exact products (16-bit values) of a
score or a state element; what may round is the score's own sum (2), and every addition of an accumulator: two terms in at most three
parts times two of the stored operand (12), the product with the other tokens' zeros being exact.  With a whole step of fp32 (2 u, u = 2^-24)
for each, of at most 2 m: 14 * 2 u * 2 m = 56 u m; the result is rounded to its type (h = eps / 2).  One 8-bit part less in a score or a
state is 2^-17 = 128 u of each term."""
import pytest
import torch
from test_temporal_gpu import check_decay, decay_case, half

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ['fp32', 'bf16', 'fp16']
H = 64                                   # heads: as many draws


@pytest.fixture(scope='module')
def tp():
    from gast_hip import temporal
    return temporal


def one_to_two(g, *shape):
    return 1 + torch.rand(*shape, generator=g)


def attend(tp, t, do, state=None, dstate=None):
    """o, dq, dk, dv without any decay and with a scale of 1; (T, H, D) inputs"""
    q, k, v = (x.cuda().unsqueeze(0).unsqueeze(2).requires_grad_(True) for x in t)
    s = None if state is None else state.cuda().view(1, 1, *state.shape)
    o, new = tp.decay_attention(q, k, v, torch.zeros(H, device='cuda'), state=s, scale=1.0, return_state=True)
    outs, grads = [o], [do.cuda().unsqueeze(0).unsqueeze(2)]
    if dstate is not None:
        outs.append(new)
        grads.append(dstate.cuda().view(1, 1, *dstate.shape))
    got = torch.autograd.grad(outs, [q, k, v], grads)
    return dict(zip(('o', 'dq', 'dk', 'dv'), (x[0, :, 0].detach().double().cpu() for x in (o,) + got)))


def near(got, ref, m, dt, what):
    f = torch.finfo(dt)
    tol = 56 * U * m
    tol = tol + f.eps / 2 * (ref.abs() + tol) + f.smallest_normal * f.eps / 2
    assert torch.all((got - ref).abs() <= tol), '%s: off by %.1f u of a term' % (what, ((got - ref).abs() / m).max() / U)


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('at,T', [(0, 2), (5, 20), (33, 40), (70, 100)])
@pytest.mark.parametrize('D', [16, 48, 128])
def test_scores_that_cancel(tp, dt, at, T, D):
    """out = s_0 w - s_1 w, s_j = x y + g b_j: the difference is g (b_0 - b_1) w"""
    g = torch.Generator().manual_seed(T + D)
    x, y, b0, b1 = (one_to_two(g, H).to(dt) for _ in range(4))
    small = (one_to_two(g, H) * 2.0 ** -12).to(dt)
    w = one_to_two(g, H, D).to(dt)
    zero = torch.zeros(T, H, D, dtype=dt)

    def rows(*tokens):
        z = zero.clone()
        for t, values in tokens:
            z[t, :, :values.shape[-1]] = values
        return z

    pair = torch.stack([x, small], -1)                         # of the token whose output it is
    others = [torch.stack([y, b], -1) for b in (b0, b1)]
    d = [(p.double() * pair.double()).sum(-1, keepdim=True) for p in others]
    ref, m = (d[0] - d[1]) * w.double(), d[0] * w.double()
    both = rows((at, others[0]), (at + 1, others[1])), rows((at, w), (at + 1, -w))
    # forward in time the later token sees both, backward in time the earlier one
    late, early = rows((at + 1, pair)), rows((at, pair))
    near(attend(tp, (late, both[0], both[1]), zero)['o'][at + 1], ref, m, dt, 'o')
    near(attend(tp, (zero, both[1], both[0]), late)['dq'][at + 1], ref, m, dt, 'dq')
    near(attend(tp, (both[0], early, zero), both[1])['dv'][at], ref, m, dt, 'dv')
    near(attend(tp, (both[1], zero, early), both[0])['dk'][at], ref, m, dt, 'dk')


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('at,T', [(0, 1), (0, 40), (33, 40), (64, 70)])
@pytest.mark.parametrize('D', [16, 48, 128])
def test_states_that_cancel(tp, dt, at, T, D):
    """out = S_0 - S_1 (1 - 2^-12 r), all bits of S count"""
    g = torch.Generator().manual_seed(T + D)
    a = one_to_two(g, H, D)
    b = -(a * (1 - 2.0 ** -12 * one_to_two(g, H, D)))
    S = torch.zeros(H, D, D)
    S[:, 3], S[:, 7] = a, b                                    # rows d of S
    ref, m = a.double() + b.double(), a.double()
    zero = torch.zeros(T, H, D, dtype=dt)
    ones = zero.clone()
    ones[at, :, 3] = ones[at, :, 7] = 1.0
    turned = S.transpose(1, 2).contiguous()
    near(attend(tp, (ones, zero, zero), zero, state=S)['o'][at], ref, m, dt, 'o')
    near(attend(tp, (zero, zero, zero), ones, state=turned)['dq'][at], ref, m, dt, 'dq')
    near(attend(tp, (zero, ones, zero), zero, dstate=S)['dv'][at], ref, m, dt, 'dv')
    near(attend(tp, (zero, zero, ones), zero, dstate=turned)['dk'][at], ref, m, dt, 'dk')


def fp32_tol(name, ref, mag, c):
    """decay_tol's bound for fp32 (n = 4 T + Dk + Dv + 64 roundings of u) whatever the type, results rounded to theirs once"""
    T, Dk, Dv = c['q'].shape[1], c['q'].shape[4], c['v'].shape[4]
    tol = (4 * T + Dk + Dv + 64) * U * mag[name]
    if name in ('state', 'dstate0'):
        return tol + 1e-37
    h, tiny = half(c['q'].dtype)
    return tol + h * (ref[name].abs() + tol) + tiny


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('B,T,H,Dk,Dv', [(2, 1, 2, 2, 64), (2, 3, 2, 1, 128), (3, 27, 4, 4, 32), (2, 33, 2, 2, 16), (2, 70, 3, 17, 33), (1, 130, 2, 128, 128), (3, 65, 1, 64, 96),
                                         (1, 530, 3, 16, 16), (2, 362, 2, 64, 48), (1, 2050, 1, 8, 128)])
def test_16_bits_meet_the_bound_of_fp32(tp, monkeypatch, dt, B, T, H, Dk, Dv):
    import test_temporal_gpu
    monkeypatch.setattr(test_temporal_gpu, 'decay_tol', fp32_tol)
    for state in (False, True):
        check_decay(tp, decay_case(B + T + Dk, dt, B, T, 1, H, Dk, Dv, ragged=B > 2, state=state, decays=[-0.001, 0.0, -0.1]))
