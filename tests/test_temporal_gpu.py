"""The sequence operators (gast_hip/temporal.py) against their definitions in 64 bits (oracle/temporal_oracle.py).

Tolerances.  u = 2^-24 is half a step of fp32, h = eps / 2 of the tensors' type.  A sum whose values take part in at most n roundings each
is off by at most n u times the sum of the absolute terms, in whatever order it is made; results are rounded once more to their type
(h |result|).  Each test says what its n counts."""
import pytest
import torch

from oracle import temporal_oracle as to

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ['fp32', 'bf16', 'fp16']


@pytest.fixture(scope='module')
def tp():
    from conftest import poison_allocations
    from gast_hip import temporal
    poison_allocations()           # (GAST_TEST_POISON=1 only)
    return temporal


def half(dt):
    """half a step of the type, relative; and of its smallest numbers, absolute"""
    f = torch.finfo(dt)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, dt, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dt)


def close(got, ref, tol, what):
    got, ref = got.detach().double().cpu(), ref.detach().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), '%s: not finite' % what
    over = ((got - ref).abs() - tol).max() if got.numel() else torch.zeros(())
    assert over <= 0, '%s: off by %.3e, %.3e more than allowed' % (what, (got - ref).abs().max(), over)


# ------------------------------------------------------------------------------------------------ rotary positions
def rotary_tol(x, positions, freqs, interleaved, scale, dt, back=False):
    """cosine and sine: the fraction of a turn is rounded to fp32 (2 pi 2^-25 < 4 u), the function is good to 2 steps (4 u), the factor, the
    product and the sum round once each: 12 u of |a| + |b|; the angle in 64 bits is off by 2 pi turns 2^-51.  Copied channels: exact."""
    R = 2 * freqs.numel()
    turns = (positions.double().abs().max() * freqs.abs().max() / 6.28).item()
    ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    m = torch.zeros_like(x, dtype=torch.float64)
    s = (x[..., ia].double().abs() + x[..., ib].double().abs()) * scale
    m[..., ia], m[..., ib] = s, s
    h, tiny = half(dt)
    ref = to.rotary(x.double(), positions, freqs, interleaved, scale, back)
    tol = m * (12 * U + 6.3 * turns * 2.0 ** -51)
    tol = tol + torch.where(m > 0, h * (ref.abs() + tol) + tiny, 0.0)
    return ref, tol


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('interleaved', [False, True], ids=['half', 'pairs'])
@pytest.mark.parametrize('B,T,J,H,D,R', [(1, 1, 1, 1, 2, 2), (2, 3, 17, 4, 32, 32), (1, 1, 17, 4, 32, 32), (3, 7, 1, 5, 33, 10), (2, 130, 1, 3, 128, 64),
                                         (1, 5, 2, 2, 90, 34), (2, 2, 1, 1, 1024, 1024), (1, 9, 1, 40, 24, 12), (1, 4, 1, 2, 20, 4)])
def test_rotary(tp, dt, interleaved, B, T, J, H, D, R):
    g = gen(B * 1000 + T + D + R)
    x = randn(g, dt, B, T, J, H, D)
    pos = torch.randint(-1000, 2000000, (B, T), generator=g)
    f = tp.rotary_frequencies(R)
    scale = 1.25
    xd = x.cuda().requires_grad_(True)
    y = tp.rotary(xd, pos.cuda(), f.cuda(), interleaved=interleaved, scale=scale)
    close(y, *rotary_tol(x, pos, f, interleaved, scale, dt), 'y')
    assert torch.equal(y[..., R:].detach().cpu(), x[..., R:])
    dy = randn(g, dt, B, T, J, H, D)
    dx, = torch.autograd.grad(y, xd, dy.cuda())
    close(dx, *rotary_tol(dy, pos, f, interleaved, scale, dt, back=True), 'dx')


def test_rotary_takes_views_several_tensors_and_any_positions(tp):
    g = gen(3)
    B, T, J, D = 2, 6, 3, 16
    f = tp.rotary_frequencies(12).cuda()
    buf = randn(g, torch.float32, B, T, J, 3, 4, D).cuda()
    q, k = buf[..., 0, :, :], buf[:, :, :, 1, :2]                      # slices of one projection, heads of their own
    shared = randn(g, torch.float32, B, T, J, 1, D).cuda().expand(B, T, J, 5, D)
    t = randn(g, torch.float32, B, J, 2, T, D).cuda().permute(0, 3, 1, 2, 4)
    odd = randn(g, torch.float32, B, T, J, 2, D + 1).cuda()[..., 1:]   # rows that start between vectors
    strided = randn(g, torch.float32, B, T, J, 2, 2 * D).cuda()[..., ::2]
    for pos in (torch.arange(T), torch.arange(T, dtype=torch.int32), torch.arange(T).view(1, T), torch.arange(B * T).view(B, T) - 5,
                torch.arange(2 * T)[::2], torch.tensor([2 ** 40 + 1] * T), torch.zeros(T, dtype=torch.int64)):
        for xs in ((q, k), (shared, t, odd), (strided,), (q, k, t, odd)):
            ys = tp.rotary(xs, pos.cuda(), f)
            for x, y in zip(xs, ys):
                close(y, *rotary_tol(x.cpu(), pos.view(-1, T).expand(B, T), f.cpu(), False, 1.0, torch.float32), 'y')
    assert tp.rotary(q[:, :0], torch.zeros(0, dtype=torch.int64).cuda(), f).shape == (B, 0, J, 4, D)
    x4 = q[:, :, 0]
    assert torch.equal(tp.rotary(x4, torch.arange(T).cuda(), f), tp.rotary(q, torch.arange(T).cuda(), f)[:, :, 0])


def test_rotary_copies_what_is_not_turned_and_keeps_empty_calls(tp):
    x = torch.full((1, 2, 1, 2, 8), float('inf')).cuda()
    x[..., :4] = 1.0
    y = tp.rotary(x, torch.arange(2).cuda(), tp.rotary_frequencies(4).cuda(), interleaved=True)
    assert torch.isinf(y[..., 4:]).all() and torch.isfinite(y[..., :4]).all()
    e = tp.rotary(x[:0], torch.arange(2).cuda(), tp.rotary_frequencies(4).cuda())
    assert e.shape == (0, 2, 1, 2, 8)


def test_rotary_in_place_through_the_c_abi(tp):
    """y may be x: the vector at a row's end overlaps the one before it, which another thread may have turned already"""
    import ctypes

    from gast_hip import binding

    class Seq(ctypes.Structure):
        _fields_ = [('p', ctypes.c_void_p)] + [(n, ctypes.c_long) for n in 'btjh']

    class Job(ctypes.Structure):
        _fields_ = [('x', Seq), ('y', Seq), ('H', ctypes.c_int)]

    B, T, J, H = 2, 300, 1, 3
    for dt in (torch.float32, torch.bfloat16):
        lib = ctypes.CDLL(binding.library_path(dt))
        for D, R, inter in ((18, 18, 0), (18, 18, 1), (45, 22, 0), (45, 22, 1), (128, 64, 0)):
            x, f, pos = randn(gen(D), dt, B, T, J, H, D).cuda(), tp.rotary_frequencies(R).cuda(), torch.arange(T).cuda()
            want = tp.rotary(x, pos, f, interleaved=bool(inter))
            job = Job(*[Seq(x.data_ptr(), *x.stride()[:4])] * 2, H)
            rc = lib.gast_rotary_multi(0 if dt == torch.float32 else 1, ctypes.byref(job), 1, B, T, J, D, R, inter, ctypes.c_void_p(pos.data_ptr()), 1,
                                       ctypes.c_long(0), ctypes.c_long(1), ctypes.c_void_p(f.data_ptr()), ctypes.c_float(1.0), 0,
                                       ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
            assert rc == 0 and torch.equal(x, want), (dt, D, R, inter)


# ------------------------------------------------------------------------------------------------ linear attention with a decay
def decay_case(seed, dt, B, T, J, H, Dk, Dv, ragged=False, state=True, decays=None):
    g = gen(seed)
    c = dict(q=randn(g, dt, B, T, J, H, Dk), k=randn(g, dt, B, T, J, H, Dk), v=randn(g, dt, B, T, J, H, Dv), do=randn(g, dt, B, T, J, H, Dv))
    c['log_decay'] = (-torch.rand(H, generator=g) * 0.2 if decays is None else torch.tensor([decays[i % len(decays)] for i in range(H)])).float()
    c['lengths'] = None
    if ragged:
        c['lengths'] = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        c['lengths'][B // 2] = 0
        c['lengths'][0] = T
    c['state'] = torch.randn(B, J, H, Dk, Dv, generator=g) if state else None
    c['dstate'] = torch.randn(B, J, H, Dk, Dv, generator=g) if state else None
    return c


def decay_reference(c, scale):
    args = [c[n] for n in ('q', 'k', 'v', 'log_decay', 'state', 'lengths')] + [scale, c['do'], c['dstate']]
    ref = to.decay_grads(*args)
    n = None if c['lengths'] is None else c['lengths'].clamp(0, c['q'].shape[1])
    a = [c['q'].double().abs(), c['k'].double().abs(), c['v'].double().abs(), c['log_decay'], None if c['state'] is None else c['state'].double().abs(), n,
         scale, c['do'].double().abs(), None if c['dstate'] is None else c['dstate'].double().abs()]
    return ref, to.decay_grads(*a)


def decay_tol(name, ref, mag, c):
    """Roundings that a term meets: at most one in every addition of its sums (T tokens, Dk or Dv channels) and three in every power of the
    decay (T more of each), 64 for the rest: n = 4 T + Dk + Dv + 64, times u, of the absolute terms.  16-bit types: a score and a state may
    be rounded to the type once on their way into a product (2 h of the absolute terms), and the result is.  States are fp32; products
    that make them may be split into parts that keep 20 bits."""
    T, Dk, Dv = c['q'].shape[1], c['q'].shape[4], c['v'].shape[4]
    tol = (4 * T + Dk + Dv + 64) * U * mag[name]
    dt = c['q'].dtype
    if name in ('state', 'dstate0'):
        return tol + (2.0 ** -20 * mag[name] if dt != torch.float32 else 0.0) + 1e-37
    h, tiny = half(dt)
    if dt != torch.float32:
        tol = tol + 2 * h * mag[name]
    return tol + h * (ref[name].abs() + tol) + tiny


def check_decay(tp, c, scale=None, views=None, quiet_tail=False):
    B, T, J, H, Dk = c['q'].shape
    ref, mag = decay_reference(c, Dk ** -0.5 if scale is None else scale)
    dev = {n: None if t is None else t.cuda() for n, t in c.items()}
    if views:
        dev.update(views)
    leaves = [dev[n].detach().requires_grad_(True) if not views or n not in views else dev[n].requires_grad_(True) for n in ('q', 'k', 'v')]
    st = None if dev['state'] is None else dev['state'].detach().requires_grad_(True)
    o, new = tp.decay_attention(*leaves, dev['log_decay'], state=st, lengths=dev['lengths'], scale=scale, return_state=True)
    outs, grads = [o], [dev['do']]
    if c['dstate'] is not None:
        outs.append(new)
        grads.append(dev['dstate'])
    got = torch.autograd.grad(outs, leaves + ([] if st is None else [st]), grads)
    res = dict(o=o, state=new, dq=got[0], dk=got[1], dv=got[2])
    if st is not None:
        res['dstate0'] = got[3]
    for name, r in res.items():
        close(r, ref[name], decay_tol(name, ref, mag, c), name)
    if c['lengths'] is not None:
        for b in range(B):
            n = int(c['lengths'][b].clamp(0, T))
            for name in ('o', 'dq', 'dk', 'dv'):
                assert not res[name][b, n:].any(), '%s behind the end of clip %d' % (name, b)
    return res


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('T', [1, 2, 15, 16, 17, 27, 31, 32, 33, 63, 64, 65, 127, 128, 129, 243])
def test_decay_lengths(tp, dt, T):
    check_decay(tp, decay_case(T, dt, 2, T, 1, 2, 32, 32))


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('Dk,Dv', [(1, 1), (1, 128), (128, 1), (8, 16), (16, 16), (17, 33), (31, 32), (48, 80), (64, 64), (64, 128), (128, 64), (127, 5), (96, 96),
                                   (128, 128), (66, 34)])
def test_decay_heads(tp, dt, Dk, Dv):
    check_decay(tp, decay_case(Dk * 131 + Dv, dt, 1, 70, 2, 3, Dk, Dv))


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('state', [False, True], ids=['fresh', 'going on'])
@pytest.mark.parametrize('B,T,J,H,D', [(5, 40, 3, 2, 32), (4, 150, 1, 3, 64), (3, 67, 2, 1, 128), (6, 1, 1, 2, 16)])
def test_decay_ragged(tp, dt, state, B, T, J, H, D):
    c = decay_case(B * T, dt, B, T, J, H, D, D, ragged=True, state=state)
    # what stands behind a clip's end is not looked at
    for n in ('q', 'k', 'v', 'do'):
        for b in range(B):
            c[n][b, int(c['lengths'][b]):] = float('nan') if n != 'k' else float('inf')
    ref_c = {n: (t.clone() if torch.is_tensor(t) else t) for n, t in c.items()}
    for n in ('q', 'k', 'v', 'do'):
        ref_c[n] = torch.nan_to_num(ref_c[n], nan=0.0, posinf=0.0)
    views = {n: c[n].cuda() for n in ('q', 'k', 'v', 'do')}
    check_decay(tp, ref_c, views=views)


def test_decay_lengths_are_clamped(tp):
    c = decay_case(5, torch.float32, 4, 20, 1, 2, 16, 16)
    c['lengths'] = torch.tensor([-3, 0, 20, 2 ** 31 - 1], dtype=torch.int32)
    check_decay(tp, c)
    c['lengths'] = torch.tensor([-2 ** 40, 7, 2 ** 40, 19])
    check_decay(tp, c)


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
def test_decay_of_any_strength(tp, dt):
    """none at all, one that forgets within a token, minus infinity (no memory: o_t = scale (q_t k_t) v_t), and a growing one"""
    check_decay(tp, decay_case(1, dt, 2, 100, 1, 4, 32, 32, decays=[0.0, -30.0, -200.0, -float('inf')]))
    check_decay(tp, decay_case(2, dt, 2, 100, 1, 2, 32, 32, decays=[0.02, -1e-7]))


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
def test_decay_long(tp, dt):
    """few sequences and many tokens: the time axis is split and joined"""
    check_decay(tp, decay_case(7, dt, 1, 4100, 1, 2, 16, 32, decays=[-0.01, -0.0005]))
    check_decay(tp, decay_case(8, dt, 2, 1500, 1, 1, 64, 64, ragged=True, decays=[-0.001]))


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('B,T,H,Dk,Dv', [(1, 530, 3, 16, 16), (3, 362, 4, 64, 48), (2, 700, 2, 128, 96), (2, 300, 2, 31, 87), (3, 65, 1, 128, 8), (1, 2050, 1, 7, 128)])
def test_decay_segments(tp, dt, B, T, H, Dk, Dv):
    """a few chunks a segment down to one, clips that end before a segment begins, states at both ends"""
    check_decay(tp, decay_case(B + T, dt, B, T, 1, H, Dk, Dv, ragged=B > 1, decays=[-0.01, -0.0005, -2.0, 0.0]))


WILD = [(20, 32, [(7, 'nan'), (19, 'inf')]), (27, 64, [(13, '-inf')]), (32, 96, [(0, 'inf'), (31, 'nan')]), (200, 48, [(40, 'inf'), (170, 'nan')]), (130, 128, [(96, 'nan')]),
        (3000, 64, [(1500, 'nan')])]


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('state', [False, True], ids=['fresh', 'going on'])
@pytest.mark.parametrize('T,D,at', WILD, ids=['T%d D%d' % w[:2] for w in WILD])
def test_decay_infinities_and_nan_reach_only_what_sees_them(tp, dt, state, T, D, at):
    """What stands at a later token (for gradients: at an earlier one) of the sequence does not count as zero times itself.  Everything that
    does not see a token is, to the bit, what it is with a zero there."""
    base = decay_case(T + D, dt, 2, T, 1, 2, D, D, state=state, decays=[0.0, -0.01])
    B, H = 2, 2
    t = torch.arange(T)

    def run(c):
        q, k, v, s = (None if c[n] is None else c[n].cuda().requires_grad_(True) for n in ('q', 'k', 'v', 'state'))
        o = tp.decay_attention(q, k, v, c['log_decay'].cuda(), state=s)
        return dict(zip(('o', 'dq', 'dk', 'dv'), (o.detach(),) + torch.autograd.grad(o, (q, k, v), c['do'].cuda())))

    # whose token (c), and what it reaches: its own channel e of one tensor and every channel of another, later ('+') or earlier ('-'), and
    # every channel of its own token in a third
    reach = dict(v=(('o', '+'), ('dq', '+'), 'dk'), k=(('dq', '+'), ('o', '+'), 'dv'), do=(('dv', '-'), ('dk', '-'), 'dq'), q=(('dk', '-'), ('dv', '-'), 'o'))
    for name, (own, every, alone) in reach.items():
        c, zero = dict(base), dict(base)
        c[name], zero[name] = base[name].clone(), base[name].clone()
        e = 5 % D
        for token, value in at:
            c[name][1, token, 0, 1, e] = float(value)
            zero[name][1, token, 0, 1, e] = 0.0
        got, want = run(c), run(zero)
        hit = {n: torch.zeros(B, T, 1, H, D, dtype=torch.bool) for n in got}
        for token, _ in at:
            for (n, way), chan in ((own, slice(e, e + 1)), (every, slice(None))):
                sees = t >= token if way == '+' else t <= token
                hit[n][1, sees, 0, 1, chan] = True
            hit[alone][1, token, 0, 1, :] = True
        for n in got:
            g, w, h = got[n].cpu(), want[n].cpu(), hit[n]
            assert torch.equal(g[~h], w[~h]), (name, n)
            assert not torch.isfinite(g[h]).any(), (name, n)


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
def test_decay_reads_views(tp, dt):
    g = gen(11)
    B, T, J, H, D = 2, 40, 3, 4, 16
    c = decay_case(9, dt, B, T, J, H, D, D)
    buf = randn(g, dt, B, T, J, 3, H, D).cuda()                            # one projection, rows of 3 H D
    views = dict(q=buf[:, :, :, 0], k=buf[:, :, :, 1], v=buf[:, :, :, 2])
    for n in 'qkv':
        c[n] = views[n].cpu()
        views[n] = views[n].detach()
    check_decay(tp, c, views=views)
    # (B, H, T, D) order; rows that start between vectors; a head shared by all
    t = randn(g, dt, B, H, J, T, D).cuda().permute(0, 3, 2, 1, 4)
    odd = randn(g, dt, B, T, J, H, D + 3).cuda()[..., 3:]
    one = randn(g, dt, B, T, J, 1, D).cuda().expand(B, T, J, H, D)
    do = randn(g, dt, B, H, T, J, D).cuda().permute(0, 2, 3, 1, 4)
    views = dict(q=t.detach(), k=odd.detach(), v=one.detach().clone(), do=do)
    for n in views:
        c[n] = views[n].cpu()
    check_decay(tp, c, views=views)


def test_decay_shared_heads_sum_their_gradients(tp):
    """k and v with one head for four query heads, expanded: read with a stride of 0, gradients summed over the heads"""
    g = gen(12)
    B, T, H, D = 2, 50, 4, 32
    c = decay_case(13, torch.float32, B, T, 1, H, D, D, state=False)
    k1, v1 = randn(g, torch.float32, B, T, 1, 1, D), randn(g, torch.float32, B, T, 1, 1, D)
    c['k'], c['v'] = k1.expand(B, T, 1, H, D), v1.expand(B, T, 1, H, D)
    ref, mag = decay_reference(c, D ** -0.5)
    kd, vd = k1.cuda().requires_grad_(True), v1.cuda().requires_grad_(True)
    qd = c['q'].cuda().requires_grad_(True)
    o = tp.decay_attention(qd, kd.expand(B, T, 1, H, D), vd.expand(B, T, 1, H, D), c['log_decay'].cuda())
    close(o, ref['o'], decay_tol('o', ref, mag, c), 'o')
    dk, dv = torch.autograd.grad(o, [kd, vd], c['do'].cuda())
    for name, got in (('dk', dk), ('dv', dv)):
        close(got, ref[name].sum(3, keepdim=True), decay_tol(name, ref, mag, c).sum(3, keepdim=True) + 4 * U * mag[name].sum(3, keepdim=True), name)


def test_decay_gradients_against_differences(tp):
    """o is linear in q, in k and in v alone: a central difference of any width is exact but for rounding, n u of the absolute terms of both
    values (see decay_tol), divided by the width (1)"""
    c = decay_case(21, torch.float32, 2, 90, 1, 2, 24, 40)
    dev = {n: None if t is None else t.cuda() for n, t in c.items()}
    for name in ('q', 'k', 'v', 'state'):
        x = dev[name].detach().requires_grad_(True)
        d = torch.randn(x.shape, generator=gen(22)).cuda()

        def f(y):
            a = dict(dev, **{name: y})
            o, new = tp.decay_attention(a['q'], a['k'], a['v'], a['log_decay'], state=a['state'], return_state=True)
            return (o.double() * dev['do'].double()).sum() + (new.double() * dev['dstate'].double()).sum()

        slope = (f(x.detach() + d) - f(x.detach() - d)) / 2
        o, new = tp.decay_attention(*[x if n == name else dev[n] for n in ('q', 'k', 'v')], dev['log_decay'],
                                    state=x if name == 'state' else dev['state'], return_state=True)
        gx, = torch.autograd.grad([o, new], x, [dev['do'], dev['dstate']])
        _, mag = decay_reference(dict(c, **{name: c[name].abs() + d.cpu().abs()}), 24 ** -0.5)
        n = 4 * 90 + 24 + 40 + 64
        bound = n * U * float((mag['o'] * c['do'].abs()).sum() + (mag['state'] * c['dstate'].abs()).sum()) * 2
        assert abs(float(slope - (gx.double() * d.double()).sum())) <= bound


def test_decay_carries_on_where_a_call_stopped(tp):
    """a sequence in pieces, the state handed on, is the sequence in one call; and token by token"""
    dt, B, T, J, H, Dk, Dv = torch.float32, 2, 100, 2, 3, 32, 48
    c = decay_case(31, dt, B, T, J, H, Dk, Dv)
    ref, mag = decay_reference(c, Dk ** -0.5)
    q, k, v, ld = (c[n].cuda() for n in ('q', 'k', 'v', 'log_decay'))
    tol = decay_tol('o', ref, mag, c)
    state, out = c['state'].cuda(), []
    for a, b in ((0, 1), (1, 33), (33, 33), (33, 97), (97, 100)):
        o, state = tp.decay_attention(q[:, a:b], k[:, a:b], v[:, a:b], ld, state=state, return_state=True)
        out.append(o)
    close(torch.cat(out, 1), ref['o'], tol, 'pieces')
    close(state, ref['state'], decay_tol('state', ref, mag, c), 'state of pieces')
    S = c['state'].cuda()
    out = [tp.decay_attention_step(q[:, t], k[:, t], v[:, t], ld, S) for t in range(T)]
    close(torch.stack(out, 1), ref['o'], tol, 'tokens')
    close(S, ref['state'], decay_tol('state', ref, mag, c), 'state of tokens')


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('B,J,H,Dk,Dv', [(1, 1, 1, 1, 1), (1, 17, 4, 32, 32), (3, 2, 2, 33, 17), (2, 1, 3, 128, 128), (2, 1, 2, 128, 4), (1, 1, 2, 5, 128),
                                         (4, 1, 1, 64, 96), (2, 3, 1, 16, 102)])
def test_decay_step(tp, dt, B, J, H, Dk, Dv):
    c = decay_case(B * 7 + Dk, dt, B, 1, J, H, Dk, Dv)
    lengths = torch.tensor([1, 0, 5, -1][:B], dtype=torch.int32)
    for n in (None, lengths):
        c['lengths'] = n
        ref, mag = decay_reference(c, Dk ** -0.5)
        S = c['state'].cuda()
        o = tp.decay_attention_step(*(c[x][:, 0].cuda() for x in 'qkv'), c['log_decay'].cuda(), S, lengths=None if n is None else n.cuda())
        close(o.unsqueeze(1), ref['o'], decay_tol('o', ref, mag, c), 'o')
        close(S, ref['state'], decay_tol('state', ref, mag, c), 'state')
        for b in range(B):
            if n is not None and n[b] < 1:
                assert torch.equal(S[b].cpu(), c['state'][b]) and not o[b].any()
    if J == 1:
        S4 = c['state'].cuda()
        o4 = tp.decay_attention_step(*(c[x][:, 0, 0].cuda() for x in 'qkv'), c['log_decay'].cuda(), S4, lengths=None if n is None else n.cuda())
        assert torch.equal(o4, o[:, 0]) and torch.equal(S4, S)


def test_decay_empty_calls(tp):
    c = decay_case(41, torch.float32, 2, 3, 1, 2, 8, 8)
    q, k, v, ld, s = (c[n].cuda() for n in ('q', 'k', 'v', 'log_decay', 'state'))
    o, new = tp.decay_attention(q[:, :0], k[:, :0], v[:, :0], ld, state=s, return_state=True)
    assert o.shape == (2, 0, 1, 2, 8) and torch.equal(new, s)
    o, new = tp.decay_attention(q[:, :0], k[:, :0], v[:, :0], ld, return_state=True)
    assert not new.any()
    assert tp.decay_attention(q[:0], k[:0], v[:0], ld).shape == (0, 3, 1, 2, 8)
    assert tp.decay_attention_step(q[:0, 0], k[:0, 0], v[:0, 0], ld, s[:0]).shape == (0, 1, 2, 8)
    # only the state is asked for, or only the outputs
    sd = s.clone().requires_grad_(True)
    _, new = tp.decay_attention(q, k, v, ld, state=sd, return_state=True)
    g, = torch.autograd.grad(new.sum(), sd)
    lam = torch.exp(ld.double() * 3).view(1, 1, 2, 1, 1).expand_as(g).cpu()
    close(g, lam, 32 * U * lam, 'dstate')


# ------------------------------------------------------------------------------------------------ layer norm
def norm_tols(s, weight, bias, eps, dt, dy=None):
    """A value takes part in at most n = 40 + C / 1024 additions of a row's sums (16 in a lane, 6 in a wave, 16 of waves; the longest
    rows are folded by 1024 threads first).  With A = mean |s| the mean is off by at most d = (n + 2) u A; x - mean by d + u |x - mean|;
    the variance relatively by (n + 4) u + (d rstd)^2, rstd by half of that and 4 u.  Results: three roundings more."""
    C = s.shape[-1]
    n = 40 + C / 1024
    y, xhat, rstd = to.layer_norm(s, weight, bias, eps)
    d = (n + 2) * U * s.abs().mean(-1, keepdim=True)
    rr = ((n + 4) * U + (d * rstd) ** 2) / 2 + 4 * U                      # of rstd, relative
    dx = rstd * d + xhat.abs() * (rr + 2 * U)                             # of xhat
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.double().abs()
    h, tiny = half(dt)
    ty = dx * w + 2 * U * (y.abs() + (xhat * w).abs())
    out = dict(y=(y, ty + h * (y.abs() + ty) + tiny))
    if dy is not None:
        ds, dw, db = to.layer_norm_grads(xhat, rstd, weight, dy)
        g = dy.abs() * w
        G, GX = g.mean(-1, keepdim=True), (g * xhat.abs()).mean(-1, keepdim=True)
        t = (n + 4) * U * (g + G + xhat.abs() * GX) + dx * GX + xhat.abs() * (g * dx).mean(-1, keepdim=True)
        td = rstd * (t + rr * (g + G + xhat.abs() * GX))
        out['ds'] = (ds, td)
        # a column's sum has one addition a row at most
        rows = dy[..., 0].numel()
        lead = tuple(range(dy.dim() - 1))
        out['dweight'] = (dw, (rows + 4) * U * (dy * xhat).abs().sum(lead) + (dy.abs() * dx).sum(lead))
        out['dbias'] = (db, (rows + 4) * U * dy.abs().sum(lead))
    return out


WIDTHS = [1, 2, 3, 8, 31, 32, 33, 64, 100, 128, 130, 255, 256, 257, 510, 512, 640, 1000, 1024, 1025, 2048, 2050, 4095, 4096, 4100, 8190, 8192, 16384, 16390, 20001]


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('C', WIDTHS)
def test_layer_norm(tp, dt, C):
    g = gen(C)
    rows = 37 if C < 5000 else 5
    x = randn(g, dt, rows, C, scale=2.0) + torch.tensor(0.5, dtype=dt)
    w, b, dy = torch.randn(C, generator=g) + 1, torch.randn(C, generator=g), randn(g, dt, rows, C)
    tols = norm_tols(x.double(), w, b, 1e-5, dt, dy.double())
    xd, wd, bd = (t.cuda().requires_grad_(True) for t in (x, w, b))
    y = tp.layer_norm(xd, wd, bd, eps=1e-5)
    close(y, *tols['y'], 'y')
    dx, dw, db = torch.autograd.grad(y, [xd, wd, bd], dy.cuda())
    h, tiny = half(dt)
    ds, td = tols['ds']
    close(dx, ds, td + h * (ds.abs() + td) + tiny, 'dx')
    close(dw, *tols['dweight'], 'dweight')
    close(db, *tols['dbias'], 'dbias')


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,C', [(1, 128), (17, 128), (3000, 128), (2050, 33), (700, 1024), (300, 4096), (5, 8192), (3, 20000), (1030, 8), (9, 102)])
@pytest.mark.parametrize('p', [0.0, 0.25, 1.0])
def test_add_layer_norm(tp, dt, rows, C, p):
    from gast_hip.binding import Dropout, dropout_params
    g = gen(rows + C)
    x, r = randn(g, dt, rows, C), randn(g, dt, rows, C, scale=2.0)
    w, b, dy, dst = torch.randn(C, generator=g) + 1, torch.randn(C, generator=g), randn(g, dt, rows, C), randn(g, dt, rows, C)
    thresh, inv_keep = dropout_params(p)
    seed, salt = 12345, 3
    keep = to.drop_keep(seed, thresh, rows * C, salt).view(rows, C).double() * float(torch.tensor(inv_keep)) if p else torch.ones(rows, C, dtype=torch.float64)
    # one rounding to fp32, one to the type: as the operator is defined
    s = (r.double() + x.double() * keep).float().to(dt)
    drop = Dropout(torch.tensor([seed], dtype=torch.int32).cuda(), thresh, inv_keep) if p else None
    xd, rd, wd, bd = (t.cuda().requires_grad_(True) for t in (x, r, w, b))
    y, stream = tp.add_layer_norm(xd, rd, wd, bd, eps=1e-6, drop=drop, salt=salt)
    assert torch.equal(stream.detach().cpu(), s)
    tols = norm_tols(s.double(), w, b, 1e-6, dt, dy.double())
    close(y, *tols['y'], 'y')
    dx, dr, dw, db = torch.autograd.grad([y, stream], [xd, rd, wd, bd], [dy.cuda(), dst.cuda()])
    h, tiny = half(dt)
    ds, td = tols['ds']
    ds = ds + dst.double()
    td = td + U * ds.abs()
    close(dr, ds, td + h * (ds.abs() + td) + tiny, 'dresidual')
    close(dx, ds * keep, (td + U * ds.abs()) * keep + h * ((ds.abs() + td) * keep) + tiny, 'dx')
    assert not dx[keep.cuda() == 0].any()
    close(dw, *tols['dweight'], 'dweight')
    close(db, *tols['dbias'], 'dbias')


@pytest.mark.parametrize('asked', ['x', 'residual', 'weight', 'bias', 'stream only', 'y only'])
def test_add_layer_norm_gives_each_gradient_alone(tp, asked):
    from gast_hip.binding import Dropout, dropout_params
    g = gen(5)
    t = {n: randn(g, torch.float32, *s).cuda() for n, s in (('x', (6, 4, 32)), ('residual', (6, 4, 32)), ('weight', (32,)), ('bias', (32,)))}
    dy, ds = randn(g, torch.float32, 6, 4, 32).cuda(), randn(g, torch.float32, 6, 4, 32).cuda()
    for p in (0.0, 0.5):
        drop = Dropout(torch.tensor([9], dtype=torch.int32).cuda(), *dropout_params(p)) if p else None
        every = {n: v.clone().requires_grad_(True) for n, v in t.items()}
        y, s = tp.add_layer_norm(every['x'], every['residual'], every['weight'], every['bias'], drop=drop)
        if asked == 'stream only':
            a = torch.autograd.grad(s, [every['x'], every['residual']], ds, retain_graph=True)
            assert torch.equal(a[1], ds)
            keep = to.drop_keep(9, 32768, 6 * 4 * 32).view(6, 4, 32).cuda().float() * 2 if p else torch.ones_like(ds)
            assert torch.equal(a[0], ds * keep)
            continue
        if asked == 'y only':
            a = torch.autograd.grad(y, list(every.values()), dy, retain_graph=True)
            c = torch.autograd.grad([y, s], list(every.values()), [dy, torch.zeros_like(ds)])
            assert all(torch.equal(i, j) for i, j in zip(a, c))
            continue
        full = torch.autograd.grad([y, s], [every[asked]], [dy, ds])[0]
        one = {n: v.clone().requires_grad_(n == asked) for n, v in t.items()}
        y, s = tp.add_layer_norm(one['x'], one['residual'], one['weight'], one['bias'], drop=drop)
        outs, gs = ([y, s], [dy, ds]) if asked in ('x', 'residual') else ([y], [dy])
        alone = torch.autograd.grad(outs, [one[asked]], gs)[0]
        assert torch.equal(full, alone)


def test_layer_norm_rows_that_lie_apart_and_odd_calls(tp):
    g = gen(6)
    big = randn(g, torch.float32, 40, 3, 70).cuda()
    for x in (big[:, 1, 3:35], big[..., :64], big[::2, :, 1:], big[:, :, ::2], big[5, 2], big.permute(1, 0, 2), big[:1, :1, :1]):
        y = tp.layer_norm(x)
        ref, tol = norm_tols(x.double().cpu(), None, None, 1e-5, torch.float32)['y']
        close(y, ref, tol, 'y')
    assert tp.layer_norm(big[:0]).shape == (0, 3, 70)
    w = torch.ones(70, device='cuda', requires_grad=True)
    e = big[:0].clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(tp.layer_norm(e, w).sum(), [e, w])
    assert dx.shape == e.shape and not dw.any()
    # a constant row: the variance is 0, what is left is the bias; half-precision weights are converted
    c = torch.full((2, 64), 3.0).cuda()
    assert torch.equal(tp.layer_norm(c, None, torch.arange(64.0).cuda()), torch.arange(64.0).cuda().expand(2, 64))
    hw = torch.ones(70, dtype=torch.bfloat16, device='cuda', requires_grad=True)
    y = tp.layer_norm(big, hw)
    assert torch.equal(y, tp.layer_norm(big))
    assert torch.autograd.grad(y.sum(), hw)[0].dtype == torch.bfloat16


def test_layer_norm_far_from_zero(tp):
    """a mean of 1000 deviations: the variance is that of the centred row, not a difference of squares"""
    g = gen(7)
    x = randn(g, torch.float32, 8, 512) + 1000.0
    ref, tol = norm_tols(x.double(), None, None, 1e-5, torch.float32)['y']
    close(tp.layer_norm(x.cuda()), ref, tol, 'y')


def test_layer_norm_gradient_against_differences(tp):
    """central difference of f = sum(dy y) along a direction v of length 1, step e = 2^-7: the third derivative leaves e^2 |f'''| / 6 with
    |f'''| <= 15 rstd^3 |dy| |w| sqrt(C) (each derivative of xhat brings a factor rstd <= 2 here and products of at most three xhat),
    rounding leaves 64 u |dy| |y| / e"""
    g = gen(8)
    C = 64
    x = randn(g, torch.float32, 1, C)
    x = (x / x.std()).cuda().requires_grad_(True)
    w = torch.ones(C, device='cuda')
    dy = randn(g, torch.float32, 1, C).cuda()
    v = randn(g, torch.float32, 1, C).cuda()
    v = v / v.norm()
    e = 2.0 ** -7

    def f(t):
        return (tp.layer_norm(t, w).double() * dy.double()).sum()

    slope = (f(x.detach() + e * v) - f(x.detach() - e * v)) / (2 * e)
    dx, = torch.autograd.grad(tp.layer_norm(x, w), x, dy)
    n = float(dy.norm())
    assert abs(float(slope - (dx.double() * v.double()).sum())) <= e * e / 6 * 15 * 8 * n * C ** 0.5 + 64 * U * n * C ** 0.5 / e


def test_layer_norm_weight_gradients_are_the_same_bits_every_time(tp):
    g = gen(9)
    x, w, dy = randn(g, torch.float32, 5000, 96).cuda(), torch.ones(96, device='cuda', requires_grad=True), randn(g, torch.float32, 5000, 96).cuda()
    y = tp.layer_norm(x, w)
    first = torch.autograd.grad(y, w, dy, retain_graph=True)[0]
    for _ in range(3):
        assert torch.equal(first, torch.autograd.grad(y, w, dy, retain_graph=True)[0])


# ------------------------------------------------------------------------------------------------ streams, graphs, the block
def together(tp, t, out=None):
    """rotary -> attention -> step on the state -> add + norm, as a model runs them"""
    q, k = tp.rotary((t['q'], t['k']), t['pos'], t['f'])
    o, new = tp.decay_attention(q, k, t['v'], t['ld'], state=t['s'], lengths=t['n'], return_state=True)
    o1 = tp.decay_attention_step(q[:, 0], k[:, 0], t['v'][:, 0], t['ld'], new)
    y, s = tp.add_layer_norm(o, t['v'], t['w'], t['b'])
    return o, new, o1, y, s


def together_inputs(dt, seed, T=70):
    g = gen(seed)
    t = {n: randn(g, dt, 2, T, 3, 4, 32).cuda() for n in 'qkv'}
    t.update(pos=torch.arange(T).cuda(), f=(10000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)).cuda(), ld=torch.tensor([-0.1, -0.01, 0.0, -1.0]).cuda(),
             s=torch.randn(2, 3, 4, 32, 32, generator=g).cuda(), n=torch.tensor([T, T // 2], dtype=torch.int32).cuda(), w=torch.ones(32).cuda(), b=torch.zeros(32).cuda())
    return t


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
def test_captured_and_replayed(tp, dt):
    a = together_inputs(dt, 1)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            together(tp, a)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = together(tp, a)
        for seed in (2, 3, 4):
            b = together_inputs(dt, seed)
            eager = together(tp, b)
            for n in a:
                a[n].copy_(b[n])
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(out, eager):
                assert torch.equal(x, y)


def test_backward_captured_and_replayed(tp):
    from gast_hip.binding import Dropout, dropout_params

    def make(seed):
        t = together_inputs(torch.bfloat16, seed)
        t['seed'] = torch.tensor([seed], dtype=torch.int32).cuda()
        t['do'] = randn(gen(seed + 50), torch.bfloat16, 2, 70, 3, 4, 32).cuda()
        return t

    def step(t):
        leaves = [t[n].detach().requires_grad_(True) for n in ('q', 'k', 'v', 's', 'w', 'b')]
        q, k, v, s, w, b = leaves
        qr, kr = tp.rotary((q, k), t['pos'], t['f'])
        o = tp.decay_attention(qr, kr, v, t['ld'], state=s, lengths=t['n'])
        y, st = tp.add_layer_norm(o, v, w, b, drop=Dropout(t['seed'], *dropout_params(0.25)))
        return torch.autograd.grad([y, st], leaves, [t['do'], t['do']])

    a = make(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(a)
    for seed in (2, 3, 4):
        b = make(seed)
        eager = step(b)
        for n in a:
            a[n].copy_(b[n])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, eager):
            assert torch.equal(x, y)


def test_two_streams_at_once(tp):
    """calls in flight on two streams share nothing"""
    sets = [together_inputs(torch.bfloat16, s, T=600) for s in (5, 6)]
    with torch.no_grad():
        want = [together(tp, t) for t in sets]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in sets]
        for _ in range(4):
            got = []
            for st, t in zip(streams, sets):
                with torch.cuda.stream(st):
                    got.append(together(tp, t))
            torch.cuda.synchronize()
            for g, w in zip(got, want):
                assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_offsets_that_pass_32_bits(tp):
    """tokens, rows and states further than 2^32 bytes and 2^31 elements from the first one"""
    g = gen(61)
    dt, T, H, D = torch.bfloat16, 40, 2, 16
    c = decay_case(61, dt, 1, T, 1, H, D, D)
    far = torch.empty(T, 2 ** 26, dtype=dt, device='cuda')                # a token every 2^27 bytes
    views = {}
    for i, n in enumerate(('q', 'k', 'v', 'do')):
        views[n] = far[:, i * 64:i * 64 + H * D].view(1, T, 1, H, D)
        views[n].copy_(c[n])
    check_decay(tp, c, views={n: t.detach() for n, t in views.items()})
    pos, f = torch.arange(T).view(1, T), tp.rotary_frequencies(D)
    close(tp.rotary(views['q'].detach(), pos.cuda(), f.cuda()), *rotary_tol(c['q'], pos, f, False, 1.0, dt), 'rotary')
    del far, views
    # 2^31 elements and more
    rows, C = 2 ** 19 + 3, 4096
    x = torch.zeros(rows, C, dtype=dt, device='cuda')
    tail = randn(g, dt, 5, C)
    x[-5:] = tail.cuda()
    x.requires_grad_(True)
    y = tp.layer_norm(x)
    tols = norm_tols(tail.double(), None, None, 1e-5, dt, tail.double())
    close(y[-5:], *tols['y'], 'y')
    assert not y[:-5].any()
    dx, = torch.autograd.grad(y, x, x.detach())
    h, tiny = half(dt)
    ds, td = tols['ds']
    close(dx[-5:], ds, td + h * (ds.abs() + td) + tiny, 'dx')
    del x, y, dx
    B, H, D = 1025, 128, 128                                              # a state of 2^31 elements and more
    S = torch.zeros(B, 1, H, D, D, device='cuda')
    c = decay_case(62, dt, 1, 1, 1, H, D, D)
    S[-1] = c['state'][0].cuda()
    q, k, v = (torch.zeros(B, 1, H, D, dtype=dt, device='cuda') for _ in range(3))
    for a, n in ((q, 'q'), (k, 'k'), (v, 'v')):
        a[-1] = c[n][0, 0].cuda()
    ref, mag = decay_reference(c, D ** -0.5)
    new = tp.decay_attention(q.unsqueeze(1), k.unsqueeze(1), v.unsqueeze(1), c['log_decay'].cuda(), state=S, return_state=True)[1]
    close(new[-1:], ref['state'], decay_tol('state', ref, mag, c), 'new state')
    o = tp.decay_attention_step(q, k, v, c['log_decay'].cuda(), S)
    close(o[-1:].unsqueeze(1), ref['o'], decay_tol('o', ref, mag, c), 'o')
    close(S[-1:], ref['state'], decay_tol('state', ref, mag, c), 'state')
    assert not S[:-1].any() and not new[:-1].any()


def test_second_derivatives_are_refused(tp):
    t = together_inputs(torch.float32, 9)
    calls = dict(rotary=lambda x: tp.rotary(x, t['pos'], t['f']), decay=lambda x: tp.decay_attention(x, t['k'], t['v'], t['ld']),
                 norm=lambda x: tp.layer_norm(x, t['w'], t['b']), add=lambda x: tp.add_layer_norm(x, t['v'], t['w'], t['b'])[0])
    for name, f in calls.items():
        x = t['q'].detach().requires_grad_(True)
        g, = torch.autograd.grad((f(x) ** 2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


def block_reference(mod, x, lengths):
    """TemporalAttention in 64 bits on the host, gradients through torch's autograd"""
    B, T, J, C = x.shape
    H = mod.heads
    D = C // H
    p = {n: t.detach().double().cpu().requires_grad_(True) for n, t in mod.named_parameters()}
    x = x.double().requires_grad_(True)
    with torch.enable_grad():
        qkv = (x @ p['qkv.weight'].t() + p['qkv.bias']).view(B, T, J, 3, H, D)
        q, k, v = qkv.unbind(3)
        ang = torch.arange(T).double()[:, None] * mod._freqs.cpu()
        cos, sin = (f(ang)[None, :, None, None] for f in (torch.cos, torch.sin))
        r = lambda z: torch.cat([z[..., :D // 2] * cos - z[..., D // 2:] * sin, z[..., :D // 2] * sin + z[..., D // 2:] * cos], -1)  # noqa: E731
        o, _ = to.decay(r(q), r(k), v, mod.log_decay.cpu(), None, lengths, D ** -0.5)
        s = x + o.reshape(B, T, J, C) @ p['out.weight'].t() + p['out.bias']
        y, _, _ = to.layer_norm(s, p['norm.weight'], p['norm.bias'], mod.norm.eps)
    return x, p, y


def test_temporal_attention_block(tp):
    """fp32 through three GEMMs, the attention and the norm: every stage is good to n u of its absolute terms, n below 400 here, and the
    norm divides by a deviation near 1: 1e-4 of the largest value covers 1600 u; so for the gradients"""
    from model.temporal_attention import TemporalAttention
    torch.manual_seed(3)
    mod = TemporalAttention(64, heads=4).cuda()
    x = torch.randn(2, 45, 5, 64, generator=gen(1))
    lengths = torch.tensor([45, 20], dtype=torch.int32)
    dy = torch.randn(2, 45, 5, 64, generator=gen(2))
    xr, pr, yr = block_reference(mod, x, lengths)
    gr = torch.autograd.grad(yr, [xr] + list(pr.values()), dy.double())
    xd = x.cuda().requires_grad_(True)
    y = mod(xd, lengths.cuda())
    g = torch.autograd.grad(y, [xd] + list(mod.parameters()), dy.cuda())
    for name, a, b in zip(['y', 'x'] + list(pr), (y,) + g, (yr,) + gr):
        close(a, b, 1e-4 * float(b.detach().abs().max()), name)


def test_temporal_attention_streams_what_it_computes_at_once(tp):
    from model.temporal_attention import TemporalAttention
    torch.manual_seed(4)
    mod = TemporalAttention(32, heads=2, dropout=0.3, rotary_dim=8).cuda().eval()
    x = torch.randn(3, 30, 2, 32, generator=gen(3)).cuda()
    with torch.no_grad():
        whole = mod(x)
        state = mod.state(3, 2)
        out = []
        for t in range(30):
            if t % 7 == 3:          # a tick without a frame for any stream
                before = state.S.clone()
                mod.step(x[:, 0], state, active=torch.zeros(3, dtype=torch.int32).cuda())
                assert torch.equal(before, state.S)
            out.append(mod.step(x[:, t], state))
    close(torch.stack(out, 1), whole.double().cpu(), 1e-4 * float(whole.abs().max()), 'stream')
    assert state.position.flatten().tolist() == [30] * 3
    s2 = mod.state(3, 2)
    active = torch.tensor([1, 0, 1], dtype=torch.int32).cuda()
    mod.step(x[:, 0], s2, active=active)
    assert s2.position.flatten().tolist() == [1, 0, 1] and not s2.S[1].any() and s2.S[0].any()


def test_temporal_attention_trains_with_dropout(tp):
    from model.temporal_attention import TemporalAttention
    torch.manual_seed(5)
    mod = TemporalAttention(32, heads=2, dropout=0.5).cuda().train()
    x = torch.randn(2, 10, 3, 32, generator=gen(4)).cuda().requires_grad_(True)
    a, b = mod(x), mod(x)
    assert not torch.equal(a, b)                     # a mask of its own each call
    a.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in mod.parameters()) and torch.isfinite(x.grad).all()
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        TemporalAttention(32)(torch.zeros(1, 2, 3, 32))
