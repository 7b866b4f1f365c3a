"""The kernel variants of the sequence operators that sizes alone choose, at the smallest sizes that reach them, and calls whose
uninitialised memory holds NaN.  Tolerances: those of test_temporal_gpu.py."""
import pytest
import torch
from test_temporal_gpu import (IDS, TYPES, check_decay, close, decay_case, decay_reference, decay_tol, gen, half, norm_tols, randn, rotary_tol)

from oracle import temporal_oracle as to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def tp():
    from gast_hip import temporal
    return temporal


# ------------------------------------------------------------------------------------------------ one token: several heads a block
@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('off', [0, 1], ids=['aligned', 'unaligned'])
@pytest.mark.parametrize('B,J,H,Dk,Dv', [(205, 1, 5, 16, 16), (205, 1, 5, 15, 17), (342, 1, 3, 32, 32), (61, 17, 1, 8, 8), (1024, 1, 1, 1, 1), (103, 5, 2, 4, 64), (257, 4, 1, 128, 2)])
def test_steps_of_many_small_states(tp, dt, off, B, J, H, Dk, Dv):
    """1024 heads and more, four to a block: a last block that is not full, streams without a token between others"""
    c = decay_case(B + Dk, dt, B, 1, J, H, Dk, Dv)
    n = torch.randint(0, 2, (B,), generator=gen(B), dtype=torch.int32)
    n[0], n[-1] = 0, 1
    for lengths in (None, n):
        c['lengths'] = lengths
        ref, mag = decay_reference(c, Dk ** -0.5)
        guard = torch.full((off + c['state'].numel() + 64,), 7.0, device='cuda')
        S = guard[off:off + c['state'].numel()].view(c['state'].shape)
        S.copy_(c['state'])
        o = tp.decay_attention_step(*(c[x][:, 0].cuda() for x in 'qkv'), c['log_decay'].cuda(), S, lengths=None if lengths is None else lengths.cuda())
        close(o.unsqueeze(1), ref['o'], decay_tol('o', ref, mag, c), 'o')
        close(S, ref['state'], decay_tol('state', ref, mag, c), 'state')
        assert torch.all(guard[:off] == 7) and torch.all(guard[off + c['state'].numel():] == 7)
        if lengths is not None:
            off_streams = n == 0
            assert torch.equal(S.cpu()[off_streams], c['state'][off_streams]) and not o.cpu()[off_streams].any()


# ------------------------------------------------------------------------------------------------ rotary: one block for all tensors
@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('interleaved', [False, True], ids=['half', 'pairs'])
@pytest.mark.parametrize('B,T,J,Hq,Hk,D,R', [(2, 22001, 1, 2, 1, 14, 14), (6300, 7, 1, 1, 2, 16, 10), (1, 70000, 1, 1, 1, 64, 64), (3, 4100, 4, 1, 1, 9, 6)])
def test_rotary_of_many_tokens_and_few_heads(tp, dt, interleaved, B, T, J, Hq, Hk, D, R):
    """the cosines of a block serve every tensor of the call, heads of their own each, and more than 16 tokens"""
    g = gen(B + T)
    q, k = randn(g, dt, B, T, J, Hq, D), randn(g, dt, B, T, J, Hk, D)
    pos = torch.randint(-1000, 1000000, (B, T), generator=g)
    f = tp.rotary_frequencies(R)
    xs = [t.cuda().requires_grad_(True) for t in (q, k)]
    ys = tp.rotary(tuple(xs), pos.cuda(), f.cuda(), interleaved=interleaved)
    ds = [randn(g, dt, *t.shape) for t in (q, k)]
    back = torch.autograd.grad(ys, xs, [d.cuda() for d in ds])
    for x, y, d, b in zip((q, k), ys, ds, back):
        close(y, *rotary_tol(x, pos, f, interleaved, 1.0, dt), 'y')
        close(b, *rotary_tol(d, pos, f, interleaved, 1.0, dt, back=True), 'dx')


# ------------------------------------------------------------------------------------------------ heads shorter than a vector
@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('state', [False, True], ids=['fresh', 'going on'])
@pytest.mark.parametrize('T', [1, 2, 27, 32])
@pytest.mark.parametrize('Dk,Dv', [(1, 1), (3, 3), (7, 7), (3, 40), (40, 7), (1, 64), (64, 2)])
def test_short_heads_in_sequences_of_one_chunk(tp, dt, state, T, Dk, Dv):
    """read element by element, in the kernels without a state too"""
    c = decay_case(T + Dk, dt, 3, T, 2, 2, Dk, Dv, state=state)
    check_decay(tp, c)
    if not state:                        # no state at either end: nothing returned
        c['lengths'] = torch.tensor([T, T // 2, 0], dtype=torch.int32)
        ref, mag = decay_reference(c, Dk ** -0.5)
        t = [c[n].cuda().requires_grad_(True) for n in 'qkv']
        o = tp.decay_attention(*t, c['log_decay'].cuda(), lengths=c['lengths'].cuda())
        got = dict(zip(('o', 'dq', 'dk', 'dv'), (o,) + torch.autograd.grad(o, t, c['do'].cuda())))
        for n, x in got.items():
            close(x, ref[n], decay_tol(n, ref, mag, c), n)


# ------------------------------------------------------------------------------------------------ memory that nobody has written
@pytest.fixture
def poisoned():
    """torch.empty and at::empty of the device give NaN (integers: the largest)"""
    was = torch.are_deterministic_algorithms_enabled(), torch.is_deterministic_algorithms_warn_only_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    torch.use_deterministic_algorithms(True, warn_only=True)
    torch.utils.deterministic.fill_uninitialized_memory = True
    assert torch.empty(1000, device='cuda').isnan().all()
    yield
    torch.use_deterministic_algorithms(was[0], warn_only=was[1])
    torch.utils.deterministic.fill_uninitialized_memory = was[2]


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('B,T,H,Dk,Dv,ragged', [(3, 1, 2, 8, 8, True), (3, 27, 2, 32, 48, True), (2, 70, 2, 5, 128, False), (1, 1500, 2, 16, 16, False), (4, 700, 1, 64, 40, True),
                                                (2, 2050, 1, 128, 128, True)])
def test_attention_reads_nothing_unwritten(tp, poisoned, dt, B, T, H, Dk, Dv, ragged):
    """segments without tokens, sums that nobody needs, states in place of sums: outputs, gradients and workspaces start as NaN"""
    c = decay_case(B + T, dt, B, T, 1, H, Dk, Dv, ragged=ragged)
    check_decay(tp, c)
    check_decay(tp, dict(c, state=None, dstate=None))
    t = [c[n].cuda().requires_grad_(True) for n in 'qkv']
    n = None if c['lengths'] is None else c['lengths'].cuda()
    o = tp.decay_attention(*t, c['log_decay'].cuda(), lengths=n)
    ref, mag = decay_reference(dict(c, state=None, dstate=None), Dk ** -0.5)
    for name, x in zip(('o', 'dq', 'dk', 'dv'), (o,) + torch.autograd.grad(o, t, c['do'].cuda())):
        close(x, ref[name], decay_tol(name, ref, mag, c), name)
    S = c['state'].cuda()
    one = dict(c, lengths=None if n is None else c['lengths'].clamp(max=1), **{x: c[x][:, :1] for x in ('q', 'k', 'v', 'do')})
    ref, mag = decay_reference(one, Dk ** -0.5)
    close(tp.decay_attention_step(*(c[x][:, 0].cuda() for x in 'qkv'), c['log_decay'].cuda(), S, lengths=n).unsqueeze(1), ref['o'], decay_tol('o', ref, mag, one), 'step')
    close(S, ref['state'], decay_tol('state', ref, mag, one), 'state')


@pytest.mark.parametrize('dt', TYPES, ids=IDS)
@pytest.mark.parametrize('rows,C', [(1, 1), (9, 7), (37, 128), (3000, 33), (1500, 1024), (300, 4100), (5, 20001)])
def test_norm_and_rotary_read_nothing_unwritten(tp, poisoned, dt, rows, C):
    from gast_hip.binding import Dropout, dropout_params
    g = gen(rows + C)
    x, r, dy, ds = (randn(g, dt, rows, C) for _ in range(4))
    w, b = torch.randn(C, generator=g) + 1, torch.randn(C, generator=g)
    thresh, inv_keep = dropout_params(0.25)
    keep = to.drop_keep(7, thresh, rows * C).view(rows, C).double() * float(torch.tensor(inv_keep))
    s = (r.double() + x.double() * keep).float().to(dt)
    t = [v.cuda().requires_grad_(True) for v in (x, r, w, b)]
    y, stream = tp.add_layer_norm(*t, eps=1e-5, drop=Dropout(torch.tensor([7], dtype=torch.int32).cuda(), thresh, inv_keep))
    tols = norm_tols(s.double(), w, b, 1e-5, dt, dy.double())
    assert torch.equal(stream.detach().cpu(), s)
    close(y, *tols['y'], 'y')
    dx, dr, dw, db = torch.autograd.grad([y, stream], t, [dy.cuda(), ds.cuda()])
    h, tiny = half(dt)
    ref, td = tols['ds']
    ref, td = ref + ds.double(), td + 2.0 ** -24 * (ref + ds.double()).abs()
    close(dr, ref, td + h * (ref.abs() + td) + tiny, 'dresidual')
    close(dx, ref * keep, (td + 2.0 ** -24 * ref.abs()) * keep + h * ((ref.abs() + td) * keep) + tiny, 'dx')
    close(dw, *tols['dweight'], 'dweight')
    close(db, *tols['dbias'], 'dbias')
    if C >= 2 and C <= 1024:
        x = randn(g, dt, 1, rows, 1, 2, C)
        pos, f = torch.arange(rows).view(1, rows), tp.rotary_frequencies(C // 2 * 2)
        close(tp.rotary(x.cuda(), pos.cuda(), f.cuda()), *rotary_tol(x, pos, f, False, 1.0, dt), 'rotary')
