"""Calls that the documentation of gast_hip.temporal allows, beside those of sizes and types."""
import math

import pytest
import torch
from test_temporal_gpu import check_decay, decay_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def tp():
    from gast_hip import temporal
    return temporal


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def test_inference_with_decays_that_are_a_parameter(tp):
    q, k, v, s = randn(2, 9, 1, 3, 8, seed=1), randn(2, 9, 1, 3, 8, seed=2), randn(2, 9, 1, 3, 16, seed=3), randn(2, 1, 3, 8, 16, seed=4)
    ld = torch.nn.Parameter(torch.tensor([-0.1, -0.01, 0.0]).cuda())
    with torch.no_grad():
        got = tp.decay_attention(q, k, v, ld, state=s, return_state=True)
        want = tp.decay_attention(q, k, v, ld.detach(), state=s, return_state=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        s1, s2 = s.clone(), s.clone()
        assert torch.equal(tp.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s1), tp.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld.detach(), s2))
        assert torch.equal(s1, s2)


def test_a_step_leaves_a_strided_state_alone(tp):
    q, k, v = randn(2, 1, 2, 4, seed=1), randn(2, 1, 2, 4, seed=2), randn(2, 1, 2, 5, seed=3)
    buf = randn(2, 1, 2, 5, 4, seed=4)
    was = buf.clone()
    with pytest.raises(ValueError, match='has to be contiguous'):
        tp.decay_attention_step(q, k, v, torch.zeros(2).cuda(), buf.transpose(3, 4))
    assert torch.equal(buf, was)
    wide = randn(2, 1, 2, 4, 10, seed=5)
    was = wide.clone()
    with pytest.raises(ValueError, match='has to be contiguous'):
        tp.decay_attention_step(q, k, v, torch.zeros(2).cuda(), wide[..., ::2])
    assert torch.equal(wide, was)


@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('T,grows', [(1, [5.0]), (2, [10.0, 5.0]), (7, [5.0, -0.1]), (20, [4.0, 3.0]), (27, [3.0])])
@pytest.mark.parametrize('D', [16, 72])
def test_strongly_growing_states_of_short_sequences(tp, dt, T, grows, D):
    """lambda^31 is no fp32 number, but nobody is 31 tokens away (tolerances: decay_tol; binary16 cannot hold the results)"""
    for state in (False, True):
        check_decay(tp, decay_case(T, dt, 2, T, 1, 2, D, D, state=state, decays=grows))
    c = decay_case(T, dt, 3, 100, 1, 2, D, D, decays=grows)
    c['lengths'] = torch.tensor([T, T // 2, 0], dtype=torch.int32)
    check_decay(tp, c)


@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16, torch.float16], ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('T,Dk,Dv', [(1, 32, 32), (27, 64, 64), (32, 48, 16), (9, 3, 64), (31, 33, 5), (5, 1, 1)])
def test_sequences_of_one_chunk_that_go_on_from_a_state(tp, dt, T, Dk, Dv):
    """their backward pass is one launch whose waves share their tiles"""
    c = decay_case(T, dt, 7, T, 2, 3, Dk, Dv, ragged=True)
    first = check_decay(tp, c)
    for _ in range(3):
        again = check_decay(tp, c)
        assert all(torch.equal(first[n], again[n]) for n in first)


@pytest.mark.parametrize('layout', ['half', 'pairs'])
@pytest.mark.parametrize('around', [0.0, 0.25, 0.5, 0.75, 1.0, 1000.5])
def test_rotations_near_quarter_turns_keep_the_bits_of_what_is_small(tp, layout, around):
    """(1, 0) turned by `around` -+ 2^-20 turns: cosine and sine are each good to 2 steps of fp32 (4 u) of themselves, a correction, the scale
    and the product with 1 round once more (3 u), and the angle is off by 2 pi turns 2^-51; 8 u of the value, where u is 2^-24"""
    g = torch.Generator().manual_seed(int(around * 4))
    turns = around + (torch.rand(64, generator=g, dtype=torch.float64) - 0.5) * 2.0 ** -19
    f = turns * (2 * math.pi)
    x = torch.zeros(1, 2, 1, 1, 128)
    a = torch.arange(0, 128, 2) if layout == 'pairs' else torch.arange(64)
    b = a + 1 if layout == 'pairs' else a + 64
    x[..., a] = 1.0
    y = tp.rotary(x.cuda(), torch.tensor([1, -1]).cuda(), f.cuda(), interleaved=layout == 'pairs')[0, :, 0, 0].double().cpu()
    for t, sign in ((0, 1), (1, -1)):
        for at, ref in ((a, torch.cos(sign * f)), (b, torch.sin(sign * f))):
            assert torch.all((y[t, at] - ref).abs() <= 8 * 2.0 ** -24 * ref.abs() + 6.3 * (around + 1) * 2.0 ** -51)
