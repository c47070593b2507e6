"""How many bits decay_attention keeps in bfloat16: outputs and gradients are rounded once, states are float32 (the criteria and the
forms that fail them: test_sequence_precision_host.py)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import sequence_reference as ref  # noqa: E402
from test_gpu_sequence import make, rand  # noqa: E402
from gym_fishing_amd import sequence  # noqa: E402

pytestmark = pytest.mark.gpu

CASES = [  # batch, steps, heads, dk, dv, time_major, starts, state
    (5, 101, 4, 64, 64, True, 0.02, True), (1, 700, 2, 128, 128, False, 0.0, True), (2, 257, 3, 48, 80, True, 0.02, True), (3, 130, 3, 40, 72, False, 0.02, False),
    (2, 90, 3, 33, 65, True, 0.02, True), (1, 700, 2, 33, 65, True, 0.005, True), (600, 5, 4, 32, 32, False, 0.2, True), (1100, 5, 4, 32, 32, False, 0.2, True),
    (500, 5, 4, 32, 32, False, 0.2, True)]


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("batch,steps,heads,dk,dv,time_major,starts,state", CASES)
def test_outputs_are_rounded_once_and_states_are_float32(batch, steps, heads, dk, dv, time_major, starts, state, far):
    q, k, v, ld, cut, s0, g, gs = make(batch, steps, heads, dk, dv, torch.bfloat16, time_major, starts, state, seed=steps + dv)
    if far:                                              # horizons of hundreds of steps: most of an output comes from the state
        ld = ld / 64
    leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([s0.requires_grad_()] if state else [])
    got = sequence.decay_attention(*leaves[:3], ld, starts=cut, state=leaves[3] if state else None, scale=0.3, return_state=state)
    grads = torch.autograd.grad(got, leaves, [g, gs] if state else g)
    want = ref.attention(q, k, v, ld, cut, s0, 0.3, g, gs)
    for name, x in zip(("out", "dq", "dk", "dv"), (got[0] if state else got, *grads)):
        ref.check_once_rounded(x, want[name], name)
    if state:
        size = ref.attention(q.abs(), k.abs(), v.abs(), ld, cut, s0.abs(), 0.3, g.abs(), gs.abs())
        ref.check(got[1], want["state"], ref.state_bound(size["state"], steps), "state")
        ref.check(grads[3], want["dstate"], ref.state_bound(size["dstate"], steps), "dstate")


@pytest.mark.parametrize("dk,dv", [(64, 64), (48, 112), (33, 65)])
@pytest.mark.parametrize("steps", [32, 704])
def test_states_that_nothing_decays_are_float32_sums(steps, dk, dv):
    """Whole and in segments, whose states the gradient's walk takes over from another's."""
    q, k, v, _, _, s0, g, gs = make(1, steps, 2, dk, dv, torch.bfloat16, False, 0.0, True, seed=dk)
    ld = torch.zeros(2, device="cuda")
    leaf, s0 = q.detach().requires_grad_(), s0.requires_grad_()
    out, last = sequence.decay_attention(leaf, k, v, ld, state=s0, scale=0.3, return_state=True)
    dstate = torch.autograd.grad((out, last), s0, (g, gs))[0]
    want = ref.attention(q, k, v, ld, None, s0, 0.3, g, gs)
    ref.check_state_norm(last, want["state"], steps, "state")
    ref.check_state_norm(dstate, want["dstate"], steps, "dstate")


@pytest.mark.parametrize("rows,levels,dim,most", [(4096, 100, 64, 1.6), (2050, 1009, 200, 1.6), (17, 4097, 512, 2.2)])
def test_loss_gradients_are_rounded_twice(rows, levels, dim, most):
    """dz, a factor of both products, is rounded once, and each gradient once: two roundings of one size that do not know of each
    other make sqrt 2 times one's error in the 2-norm (and a tenth for the norm of few values).  A row whose gradient is mostly its target's
    term takes that term's one error in every column: at worst 2^-8 where the columns' own is 2^-8 / sqrt 3 in the mean, so twice, and a tenth."""
    hidden = rand(rows, dim, seed=1, dtype=torch.bfloat16).requires_grad_()
    head = rand(levels, dim, seed=2, dtype=torch.bfloat16, scale=1.5 * dim ** -0.5).requires_grad_()
    target = torch.randint(0, levels, (rows,), generator=torch.Generator().manual_seed(3)).cuda()
    grad = rand(rows, seed=4)
    got = torch.autograd.grad(sequence.cross_entropy(hidden, head, target), (hidden, head), grad)
    want, _ = ref.loss(hidden, head, target, grad)
    for name, x in zip(("dhidden", "dhead"), got):
        once = (want[name].to(torch.bfloat16).double() - want[name]).norm()
        assert (x.cpu().double() - want[name]).norm() <= most * once, name
