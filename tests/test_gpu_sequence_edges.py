"""The sequence operators where their forms have to agree with each other, and what they refuse or leave alone."""
import os
import sys

import pytest
import torch
from torch.autograd import forward_ad

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import sequence_reference as ref  # noqa: E402
from test_gpu_sequence import make, rand  # noqa: E402
from gym_fishing_amd import sequence  # noqa: E402

pytestmark = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("batch,dk,dv", [(3, 32, 32), (2, 33, 7), (700, 16, 48)])
def test_a_decay_of_zero_lets_nothing_through_not_even_nan(batch, dk, dv, dtype):
    """By the step as over whole sequences, for none at all (-inf) and for one that float32 cannot hold; a decay that is left does."""
    q, k, v, _, _, s0, _, _ = make(batch, 1, 4, dk, dv, dtype, False, 0.0, True, seed=dk)
    ld = torch.tensor([float("-inf"), -200.0, -1.0, -0.1], device="cuda")
    s0[:, :2, 0], s0[:, :2, 1], s0[0, 3] = float("nan"), float("inf"), float("nan")
    whole, last = sequence.decay_attention(q, k, v, ld, state=s0, scale=0.5, return_state=True)
    state = s0.clone()
    out = sequence.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state, scale=0.5)
    clean = torch.where(torch.isfinite(s0), s0, torch.zeros((), device="cuda"))
    clean[:, :2] = 0.0
    args = (q, k, v, torch.tensor([-200.0, -200.0, -1.0, -0.1], device="cuda"), None, clean, 0.5)
    want, bound = ref.attention(*args), ref.attention_bounds(*args)
    for got, what in ((whole[:, 0], "whole"), (out, "step")):
        ref.check(got[:, :3], want["out"][:, 0, :3], bound["out"][:, 0, :3], what)
        ref.check(got[1:, 3], want["out"][1:, 0, 3], bound["out"][1:, 0, 3], what)
        assert torch.isnan(got[0, 3]).all()
    for got, what in ((last, "whole"), (state, "step")):
        ref.check(got[:, :3], want["state"][:, :3], bound["state"][:, :3], what)
        assert torch.isnan(got[0, 3]).all()


def test_forward_mode_tangents_are_refused_in_every_operand_and_gradient():
    q, k, v, ld, _, s0, g, gs = make(2, 5, 2, 8, 12, torch.float32, False, 0.0, True)
    table, hidden, head, i = rand(5, 8), rand(3, 8), rand(5, 8), torch.zeros(3, dtype=torch.int64, device="cuda")
    calls = [(sequence.embedding, dict(tokens=i, table=table)), (sequence.cross_entropy, dict(hidden=hidden, head=head, target=i)),
             (sequence.decay_attention, dict(q=q, k=k, v=v, log_decay=ld, state=s0)),
             (sequence.decay_attention_step, dict(q=q[:, 0], k=k[:, 0], v=v[:, 0], log_decay=ld, state=s0, state_out=s0.clone(), out=g[:, 0].contiguous()))]
    for f, kw in calls:
        for name, x in kw.items():
            if x.is_floating_point():
                with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                    f(**{**kw, name: forward_ad.make_dual(x, torch.ones_like(x))})
    t, w, h = table.requires_grad_(), head.requires_grad_(), hidden.requires_grad_()
    leaf = q.detach().requires_grad_()
    with forward_ad.dual_level():
        out, last = sequence.decay_attention(leaf, k, v, ld, state=s0, return_state=True)
        for y, x in ((sequence.embedding(i, t), t), (sequence.cross_entropy(h, w, i), w), (out, leaf), (last, leaf)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, x, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)
            assert torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)[0].shape == x.shape
