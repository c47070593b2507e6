"""What tests/test_gpu_sequence_precision.py holds decay_attention to, tried on the CPU against forms that keep too few bits: a
correct form has to pass it and each of them has to fail it."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import sequence_reference as ref  # noqa: E402


def short(x):
    return x.to(torch.bfloat16).to(x.dtype)


def walk(q, k, v, ld, scale, state=None, kept=lambda s: s, read=lambda s: s):
    """The recurrence in 64 bits, with a rounding of the state that is kept (`kept`) or of the copy that is read (`read`)."""
    q, k, v = (x.double() for x in (q, k, v))
    S = torch.zeros(q.shape[0], q.shape[2], q.shape[3], v.shape[3], dtype=torch.float64) if state is None else state.double()
    a, outs = torch.exp(ld.double())[None, :, None, None], []
    for t in range(q.shape[1]):
        S = kept(S * a + k[:, t, :, :, None] * v[:, t, :, None, :])
        outs.append(scale * (q[:, t, :, None, :] @ read(S)).squeeze(2))
    return torch.stack(outs, 1).to(torch.bfloat16), S.float()


def scored(q, k, v, ld, scale, terms):
    """The same as weighted scores times v, the scores as this many bfloat16 terms."""
    q, k, v = (x.double().transpose(1, 2) for x in (q, k, v))
    i = torch.arange(q.shape[2])
    apart = (i[:, None] - i[None, :]).clamp(min=0)
    z = (q @ k.transpose(2, 3)) * torch.exp(apart * ld.double()[:, None, None]) * (i[:, None] >= i[None, :]) * scale
    kept = torch.zeros_like(z)
    for _ in range(terms):
        kept = kept + short(z - kept)
    return (kept @ v).transpose(1, 2).to(torch.bfloat16)


@pytest.mark.parametrize("steps,d", [(101, 64), (700, 32)])
def test_forms_with_too_few_bits_fail_and_one_with_enough_passes(steps, d):
    g = torch.Generator().manual_seed(steps)
    q, k, v = (torch.randn((1, steps, 2, d), generator=g).to(torch.bfloat16) for _ in range(3))
    s0 = torch.randn((1, 2, d, d), generator=g)
    ld = torch.tensor([-0.3, -0.01])
    want = ref.attention(q, k, v, ld, None, s0, 0.3)
    out, state = walk(q, k, v, ld, 0.3, s0)
    ref.check_once_rounded(out, want["out"], "out")
    size = ref.attention(q.abs(), k.abs(), v.abs(), ld, None, s0.abs(), 0.3)["state"]
    ref.check(state, want["state"], ref.state_bound(size, steps), "state")
    two = walk(q, k, v, ld, 0.3, s0, read=lambda s: short(s) + short(s - short(s)))[0]
    ref.check_once_rounded(two, want["out"], "a copy of 16 bits")
    for what, bad in (("the state kept in bfloat16", dict(kept=short)), ("a copy of the state in bfloat16", dict(read=short))):
        out, state = walk(q, k, v, ld, 0.3, s0, **bad)
        with pytest.raises(AssertionError):
            ref.check_once_rounded(out, want["out"], what)
        if "kept" in bad:
            with pytest.raises(AssertionError):
                ref.check(state, want["state"], ref.state_bound(size, steps), what)
    with pytest.raises(AssertionError):          # the decayed v as two terms where the state is an answer
        ref.check(want["state"] * (1 + 2.0 ** -17), want["state"], ref.state_bound(want["state"].abs(), 8), "two terms")
    want = ref.attention(q, k, v, ld, None, None, 0.3)["out"]
    ref.check_once_rounded(scored(q, k, v, ld, 0.3, 2), want, "scores of 16 bits")
    with pytest.raises(AssertionError):
        ref.check_once_rounded(scored(q, k, v, ld, 0.3, 1), want, "scores of 8 bits")


def test_a_state_made_of_terms_of_16_bits_fails():
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn((704, 64), generator=g).to(torch.bfloat16) for _ in range(2))
    w = v.float() * 0.3
    want = k.double().t() @ v.double() * 0.3
    S = torch.zeros((64, 64))
    for t in range(704):
        S = S + k[t].float()[:, None] * w[t][None]
    ref.check_state_norm(S, want, 704)
    two = short(w) + short(w - short(w))
    with pytest.raises(AssertionError):
        ref.check_state_norm(k.double().t() @ two.double(), want, 704)
