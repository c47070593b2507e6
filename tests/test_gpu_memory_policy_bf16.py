"""policies.memory acting in bfloat16: the logits of every step against the network in 64 bits, and the simulate helpers."""
import numpy as np
import pytest
import torch

import gym_fishing_amd as gf
from gym_fishing_amd import policies, rollout

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8                                          # the most a rounding to bfloat16 is off by, relative


def predict_and_logits(m, *args, **kw):
    seen, real = {}, torch.Tensor.argmax

    def grab(self, *a, **k):
        seen["logits"] = self
        return real(self, *a, **k)
    torch.Tensor.argmax = grab
    try:
        action, state = m.predict(*args, **kw)
    finally:
        torch.Tensor.argmax = real
    return action, state, seen["logits"]


@pytest.mark.parametrize("env_id", ["fishing-v0", "fishing-v1", "fishing-v4"])
def test_every_step_is_the_network(env_id):
    env = gf.make(env_id, num_envs=48, seed=3, Tmax=9)
    m = policies.memory(env, dim=32, heads=2, head_dim=16, bins=64, levels=21, dtype=torch.bfloat16, seed=1)
    out, head = (m.params[k].detach().double() for k in ("out", "head"))
    obs, state, done = env.reset(), None, None
    S = torch.zeros((48, 2, 16, 16), dtype=torch.float64, device="cuda")
    size, last = torch.zeros_like(S), torch.full((48,), m.none, device="cuda")
    cut = 0
    for t in range(25):
        o = obs.reshape(-1).clone()
        if t:
            S[done], size[done], last = 0.0, 0.0, torch.where(done, torch.full_like(last, m.none), last)
            cut += int(done.sum())
        with torch.no_grad():
            x, q, k, v = (y.double() for y in m._rows(o, last))          # tokens and projections: the call's own
        a = torch.exp(m.log_decay.double())[None, :, None, None]
        S, size = S * a + k.unsqueeze(-1) * v.unsqueeze(-2), size * a + k.abs().unsqueeze(-1) * v.abs().unsqueeze(-2)
        read = (0.25 * (q.unsqueeze(-2) @ S)).reshape(48, 32)
        # off by, step by step: the memory's sums in float32 and one rounding each of what is read, its product, the sum, the normed row, the logits
        off = HALF * read.abs() + 64 * 25 * 2.0 ** -24 * (0.25 * (q.abs().unsqueeze(-2) @ size)).reshape(48, 32)
        p = read @ out
        off = off @ out.abs()
        off = off + HALF * (p.abs() + off)
        h = x + p
        off = off + HALF * (h.abs() + off)
        r = torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6)
        assert ((off.norm(dim=1) / h.norm(dim=1)) < 0.05).all()          # (the norm's own change, to first order, with room for the second)
        off = r * off + 1.1 * r * h.abs() * (off.norm(dim=1) / h.norm(dim=1)).unsqueeze(1)
        off = off + HALF * ((r * h).abs() + off)
        want = (r * h) @ head.t()
        off = off @ head.abs().t()
        off = off + HALF * (want.abs() + off) + 1e-6
        action, state, logits = predict_and_logits(m, o, state=state, mask=done)
        assert ((logits.double() - want).abs() <= off).all()
        assert state[0].dtype == torch.float32 and torch.equal(state[1] - m.bins, logits.argmax(1))
        last = state[1].clone()
        obs, _, done, _ = env.step(action)
        done = done.reshape(-1).bool().clone()
    assert cut > 0                                                       # episodes ended on the way


@pytest.mark.parametrize("env_id", ["fishing-v0", "fishing-v1", "fishing-v4"])
def test_simulate_drives_it_in_bfloat16(env_id):
    kw = {} if env_id == "fishing-v4" else {"sigma": 0.05}
    sizes = dict(dim=16, heads=2, head_dim=8, bins=32, levels=9, dtype=torch.bfloat16)
    env = gf.make(env_id, num_envs=8, seed=1, Tmax=15, **kw)
    m = policies.memory(env, **sizes)
    df = env.simulate(m, reps=1)
    assert len(df["time"]) > 0 and np.isfinite(np.asarray(df["state"])).all()
    assert len(rollout.simulate_mdp_vec(env, m, 16)["time"]) == 16 * (env.Tmax + 1)
    one = gf.make(env_id, Tmax=15, **kw)
    df = one.simulate(policies.memory(one, **sizes), reps=2)
    assert set(np.asarray(df["rep"]).astype(int)) == {0, 1}
    a, state = m.predict(torch.zeros((8, 1), device="cuda"), deterministic=False)
    assert a.shape == (8, 1) and state[0].dtype == torch.float32
