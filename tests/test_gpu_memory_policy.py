"""policies.memory: acting through the simulate helpers, scoring rollout records, gradients."""
import numpy as np
import pytest
import torch

import gym_fishing_amd as gf
from gym_fishing_amd import policies, rollout

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("env_id", ["fishing-v0", "fishing-v1", "fishing-v4", "fishing-v11"])
def test_record_scores_are_the_steps_own(env_id):
    """log_prob(record) == the log softmax of the logits that acting through the same record, step by step, would see."""
    env = gf.make(env_id, num_envs=64, seed=3, Tmax=20, **({} if env_id == "fishing-v11" else {"sigma": 0.1}))
    env.reset()
    record = env.rollout(50, policy="random", record=True).float()
    assert (record[:, 3] != 0).any()                                 # episodes end inside the record
    m = policies.memory(env, dim=32, heads=2, head_dim=16, bins=64, levels=21, seed=1)
    got = m.log_prob(record)
    assert got.shape == (50, 64) and got.dtype == torch.float32
    state, want, seen = None, [], {}
    real = torch.Tensor.argmax
    for t in range(50):
        def grab(self, *a, **k):
            seen["logits"] = self
            return real(self, *a, **k)
        torch.Tensor.argmax = grab
        try:
            _, state = m.predict(record[t, 0], state=state, mask=None if t == 0 else record[t - 1, 3])
        finally:
            torch.Tensor.argmax = real
        level = m._level(record[t, 1])
        want.append(torch.log_softmax(seen["logits"].double(), 1).gather(1, level.unsqueeze(1)).squeeze(1))
        state = (state[0], m.bins + level)                           # what the record's actor did, not what this one would
    # float32 throughout: 50 steps and three products of up to 64 terms between the token and the logit, logits of a few units
    assert (got.double() - torch.stack(want)).abs().max() <= 2.0 ** -24 * 64 * 50 * 8


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_reach_every_parameter_and_are_the_differences(dtype):
    env = gf.make("fishing-v1", sigma=0.1, num_envs=32, seed=0, Tmax=10)
    env.reset()
    record = env.rollout(25, policy="random", record=True)
    m = policies.memory(env, dim=24, heads=3, head_dim=8, bins=40, levels=11, dtype=dtype)
    loss = -m.log_prob(record).mean()
    grads = torch.autograd.grad(loss, m.parameters())
    assert all(torch.isfinite(g).all() and g.abs().sum() > 0 for g in grads)
    if dtype == torch.float32:
        for i, (name, g) in enumerate(zip(m.params, grads)):
            d = torch.randn(g.shape, generator=torch.Generator().manual_seed(i)).cuda()
            d = d / d.norm()
            ends = [-float(policies.memory(env, dim=24, heads=3, head_dim=8, bins=40, levels=11,
                                           params={**m.params, name: m.params[name].detach() + s * d}).log_prob(record).double().mean()) for s in (2e-3, -2e-3)]
            # a mean over 800 rows of float32 logits of a few units: 1e-6 over the step's 4e-3, and the third derivative's step squared
            assert abs((ends[0] - ends[1]) / 4e-3 - float((g.double() * d.double()).sum())) <= 1e-6 / 4e-3 + 50 * 4e-6, name


def test_frozen_records_count_each_episode_once():
    env = gf.make("fishing-v1", sigma=0.1, num_envs=16, seed=2, Tmax=12, auto_reset=False)
    env.reset()
    record = env.rollout(30, policy="random", record=True)
    m = policies.memory(env, dim=16, heads=1, head_dim=8, bins=16, levels=5)
    done = record[:, 3] != 0
    behind = done.cumsum(0) - done.long() > 0
    assert behind.any()
    got = m.log_prob(record, frozen=True)
    assert (got[behind] == 0).all() and (got[~behind] < 0).all()


@pytest.mark.parametrize("env_id", ["fishing-v0", "fishing-v1", "fishing-v4"])
def test_simulate_drives_it(env_id):
    kw = {} if env_id == "fishing-v4" else {"sigma": 0.05}
    env = gf.make(env_id, num_envs=8, seed=1, Tmax=15, **kw)
    m = policies.memory(env, dim=16, heads=2, head_dim=8, bins=32, levels=9)
    df = env.simulate(m, reps=1)
    assert len(df["time"]) > 0 and np.isfinite(np.asarray(df["state"])).all()
    df = rollout.simulate_mdp_vec(env, m, 16)
    assert len(df["time"]) == 16 * (env.Tmax + 1)
    one = gf.make(env_id, Tmax=15, **kw)                              # the scalar protocol, answered in NumPy
    df = one.simulate(policies.memory(one, dim=16, heads=2, head_dim=8, bins=32, levels=9), reps=2)
    assert set(np.asarray(df["rep"]).astype(int)) == {0, 1}
    assert len(one.policyfn(policies.memory(one, dim=16, heads=2, head_dim=8, bins=32, levels=9))["state"]) > 0


def test_sampled_actions_follow_the_distribution_and_bad_inputs_are_refused():
    env = gf.make("fishing-v0", num_envs=4096, seed=0, n_actions=4)
    m = policies.memory(env, dim=16, heads=1, head_dim=8, bins=8)
    obs = torch.zeros((4096, 1), device="cuda")
    torch.manual_seed(0)
    a, state = m.predict(obs, deterministic=False)
    assert a.shape == (4096, 1) and len(a.unique()) > 1
    with pytest.raises(ValueError):
        m.predict(obs[:5], state=state)
    with pytest.raises(ValueError):
        m.log_prob(torch.zeros((5, 3, 8), device="cuda"))
    with pytest.raises(ValueError):
        policies.memory(env, head_dim=129)
    with pytest.raises(ValueError):
        policies.memory(env, dim=16, heads=1, head_dim=8, bins=9, params=m.params)
    nan = obs.clone()
    nan[0] = float("nan")
    a, _ = m.predict(nan)                                             # an observation that is not a number is padding
    assert ((a >= 0) & (a < 4)).all()
