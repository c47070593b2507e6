"""A policy that remembers its episode, for N envs in lockstep: `policies.memory`.

fishing-v4 draws (K, r) at every reset, fishing-v10 lets r drift, fishing-v11 draws the growth function: none of it is observed.
The agents the reference trains (PPO / DQN with "MlpPolicy": tests/test-PPO.py:10-21, tests/test-DQN.py:10-24) see one observation
at a time.  This one reads, per step, two tokens -- the observation's bin and the quota level it took the step before -- into a
memory per env that decays with a horizon per head and is cut where an episode starts, and answers with a distribution over quota
levels:

    x_t = embedding(bin(obs_t)) + embedding(level_{t-1})          sequence.embedding
    o_t = decay_attention(x_t Wq, x_t Wk, x_t Wv)                 sequence.decay_attention (whole records), _step (acting)
    h_t = rms(x_t + o_t Wo)          logits_t = h_t head^T        sequence.cross_entropy (scoring)

Acting is SB3's recurrent protocol, `predict(obs, state=state, mask=done) -> (action, state)`, so env.simulate(),
rollout.simulate_mdp_vec and env.policyfn() drive it like any model.  log_prob(record) scores the record of env.rollout(record=True)
for training: behind it stand the gradients of all three operators; optimisers are torch's.
"""
import numpy as np
import torch

from . import sequence
from .spaces import is_discrete


class memory:
    """`levels`: quota levels to choose from (fishing-v0: its n_actions, whatever is given); `bins` of the observation's range.
    `params`: name -> leaf tensor; pass an earlier policy's to go on with it.  dtype: float32 or bfloat16."""

    recurrent = True

    def __init__(self, env, dim=64, heads=4, head_dim=32, bins=256, levels=101, dtype=torch.float32, seed=0, params=None, **kwargs):
        self.env, self.device, self.dtype = env, env.device, dtype
        self.dim, self.heads, self.head_dim, self.bins = int(dim), int(heads), int(head_dim), int(bins)
        self.discrete = is_discrete(env.action_space)
        self.levels = int(env.action_space.n) if self.discrete else int(levels)
        if min(self.dim, self.heads, self.head_dim, self.bins) < 1 or self.levels < 2:
            raise ValueError("dim, heads, head_dim and bins must be at least 1, levels at least 2")
        if self.head_dim > sequence.MAX_HEAD_DIM:
            raise ValueError("head_dim must be at most %d" % sequence.MAX_HEAD_DIM)
        self.none = self.bins + self.levels             # the token of "no level yet"
        self._low = float(np.asarray(env.observation_space.low).reshape(-1)[0])
        self._span = float(np.asarray(env.observation_space.high).reshape(-1)[0]) - self._low
        shapes = dict(table=(self.none + 1, self.dim), qkv=(self.dim, 3 * self.heads * self.head_dim),
                      out=(self.heads * self.head_dim, self.dim), head=(self.levels, self.dim))
        if params is None:
            g = torch.Generator().manual_seed(int(seed))
            params = {k: (torch.randn(s, generator=g) * s[-1 if k in ("table", "head") else 0] ** -0.5).to(device=self.device, dtype=dtype).requires_grad_()
                      for k, s in shapes.items()}
        for k, s in shapes.items():
            if tuple(params[k].shape) != s or params[k].dtype != dtype or params[k].device != self.device:
                raise ValueError("params[%r] must be %s %s on %s" % (k, s, dtype, self.device))
        self.params = dict(params)
        # horizons of 4, 8, 16, ... steps: a head's memory falls to 1/e over its horizon
        self.log_decay = -torch.exp2(-torch.arange(2, 2 + self.heads, dtype=torch.float32, device=self.device))

    def parameters(self):
        return list(self.params.values())

    # ---- tokens and actions ----
    def _bin(self, obs):
        """The observation's bin; padding (-1) where it is not a number."""
        x = (obs.to(torch.float32) - self._low) / self._span
        return torch.where(torch.isfinite(x), (x.clamp(0.0, 1.0) * (self.bins - 1)).round(), torch.full_like(x, -1.0)).to(torch.int64)

    def _level(self, action):
        """The level nearest to an action; padding (-1) where it is not a number."""
        a = action.to(torch.float32)
        x = a if self.discrete else (a + 1.0) * (0.5 * (self.levels - 1))
        return torch.where(torch.isfinite(x), x.clamp(0, self.levels - 1).round(), torch.full_like(x, -1.0)).to(torch.int64)

    def _action(self, level):
        return level if self.discrete else level.to(torch.float32) * (2.0 / (self.levels - 1)) - 1.0

    # ---- the network ----
    def _rows(self, obs, last):
        """Tokens -> rows [..., dim] -> (rows, q, k, v)."""
        scale = self.dim ** 0.5
        table = self.params["table"]
        x = sequence.embedding(self._bin(obs), table, scale) + sequence.embedding(last, table, scale)
        qkv = (x @ self.params["qkv"]).reshape(x.shape[:-1] + (3, self.heads, self.head_dim))
        return (x,) + tuple(qkv.unbind(-3))

    def _hidden(self, x, o):
        h = x + o.reshape(x.shape[:-1] + (self.heads * self.head_dim,)) @ self.params["out"]
        wide = h.to(torch.float32)
        return (wide * torch.rsqrt(wide.square().mean(-1, keepdim=True) + 1e-6)).to(self.dtype)

    # ---- acting ----
    @torch.no_grad()
    def predict(self, obs, state=None, mask=None, deterministic=True, **kwargs):
        """One step of a batch: (actions, state).  `state` is what the step before returned (None: nothing remembered yet) and moves on in
        place; `mask`: the done flags of the step before.  A NumPy observation is answered in NumPy."""
        numpy = not isinstance(obs, torch.Tensor)
        o = torch.as_tensor(np.asarray(obs) if numpy else obs, device=self.device).reshape(-1)
        n = o.shape[0]
        starts = None
        if state is None:
            kept = torch.zeros((n, self.heads, self.head_dim, self.head_dim), dtype=torch.float32, device=self.device)
            last = torch.full((n,), self.none, dtype=torch.int64, device=self.device)
        else:
            kept, last = state
            if kept.shape[0] != n:
                raise ValueError("the state remembers %d envs, the observation holds %d" % (kept.shape[0], n))
            if mask is not None:
                starts = torch.as_tensor(mask, device=self.device).reshape(-1).to(torch.bool)
                last = torch.where(starts, torch.full_like(last, self.none), last)
        x, q, k, v = self._rows(o, last)
        h = self._hidden(x, sequence.decay_attention_step(q, k, v, self.log_decay, kept, starts=starts))
        logits = (h @ self.params["head"].t()).to(torch.float32)
        if not deterministic:                            # the largest of logits + Gumbel noise is a draw from the distribution
            logits = logits - torch.log(-torch.log(torch.rand_like(logits).clamp(1e-20, 1.0 - 1e-7)))
        level = logits.argmax(-1)
        action = self._action(level)
        state = (kept, self.bins + level)
        if numpy:
            action = action.cpu().numpy()
            return (int(action[0]) if self.discrete and n == 1 else action), state
        return action.reshape(-1, 1), state

    # ---- scoring ----
    def log_prob(self, record, frozen=False):
        """log probability [T, N] (float32) of the actions in env.rollout(T, record=True)'s [T, 4, N] table {obs_in, action, reward,
        done} under this policy, each level given the episode so far; differentiable in `parameters()`.  frozen: the record of
        an env without auto-reset -- steps behind an env's first done count 0 and take no gradient."""
        if record.dim() != 3 or record.shape[1] != 4:
            raise ValueError("record must be [T, 4, N], got %s" % (tuple(record.shape),))
        steps, _, n = record.shape
        level, done = self._level(record[:, 1]), record[:, 3] != 0
        starts = torch.zeros((steps, n), dtype=torch.bool, device=self.device)
        if steps:
            starts[0] = True
            starts[1:] = done[:-1]
        last = torch.full((steps, n), self.none, dtype=torch.int64, device=self.device)
        last[1:] = torch.where(starts[1:] | (level[:-1] < 0), last[1:], self.bins + level[:-1])
        x, q, k, v = self._rows(record[:, 0], last)
        o = sequence.decay_attention(q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1), self.log_decay, starts=starts.t())
        h = self._hidden(x, o.transpose(0, 1))
        if frozen:
            level = torch.where(done.cumsum(0) - done.to(torch.int64) > 0, torch.full_like(level, -1), level)
        return -sequence.cross_entropy(h.reshape(steps * n, self.dim), self.params["head"], level.reshape(-1)).reshape(steps, n)
