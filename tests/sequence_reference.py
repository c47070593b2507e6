"""The sequence operators' definitions in 64 bits on the CPU, step by step, and the error bounds their kernels are held to.

Bounds: a float32 sum of n products is off by at most n 2^-24 of the sum of their magnitudes; a rounding to bfloat16 by 2^-8 of
the value.  Each reference is therefore also run on the magnitudes of its operands."""
import torch

F64 = torch.float64
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def embedding(tokens, table, scale, grad=None):
    tokens, table = tokens.cpu().long(), table.detach().cpu().to(F64)
    there = ((tokens >= 0) & (tokens < len(table))).unsqueeze(-1)
    at = tokens.clamp(0, len(table) - 1)
    out = torch.where(there, table[at] * scale, torch.zeros((), dtype=F64))
    if grad is None:
        return out, None
    rows = torch.where(there, grad.cpu().to(F64) * scale, torch.zeros((), dtype=F64))
    return out, torch.zeros_like(table).index_add_(0, at.reshape(-1), rows.reshape(-1, table.shape[1]))


def attention(q, k, v, log_decay, starts=None, state=None, scale=1.0, grad=None, grad_state=None):
    """{out, state, dq, dk, dv, dstate}; a start lets nothing through, not even NaN."""
    q, k, v = (x.detach().cpu().to(F64) for x in (q, k, v))
    batch, steps, heads, dk_ = q.shape
    zero = torch.zeros((), dtype=F64)
    a = torch.exp(log_decay.cpu().to(F64))[None, :, None, None]
    cut = torch.zeros((batch, steps), dtype=torch.bool) if starts is None else starts.cpu()
    S = torch.zeros((batch, heads, dk_, v.shape[3]), dtype=F64) if state is None else state.detach().cpu().to(F64)
    out, dq, dk, dv = torch.empty_like(v), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    do = None if grad is None else grad.cpu().to(F64)
    for t in range(steps):
        S = torch.where(cut[:, t, None, None, None], zero, S * a) + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = scale * (q[:, t, :, None, :] @ S).squeeze(2)
        if do is not None:
            dq[:, t] = scale * (S @ do[:, t, :, :, None]).squeeze(3)
    got = {"out": out, "state": S}
    if do is not None:
        R = torch.zeros_like(S) if grad_state is None else grad_state.cpu().to(F64)
        for t in range(steps - 1, -1, -1):
            R = R + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
            dk[:, t] = (R @ v[:, t, :, :, None]).squeeze(3)
            dv[:, t] = (k[:, t, :, None, :] @ R).squeeze(2)
            R = torch.where(cut[:, t, None, None, None], zero, R * a)
        got.update(dq=dq, dk=dk, dv=dv, dstate=R)
    return got


def attention_bounds(q, k, v, log_decay, starts=None, state=None, scale=1.0, grad=None, grad_state=None):
    """How far each result may be off: float32 sums over steps and head dimensions and a decay kept as a product of up to `steps`
    float32 factors, and, in bfloat16, four roundings on a term's way -- a decayed operand, a score or a copy of the state, and its
    partner's, and the output's own."""
    mags = [x.detach().abs() for x in (q, k, v)]
    opt = [None if x is None else x.detach().abs() for x in (state, grad, grad_state)]
    got = attention(*mags, log_decay, starts, opt[0], abs(scale), opt[1], opt[2])
    n = 2 * q.shape[1] + q.shape[3] + v.shape[3] + 64
    rel = n * 2.0 ** -24 + (4 * 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0)
    return {x: rel * y for x, y in got.items()}


def loss(hidden, head, target, grad=None):
    """{loss, dhidden, dhead} and their bounds: a logit is a float32 sum of dim products, off by (dim + 8) 2^-24 of the magnitudes'
    sum; exp and log by a few units more; dz is rounded once to the operands' type, each output once."""
    h, w = hidden.detach().cpu().to(F64), head.detach().cpu().to(F64)
    y = target.cpu().long()
    rows, levels, dim = h.shape[0], w.shape[0], h.shape[1]
    there = (y >= 0) & (y < levels)
    h = torch.where(there[:, None], h, torch.zeros((), dtype=F64))
    z = h @ w.t()
    lse = torch.logsumexp(z, 1)
    at = y.clamp(0, levels - 1).unsqueeze(1)
    got = {"loss": torch.where(there, lse - z.gather(1, at).squeeze(1), torch.zeros((), dtype=F64))}
    u = 2.0 ** -24
    off = ((dim + 8) * u * (h.abs() @ w.abs().t())).amax(1) + 16 * u * (1 + lse.abs() + z.abs().amax(1))    # of a logit and of lse
    bound = {"loss": 3 * off + (levels + 16) * u}
    if grad is not None:
        g = torch.where(there, grad.cpu().to(F64), torch.zeros((), dtype=F64)).unsqueeze(1)
        share = torch.exp(z - lse[:, None])
        taken = torch.zeros_like(z).scatter_(1, at, 1.0)
        dz = g * (share - taken)
        got.update(dhidden=dz @ w, dhead=dz.t() @ h)
        step = STEP[hidden.dtype]
        # dz: the share's error (3 off relative) and its own rounding; then the products' float32 sums and the output's rounding
        ddz = g.abs() * (share * (4 * off + (levels + 16) * u)[:, None] + 4 * u) + 2 * step * dz.abs()
        bound["dhidden"] = ddz @ w.abs() + ((levels + 8) * u + 2 * step) * (dz.abs() @ w.abs()) + 1e-37
        bound["dhead"] = ddz.t() @ h.abs() + ((rows + 8) * u + 2 * step) * (dz.abs().t() @ h.abs()) + 1e-37
    return got, bound


def check(got, want, bound, what=""):
    got = got.detach().cpu().to(F64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound)
    assert (over <= 1e-30).all(), "%s: off by %.3g where %.3g is allowed" % (what, (got - want).abs().flatten()[over.argmax()], bound.flatten()[over.argmax()])


def check_once_rounded(got, want, what="", low=1 << 11):
    """A bfloat16 result whose only rounding worth speaking of is its last: its error in the 2-norm is at most 1.1 times that of `want`
    rounded once.  What comes before keeps 16 bits or more: terms off by at most 2^-16 of themselves, two thousandths of the last
    rounding's 2^-8 each, whose errors add up like the terms they belong to.  The last rounding's own error is spread over a step, so its
    norm over n values is known to about 0.45 n^-1/2 (2048 values: 1%).  One more rounding to bfloat16 on the way makes it 1.4."""
    got = got.detach().cpu()
    assert got.dtype == torch.bfloat16 and got.numel() >= low, (what, got.dtype, got.numel())
    once = (want.to(torch.bfloat16).to(F64) - want).norm()
    off = (got.to(F64) - want).norm()
    assert off <= 1.1 * once, "%s: off by %.3g, one rounding by %.3g" % (what, off, once)


def state_bound(size, steps):
    """How far a float32 state may be off, `size` the state of the operands' magnitudes: a product of bfloat16 values is exact in float32; the
    decays weigh it as a product of float32 factors, one a chunk or step, and are exp2 of a rounded exponent; v's three bfloat16 terms leave 2^-26."""
    return (2 * steps + 64) * 2.0 ** -24 * size


def check_state_norm(got, want, steps, what=""):
    """A float32 state that nothing decays, in the 2-norm: each of `steps` additions rounds its partial sum by up to 2^-24 of it, 2^-24 / sqrt 3 in
    the mean; partial sums of terms of random sign grow like the root of their count: 2^-24 sqrt(steps / 6) of the whole, and 4 units of 2^-24 for
    scaling the terms and what is left.  Terms of 16 bits (two of bfloat16) are off by 2^-19.3."""
    got = got.detach().cpu().to(F64)
    off, most = (got - want).norm(), (0.41 * steps ** 0.5 + 4) * 2.0 ** -24 * want.norm()
    assert off <= most, "%s: off by %.3g where %.3g is allowed" % (what, off, most)
