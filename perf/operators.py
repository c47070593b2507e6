"""What the sequence operators of gym_fishing_amd are measured on: an agent that remembers its episode reads tokens
(binned observations, the previous quota's level), keeps a decaying memory per env, and is scored on the quota levels.

    embedding                rows of a table for tokens, and the table's gradient
    decay_attention          linear attention with a decay for each head over whole episodes, and its gradients
    decay_attention_step     the same for the one step an env batch has just taken, on a kept memory
    cross_entropy            -log softmax of the level taken, over all levels, and the gradients

`own` False: the operators' definitions in elementary torch operations, in 32 bits.  `own` True: the package's calls.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one step of a 4096-env batch: the previous levels (101 tokens: 100 quota levels and "none yet"); latency counts
        dict(name="embed_step", op="embedding", train=False, tokens=4096, vocab=101, dim=64, dtype="bfloat16", index="int32"),
        # a recorded batch of whole episodes (101 steps, 4096 envs), observations on the growth sweep's grid of 10001 states
        dict(name="embed_train_grid", op="embedding", train=True, tokens=101 * 4096, vocab=10001, dim=128, dtype="bfloat16", index="int64"),
        # the largest: 1010 steps of 1024 envs, the 100 quota levels of the discrete env, each of them met thousands of times
        dict(name="embed_train_levels", op="embedding", train=True, tokens=1010 * 1024, vocab=100, dim=256, dtype="float32", index="int32"),
        # acting with a few envs: latency
        dict(name="step_few", op="step", batch=64, heads=4, dk=32, dv=32, dtype="bfloat16"),
        # acting with a large batch: a memory of 1 GB goes through once
        dict(name="step_many", op="step", batch=65536, heads=4, dk=32, dv=32, dtype="float32"),
        # one long history, read to go on from: few rows, a long axis
        dict(name="prompt_long", op="attention", train=False, batch=1, steps=16381, heads=8, dk=128, dv=128, dtype="bfloat16", starts=False, state=True, time_major=False),
        # training on recorded episodes, time-major as a rollout records them, cut where episodes end
        dict(name="attend_train_episodes", op="attention", train=True, batch=2048, steps=101, heads=4, dk=64, dv=64, dtype="bfloat16", starts=True, state=False, time_major=True),
        # the same in 32 bits with ragged sizes, ten episodes long, from a memory carried in
        dict(name="attend_train_odd", op="attention", train=True, batch=97, steps=1009, heads=3, dk=48, dv=80, dtype="float32", starts=True, state=True, time_major=True),
        # scoring a few steps against a very fine grid of levels
        dict(name="loss_few_rows", op="loss", train=False, rows=17, levels=65537, dim=512, dtype="bfloat16"),
        # training on recorded episodes of 1024 envs with the discrete env's 100 levels
        dict(name="loss_train_levels", op="loss", train=True, rows=101 * 1024, levels=100, dim=128, dtype="bfloat16"),
        # the same in 32 bits, ragged
        dict(name="loss_train_odd", op="loss", train=True, rows=5001, levels=1009, dim=200, dtype="float32"),
        # the largest: a fine grid of levels and a wide agent
        dict(name="loss_train_wide", op="loss", train=True, rows=8192, levels=32771, dim=1024, dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16"])
    size = 4 if dtype == "float32" else 2
    kind = rng.choice(["embedding", "step", "attention", "attention", "loss", "loss"])
    if kind == "embedding":
        dim = _log_int(rng, 8, 512)
        return dict(op=kind, train=rng.random() < 0.6, tokens=_log_int(rng, 1, min(1 << 20, 264_000_000 * 4 // (dim * size) // 4)), vocab=_log_int(rng, 16, 1 << 17),
                    dim=dim, dtype=dtype, index=rng.choice(["int32", "int64"]))
    heads = rng.randint(1, 8)
    if kind == "step":
        dk, dv = _log_int(rng, 8, 128), _log_int(rng, 8, 128)
        return dict(op=kind, batch=_log_int(rng, 1, min(65536, (1 << 28) // (heads * dk * dv))), heads=heads, dk=dk, dv=dv, dtype=dtype)
    if kind == "attention":
        dk, dv = _log_int(rng, 8, 128), _log_int(rng, 8, 128)
        steps = _log_int(rng, 1, 16384)
        most = min(2_100_000_000 // (heads * steps * steps), 53_000_000 // (heads * steps * max(dk, dv)))
        return dict(op=kind, train=rng.random() < 0.6, batch=_log_int(rng, 1, max(1, min(4096, most))), steps=steps, heads=heads, dk=dk, dv=dv, dtype=dtype,
                    starts=rng.random() < 0.7, state=rng.random() < 0.5, time_major=rng.random() < 0.5)
    dim, levels = _log_int(rng, 16, 1024), _log_int(rng, 2, 65536)
    most = min(268_000_000 // levels, (1 << 35 if dtype == "float32" else 1 << 38) // (levels * dim))
    return dict(op=kind, train=rng.random() < 0.6, rows=_log_int(rng, 1, max(1, min(1 << 17, most))), levels=levels, dim=dim, dtype=dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    s = dict(case)
    if case["op"] == "embedding":
        # stocks and quotas gather around a few values: the tokens' frequencies fall off from the middle of the table
        n, vocab = case["tokens"], case["vocab"]
        at = (0.5 + 0.15 * torch.randn(n, generator=g, device="cuda", dtype=torch.float64)).clamp(0, 1) * (vocab - 1)
        tokens = at.round().to(torch.int64)
        gone = torch.rand(n, generator=g, device="cuda") < 0.03     # steps behind an episode's end: padding
        s["token"] = torch.where(gone, torch.full_like(tokens, -1), tokens).to(torch.int32 if case["index"] == "int32" else torch.int64)
        s["table"] = normal(vocab, case["dim"], scale=case["dim"] ** -0.5)
        s["scale"] = math.sqrt(case["dim"])
        if case["train"]:
            s["grad"] = normal(n, case["dim"], scale=n ** -0.5)
        return s
    if case["op"] == "loss":
        rows, levels, dim = case["rows"], case["levels"], case["dim"]
        s["hidden"] = normal(rows, dim)
        s["head"] = normal(levels, dim, scale=1.5 * dim ** -0.5)
        target = torch.randint(0, levels, (rows,), generator=g, device="cuda")
        gone = torch.rand(rows, generator=g, device="cuda") < 0.06   # steps behind an episode's end
        s["target"] = torch.where(gone, torch.full_like(target, -1), target)
        if case["train"]:
            s["grad"] = normal(rows, scale=1.0 / rows, dtype=torch.float32)     # advantages, averaged
        return s
    batch, heads, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    steps = case.get("steps", 1)
    s["log_decay"] = torch.log1p(-torch.exp2(-torch.arange(3, 3 + heads, device="cuda", dtype=torch.float64))).float()

    def sequence(d, scale=1.0):
        if case["op"] == "step":
            return normal(batch, heads, d, scale=scale)
        if case["time_major"]:
            return normal(steps, batch, heads, d, scale=scale).transpose(0, 1)
        return normal(batch, steps, heads, d, scale=scale)

    s["q"], s["k"], s["v"] = sequence(dk), sequence(dk), sequence(dv)
    s["scale"] = dk ** -0.5
    if case["op"] == "step":
        s["state"] = normal(batch, heads, dk, dv, dtype=torch.float32)
        s["state_out"] = torch.empty_like(s["state"])
        s["starts"] = torch.rand(batch, generator=g, device="cuda") < 0.01
        return s
    # episodes of about 60 steps, some much shorter: the stock collapses
    s["starts"] = (torch.rand(steps, batch, generator=g, device="cuda") < 1 / 60).transpose(0, 1) if case["starts"] else None
    s["state"] = normal(batch, heads, dk, dv, dtype=torch.float32) if case["state"] else None
    if case["train"]:
        s["grad"] = sequence(dv)
        s["grad_state"] = normal(batch, heads, dk, dv, dtype=torch.float32) if case["state"] else None
    return s


def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _plain_embedding(s):
    table, vocab = s["table"], s["vocab"]
    token = s["token"].long()
    there = ((token >= 0) & (token < vocab)).unsqueeze(1)
    at = token.clamp(0, vocab - 1)
    out = {"out": torch.where(there, table[at].float() * s["scale"], torch.zeros((), device="cuda")).to(table.dtype)}
    if s["train"]:
        rows = torch.where(there, s["grad"].float() * s["scale"], torch.zeros((), device="cuda"))
        out["table"] = torch.zeros(table.shape, dtype=torch.float32, device="cuda").index_add_(0, at, rows).to(table.dtype)
    return out


def _plain_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    keep = torch.exp(s["log_decay"])[None, :] * (~s["starts"])[:, None]
    memory = torch.where((keep == 0)[:, :, None, None], torch.zeros((), device="cuda"), keep[:, :, None, None] * s["state"])
    memory = memory + k[:, :, :, None] * v[:, :, None, :]
    out = (q[:, :, None, :] @ memory).squeeze(2) * s["scale"]
    return {"out": out.to(s["q"].dtype), "state": memory}


def _plain_attention(s):
    q, k, v = (s[x].float().transpose(1, 2) for x in "qkv")            # [batch, heads, steps, d]
    batch, heads, steps, _ = q.shape
    dtype, scale, ld = s["q"].dtype, s["scale"], s["log_decay"]
    i = torch.arange(steps, device="cuda")
    apart = i[:, None] - i[None, :]
    weight = (torch.exp(apart.clamp(min=0) * ld[:, None, None]) * (apart >= 0))[None]       # [1, heads, steps, steps]
    if s["starts"] is not None:
        episode = s["starts"].long().cumsum(1)
        weight = weight * (episode[:, :, None] == episode[:, None, :])[:, None]
    else:
        episode = torch.zeros((batch, steps), dtype=torch.int64, device="cuda")
    score = (q @ k.transpose(2, 3)) * weight * scale
    out = score @ v
    into = torch.exp((i + 1) * ld[:, None]) * (episode == 0)[:, None]                        # [batch, heads, steps]
    rest = torch.exp((steps - 1 - i) * ld[:, None]) * (episode == episode[:, -1:])[:, None]
    through = torch.exp(steps * ld) * (episode[:, -1] == 0)[:, None]                         # [batch, heads]
    if s["state"] is not None:
        out = out + scale * into[..., None] * (q @ s["state"])
    got = {"out": out.transpose(1, 2).to(dtype)}
    if s["state"] is not None:
        got["state"] = (k * rest[..., None]).transpose(2, 3) @ v + through[..., None, None] * s["state"]
    if s["train"]:
        do = s["grad"].float().transpose(1, 2)
        dv = score.transpose(2, 3) @ do
        del score
        dscore = (do @ v.transpose(2, 3)) * weight * scale
        dq, dk = dscore @ k, dscore.transpose(2, 3) @ q
        if s["state"] is not None:
            ds = s["grad_state"]
            dq = dq + scale * into[..., None] * (do @ s["state"].transpose(2, 3))
            dk = dk + rest[..., None] * (v @ ds.transpose(2, 3))
            dv = dv + rest[..., None] * (k @ ds)
            got["dstate"] = scale * (q * into[..., None]).transpose(2, 3) @ do + through[..., None, None] * ds
        got.update(dq=dq.transpose(1, 2).to(dtype), dk=dk.transpose(1, 2).to(dtype), dv=dv.transpose(1, 2).to(dtype))
    return got


def _plain_loss(s):
    hidden, head, target = s["hidden"].float(), s["head"].float(), s["target"]
    levels, dtype = s["levels"], s["hidden"].dtype
    there = (target >= 0) & (target < levels)
    at = target.clamp(0, levels - 1).unsqueeze(1)
    logits = hidden @ head.t()
    top = logits.amax(1, keepdim=True)
    share = torch.exp(logits - top)
    total = share.sum(1, keepdim=True)
    zero = torch.zeros((), device="cuda")
    loss = torch.where(there, (torch.log(total) + top - logits.gather(1, at)).squeeze(1), zero)
    if not s["train"]:
        return {"loss": loss}
    del logits
    taken = torch.zeros_like(share).scatter_(1, at, 1.0)
    dlogits = torch.where(there, s["grad"], zero).unsqueeze(1) * (share / total - taken)
    return {"loss": loss, "dhidden": (dlogits @ head).to(dtype), "dhead": (dlogits.t() @ hidden).to(dtype)}


_plain = {"embedding": _plain_embedding, "step": _plain_step, "attention": _plain_attention, "loss": _plain_loss}


def _own_embedding(s):
    from gym_fishing_amd import sequence
    if not s["train"]:
        return {"out": sequence.embedding(s["token"], s["table"], scale=s["scale"])}
    table = s["table"].detach().requires_grad_()
    out = sequence.embedding(s["token"], table, scale=s["scale"])
    return {"out": out.detach(), "table": torch.autograd.grad(out, table, s["grad"])[0]}


def _own_step(s):
    from gym_fishing_amd import sequence
    out = sequence.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], starts=s["starts"], scale=s["scale"], state_out=s["state_out"])
    return {"out": out, "state": s["state_out"]}


def _own_attention(s):
    from gym_fishing_amd import sequence
    with_state = s["state"] is not None
    if not s["train"]:
        got = sequence.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], starts=s["starts"], state=s["state"], scale=s["scale"], return_state=with_state)
        return {"out": got[0], "state": got[1]} if with_state else {"out": got}
    q, k, v = (s[x].detach().requires_grad_() for x in "qkv")
    leaves = [q, k, v]
    if with_state:
        leaves.append(s["state"].detach().requires_grad_())
    got = sequence.decay_attention(q, k, v, s["log_decay"], starts=s["starts"], state=leaves[3] if with_state else None, scale=s["scale"], return_state=with_state)
    grads = torch.autograd.grad(got, leaves, [s["grad"], s["grad_state"]] if with_state else s["grad"])
    named = dict(zip(("dq", "dk", "dv", "dstate"), grads))
    return {"out": got[0].detach(), "state": got[1].detach(), **named} if with_state else {"out": got.detach(), **named}


def _own_loss(s):
    from gym_fishing_amd import sequence
    if not s["train"]:
        return {"loss": sequence.cross_entropy(s["hidden"], s["head"], s["target"])}
    hidden, head = s["hidden"].detach().requires_grad_(), s["head"].detach().requires_grad_()
    loss = sequence.cross_entropy(hidden, head, s["target"])
    dhidden, dhead = torch.autograd.grad(loss, (hidden, head), s["grad"])
    return {"loss": loss.detach(), "dhidden": dhidden, "dhead": dhead}


_own = {"embedding": _own_embedding, "step": _own_step, "attention": _own_attention, "loss": _own_loss}


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "embedding":
        n, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        met = min(n, vocab)
        rows = n * dim * size + n * (4 if case["index"] == "int32" else 8) + met * dim * size
        return {"bytes": rows + (n * dim * size + vocab * dim * size if case["train"] else 0), "flops": (2 if case["train"] else 1) * n * dim}
    if case["op"] == "loss":
        rows, levels, dim = case["rows"], case["levels"], case["dim"]
        both = (rows + levels) * dim * size
        if case["train"]:
            return {"bytes": 2 * both + 16 * rows, "flops": 6 * rows * levels * dim}
        return {"bytes": both + 12 * rows, "flops": 2 * rows * levels * dim}
    batch, heads, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    steps = case.get("steps", 1)
    lanes = batch * steps * heads
    kept = 4 * batch * heads * dk * dv
    forward = lanes * 2 * (dk + dv) * size + batch * steps * (1 if case.get("starts", True) else 0)
    if case["op"] == "step":
        return {"bytes": forward + 2 * kept, "flops": 4 * lanes * dk * dv}
    memory = 2 * kept if case["state"] else 0
    if not case["train"]:
        return {"bytes": forward + memory, "flops": 4 * lanes * dk * dv}
    # forward: q, k, v in, out; backward: the output's gradient in, three gradients out
    return {"bytes": forward + lanes * (2 * dk + 2 * dv) * size + 2 * memory, "flops": 12 * lanes * dk * dv}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "embedding":
        token = s["token"].long()
        there = (token >= 0) & (token < case["vocab"])
        table = s["table"].to(f64)
        padded = torch.cat([table, torch.zeros_like(table[:1])])
        at = torch.where(there, token, torch.full_like(token, case["vocab"]))
        got = {"out": padded.index_select(0, at) * s["scale"]}
        if case["train"]:
            total = torch.zeros_like(padded)
            total.index_put_((at,), s["grad"].to(f64) * s["scale"], accumulate=True)
            got["table"] = total[:-1].clone()
        return got
    if case["op"] == "loss":
        hidden, head = s["hidden"].to(f64).requires_grad_(), s["head"].to(f64).requires_grad_()
        there = ((s["target"] >= 0) & (s["target"] < case["levels"])).nonzero().squeeze(1)
        some = torch.log_softmax(hidden[there] @ head.t(), 1)
        nll = torch.zeros(case["rows"], dtype=f64, device="cuda").index_add(0, there, -some[torch.arange(len(there), device="cuda"), s["target"][there]])
        if not case["train"]:
            return {"loss": nll.detach()}
        dhidden, dhead = torch.autograd.grad(nll, (hidden, head), s["grad"].to(f64))
        return {"loss": nll.detach(), "dhidden": dhidden, "dhead": dhead}
    # the recurrence, one step after the other
    batch, heads, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    decay = torch.exp(s["log_decay"].to(f64))[None, :, None, None]
    one = case["op"] == "step"
    q, k, v = (s[x].to(f64).unsqueeze(1) if one else s[x].to(f64) for x in "qkv")
    steps = q.shape[1]
    starts = s["starts"]
    starts = torch.zeros((batch, steps), dtype=torch.bool, device="cuda") if starts is None else starts.reshape(batch, steps)
    kept = (~starts).to(f64)[:, :, None, None, None]
    memory = torch.zeros((batch, heads, dk, dv), dtype=f64, device="cuda") if s["state"] is None else s["state"].to(f64).clone()
    train = case.get("train", False)
    out = torch.empty((batch, steps, heads, dv), dtype=f64, device="cuda")
    if train:
        do = s["grad"].to(f64)
        dq, dk_, dv_ = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for t in range(steps):
        memory = memory * (decay * kept[:, t]) + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = s["scale"] * (q[:, t, :, None, :] @ memory).squeeze(2)
        if train:
            dq[:, t] = s["scale"] * (memory @ do[:, t, :, :, None]).squeeze(3)
    if one:
        return {"out": out.squeeze(1), "state": memory}
    got = {"out": out}
    if s["state"] is not None:
        got["state"] = memory
    if train:
        back = torch.zeros((batch, heads, dk, dv), dtype=f64, device="cuda") if s["state"] is None else s["grad_state"].to(f64).clone()
        for t in range(steps - 1, -1, -1):
            back = back + s["scale"] * q[:, t, :, :, None] * do[:, t, :, None, :]
            dk_[:, t] = (back @ v[:, t, :, :, None]).squeeze(3)
            dv_[:, t] = (k[:, t, :, None, :] @ back).squeeze(2)
            back = back * (decay * kept[:, t])
        got.update(dq=dq, dk=dk_, dv=dv_)
        if s["state"] is not None:
            got["dstate"] = back
    return got
