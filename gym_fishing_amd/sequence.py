"""Sequence operators for agents that remember their episode, next to the envs that make the episodes.

fishing-v4 draws (K, r) at every reset, fishing-v10 lets r drift and fishing-v11 draws the growth function: what an env is
like shows only in the episode so far, and a policy that looks at one observation (the reference's, and its PPO / DQN agents:
tests/test-PPO.py:10-21) cannot use it.  These are the operators of one that can, for N envs in lockstep:

    embedding(tokens, table, scale=1.0)                    binned observations and past quota levels -> rows; the table's gradient
    decay_attention(q, k, v, log_decay, ...)               linear attention with a decay per head over recorded episodes, cut where
                                                           episodes start; gradients of q, k, v and the memory carried in
    decay_attention_step(q, k, v, log_decay, state, ...)   the same for the step an env batch has just taken, on a kept memory
    cross_entropy(hidden, head, target)                    -log softmax of the quota level taken, without keeping the logits

`policies.memory` is the policy built on them.  Everything runs in hand-written HIP kernels behind the C ABI
(include/fishing_hip.h) on torch's current stream of the tensors' device; there is no CPU fallback.  Values are float32 or
bfloat16 (float16's range is too narrow for the products of states and for dz); sums, softmax statistics and states are float32.
What comes back in bfloat16 is rounded once, from 16 bits or more, but for cross_entropy's gradients: dz, the logits' gradient that both
products take as a factor, is rounded to bfloat16 before them (as two terms it would double their work), so they are 1.4 times as far off as
one rounding, and dhidden of a handful of rows up to twice.  The same inputs give the same bits.  Derivatives are reverse-mode and of the first order: an operand or gradient that carries a
forward-mode tangent is refused.

Tensors made on another stream are the caller's to order, as for any torch operator.  Captured into a hipGraph, an operator
takes its workspace from the graph's memory pool, so graphs share none.  torch's own rule holds for a captured backward(): no
eager autograd graph over the same leaves may be alive while it is captured (use torch.autograd.grad, or drop the eager loss first).
"""
import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _capi
from ._capi import DTYPE_BF16, DTYPE_F32, FishingDecayAttention, FishingLibraryError

MAX_HEAD_DIM, MAX_HEADS = 128, 65536
_DTYPES = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16}
_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_DEVICE = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)      # (behind a tensor on the device: initialised)


def _stream(index):
    return _RAW_STREAM(index) if _RAW_STREAM is not None else torch.cuda.current_stream(index).cuda_stream


def _call(fn, device, *args):
    """The C entry on `device`'s current stream, with that device the current one."""
    index = device.index
    if _DEVICE() == index:
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc != 0:
        _capi.check(rc, fn.__name__)


def _no_tangent(x, name):
    """A kernel sees a dual tensor's value alone: its derivative would come out as zero."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise NotImplementedError("%s carries a forward-mode tangent: the sequence operators have no forward-mode derivative" % name)


def _tensor(x, name, dims=None, dtypes=None, device=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(x).__name__))
    _no_tangent(x, name)
    if dims is not None and x.dim() != dims:
        raise ValueError("%s must have %d dimensions, got shape %s" % (name, dims, tuple(x.shape)))
    if dtypes is not None and x.dtype not in dtypes:
        raise TypeError("%s must be %s, got %s" % (name, " or ".join(str(d) for d in dtypes), x.dtype))
    if not x.is_cuda:
        raise FishingLibraryError("%s must live on a HIP ('cuda') device, got %s: there is no CPU backend" % (name, x.device))
    if device is not None and x.device != device:
        raise ValueError("%s is on %s, the other operands on %s" % (name, x.device, device))
    return x


def _unit(x):
    """x, or a copy where its last axis has gaps (an expanded gradient, a transposed view)."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 and x.is_contiguous() else x.contiguous()


def _rows(x):
    """x [n, d] with unit-stride, non-overlapping rows."""
    return x if (x.stride(1) == 1 or x.shape[1] == 1) and (x.stride(0) >= x.shape[1] or x.shape[0] <= 1) else x.contiguous()


def _row_stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _workspace(size, device):
    if size < 0:
        _capi.check(size, "workspace")
    return torch.empty(size, dtype=torch.uint8, device=device)


# ---- embedding ------------------------------------------------------------------------------------------------------

class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale):
        ctx.save_for_backward(tokens)
        ctx.shape, ctx.scale = table.shape, scale
        return _embed(tokens, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        tokens, = ctx.saved_tensors
        _no_tangent(grad, "the gradient")
        vocab, dim = ctx.shape
        lib, n = _capi.lib(), tokens.numel()
        grad = _rows(grad.reshape(n, dim))
        out = torch.empty((vocab, dim), dtype=grad.dtype, device=grad.device)
        work = _workspace(lib.fishing_embedding_workspace(_DTYPES[grad.dtype], n, vocab, dim), grad.device)
        _call(lib.fishing_embedding_backward, grad.device, _DTYPES[grad.dtype], tokens.element_size(), n, vocab, dim, grad.data_ptr(), _row_stride(grad),
              tokens.data_ptr(), ctx.scale, out.data_ptr(), work.data_ptr(), work.numel())
        return None, out, None


def _embed(tokens, table, scale):
    vocab, dim = table.shape
    out = torch.empty(tokens.shape + (dim,), dtype=table.dtype, device=table.device)
    table = _rows(table)
    _call(_capi.lib().fishing_embedding_forward, table.device, _DTYPES[table.dtype], tokens.element_size(), tokens.numel(), vocab, dim, table.data_ptr(),
          _row_stride(table), tokens.data_ptr(), scale, out.data_ptr())
    return out


def embedding(tokens, table, scale=1.0):
    """`scale * table[tokens]`: [*tokens.shape, dim], in the table's type.  tokens: int32 / int64 of any shape; one outside
    [0, vocab) is padding: a row of zeros that takes no gradient.  table: [vocab, dim], float32 / bfloat16.  The table's
    gradient is summed in float32 over each token's rows, in their order, from the tokens sorted."""
    _tensor(table, "table", 2, _DTYPES)
    _tensor(tokens, "tokens", None, (torch.int32, torch.int64), table.device)
    if table.shape[0] < 1 or table.shape[1] < 1 or table.shape[1] > 65536:
        raise ValueError("table must be [vocab >= 1, 1 <= dim <= 65536], got %s" % (tuple(table.shape),))
    if tokens.numel() > 0x7FFFFFFF:
        raise ValueError("at most 2^31 - 1 tokens a call, got %d" % tokens.numel())
    tokens, scale = tokens.contiguous(), float(scale)
    if torch.is_grad_enabled() and table.requires_grad:
        return _Embedding.apply(tokens, table, scale)
    return _embed(tokens, table, scale)


# ---- linear attention with a decay for each head ----------------------------------------------------------------------

def _like(x, d):
    """An empty [batch, steps, heads, d] in x's order of batch and steps (a rollout records time-major)."""
    b, t, h, _ = x.shape
    if x.stride(1) > x.stride(0):
        return torch.empty((t, b, h, d), dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((b, t, h, d), dtype=x.dtype, device=x.device)


def _strides(x):
    return (x.stride(0), x.stride(1), x.stride(2))


def _ptr(x):
    return None if x is None else x.data_ptr()


def _attention_args(q, k, v, log_decay, starts, state, scale):
    a = FishingDecayAttention()
    a.dtype, a.heads, a.dk, a.dv = _DTYPES[q.dtype], q.shape[2], q.shape[3], v.shape[3]
    a.batch, a.steps, a.scale = q.shape[0], q.shape[1], scale
    a.q, a.k, a.v, a.log_decay, a.state = q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), _ptr(state)
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = _strides(q), _strides(k), _strides(v)
    if starts is not None:
        a.starts = starts.data_ptr()
        a.starts_stride[:] = (starts.stride(0), starts.stride(1))
    return a


def _attend(q, k, v, log_decay, starts, state, scale, with_state):
    q, k, v = _unit(q), _unit(k), _unit(v)
    lib, dev = _capi.lib(), q.device
    out = _like(q, v.shape[3])
    last = torch.empty((q.shape[0], q.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32, device=dev) if with_state else None
    a = _attention_args(q, k, v, log_decay, starts, state, scale)
    a.out, a.state_out = out.data_ptr(), _ptr(last)
    a.out_stride[:] = _strides(out)
    work = _workspace(lib.fishing_decay_attention_workspace(a, 0), dev)
    _call(lib.fishing_decay_attention_forward, dev, ctypes.byref(a), work.data_ptr(), work.numel())
    return out, last


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, state, log_decay, starts, scale, with_state):
        q, k, v = _unit(q), _unit(k), _unit(v)
        out, last = _attend(q, k, v, log_decay, starts, state, scale, with_state)
        ctx.save_for_backward(q, k, v, state, log_decay, starts)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, last) if with_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast=None):
        q, k, v, state, log_decay, starts = ctx.saved_tensors
        if dout is None and dlast is None:
            return (None,) * 8
        for x in (dout, dlast):
            if x is not None:
                _no_tangent(x, "the gradient")
        lib, dev = _capi.lib(), q.device
        dout = _unit(dout) if dout is not None else torch.zeros(q.shape[:3] + v.shape[3:], dtype=q.dtype, device=dev)
        dlast = dlast.contiguous() if dlast is not None else None
        dq, dk, dv = _like(q, q.shape[3]), _like(q, q.shape[3]), _like(q, v.shape[3])
        dstate = torch.empty_like(state) if state is not None and ctx.needs_input_grad[3] else None
        a = _attention_args(q, k, v, log_decay, starts, state, ctx.scale)
        a.dout, a.dstate_out, a.dq, a.dk_out, a.dv_out, a.dstate = dout.data_ptr(), _ptr(dlast), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dstate)
        a.dout_stride[:], a.dq_stride[:], a.dk_stride[:], a.dv_stride[:] = _strides(dout), _strides(dq), _strides(dk), _strides(dv)
        work = _workspace(lib.fishing_decay_attention_workspace(a, 1), dev)
        _call(lib.fishing_decay_attention_backward, dev, ctypes.byref(a), work.data_ptr(), work.numel())
        return dq, dk, dv, dstate, None, None, None, None


def _check_heads(q, k, v, log_decay, state, dims):
    _tensor(q, "q", dims, _DTYPES)
    dev = q.device
    _tensor(k, "k", dims, (q.dtype,), dev)
    _tensor(v, "v", dims, (q.dtype,), dev)
    qs, vs = q.shape, v.shape
    if k.shape != qs:
        raise ValueError("k must have q's shape %s, got %s" % (tuple(qs), tuple(k.shape)))
    if vs[:-1] != qs[:-1]:
        raise ValueError("v must have q's leading shape %s, got %s" % (tuple(qs[:-1]), tuple(vs)))
    heads, dk, dv = qs[-2], qs[-1], vs[-1]
    if not (1 <= dk <= MAX_HEAD_DIM and 1 <= dv <= MAX_HEAD_DIM):
        raise ValueError("head dimensions must be in 1 .. %d, got q, k: %d and v: %d" % (MAX_HEAD_DIM, dk, dv))
    if not 1 <= heads <= MAX_HEADS:
        raise ValueError("1 .. %d heads are needed, got %d" % (MAX_HEADS, heads))
    _tensor(log_decay, "log_decay", 1, (torch.float32,), dev)
    if log_decay.numel() != heads:
        raise ValueError("log_decay must hold one value for each of %d heads, got %d" % (heads, log_decay.numel()))
    if torch.is_grad_enabled() and log_decay.requires_grad:
        raise ValueError("log_decay has no gradient here: a head's decay is a fixed horizon (detach it)")
    if qs[0] * heads > 0x7FFFFFFF:
        raise ValueError("at most 2^31 - 1 (batch, head) pairs a call")
    shape = (qs[0], heads, dk, dv)
    if state is not None:
        _tensor(state, "state", 4, (torch.float32,), dev)
        if state.shape != shape:
            raise ValueError("state must be [batch, heads, dk, dv] = %s, got %s" % (shape, tuple(state.shape)))
    return shape


def _check_starts(starts, shape, device):
    _tensor(starts, "starts", len(shape), (torch.bool,), device)
    if tuple(starts.shape) != tuple(shape):
        raise ValueError("starts must be %s, got %s" % (tuple(shape), tuple(starts.shape)))


def decay_attention(q, k, v, log_decay, starts=None, state=None, scale=None, return_state=False):
    """Linear attention with a decay for each head, over whole sequences: with S_t = a_t S_{t-1} + k_t v_t^T,
    out_t = scale * q_t S_t, where a_t = exp(log_decay[head]), or 0 where `starts[batch, t]`.

    q, k: [batch, steps, heads, dk], v: [batch, steps, heads, dv], float32 or bfloat16, dk and dv in 1 .. 128; any strides (a
    time-major record's `x.transpose(0, 1)` is read in place and answered in the same order; a last axis with gaps is copied).
    log_decay: float32 [heads], a head's horizon (no gradient; -inf, or where float32's exp is 0: nothing is kept, not even NaN).
    starts: bool [batch, steps], True where an episode begins -- the done flags of the step before (SB3's `episode_starts`):
    nothing passes from before it, not even NaN.
    state: float32 [batch, heads, dk, dv], the memory from earlier steps (None: zeros).  scale: dk ** -0.5 by default.
    Returns out [batch, steps, heads, dv], or (out, state behind the last step) with return_state.
    Differentiable in q, k, v and state."""
    shape = _check_heads(q, k, v, log_decay, state, 4)
    if starts is not None:
        _check_starts(starts, q.shape[:2], q.device)
    scale = shape[2] ** -0.5 if scale is None else float(scale)
    log_decay = log_decay.detach().contiguous()
    state = state.contiguous() if state is not None else None
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad)):
        return _DecayAttention.apply(q, k, v, state, log_decay, starts, scale, bool(return_state))
    out, last = _attend(q, k, v, log_decay, starts, state, scale, return_state)
    return (out, last) if return_state else out


def _span(x):
    """The addresses from x's first element to behind its last."""
    at = x.data_ptr()
    return at, at + (x.nbytes if x.is_contiguous() else x.element_size() + x.element_size() * sum((n - 1) * s for n, s in zip(x.shape, x.stride())))


def _overlap(x, y):
    """Whether the memory between x's first and last element meets y's."""
    if x.numel() == 0 or y.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(x), _span(y)
    return a0 < b1 and b0 < a1


def _check_written(x, name, operands):
    """What a call writes (contiguous) may not lie where it reads: its workgroups run in any order."""
    lo = x.data_ptr()
    hi = lo + x.nbytes
    for y in operands:
        if y is not None:
            at = y.data_ptr()
            if at < hi and (at >= lo or _span(y)[1] > lo) and lo < hi and y.numel():
                raise ValueError("%s overlaps an operand" % name)


def decay_attention_step(q, k, v, log_decay, state, starts=None, scale=None, out=None, state_out=None):
    """One step of decay_attention for a batch: q, k [batch, heads, dk], v [batch, heads, dv], starts bool [batch] (the done flags of
    the step before).  `state` (float32 [batch, heads, dk, dv], contiguous) moves on in place, or into `state_out` (which may be
    `state` itself; it may not overlap it otherwise); neither it nor `out` may overlap another operand.  Returns out [batch, heads, dv]
    (written into `out` if given).  Acting, not training: there is no gradient, and while gradients are recorded tensors that require one
    are refused, to read or to write."""
    if state is None:
        raise TypeError("state must be a torch.Tensor: the memory that moves on")
    shape = _check_heads(q, k, v, log_decay, state, 3)
    batch, heads, dk, dv = shape
    dev = q.device
    if torch.is_grad_enabled() and any(getattr(x, "requires_grad", False) for x in (q, k, v, state, out, state_out)):
        raise ValueError("the single step has no gradient: call it under torch.no_grad(), or train with decay_attention")
    if starts is not None:
        _check_starts(starts, (batch,), dev)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it moves on in place")
    operands = (q, k, v, log_decay, starts)
    if state_out is None:
        state_out = state
    else:
        _tensor(state_out, "state_out", 4, (torch.float32,), dev)
        if tuple(state_out.shape) != shape or not state_out.is_contiguous():
            raise ValueError("state_out must be contiguous %s, got %s" % (shape, tuple(state_out.shape)))
        if state_out.data_ptr() != state.data_ptr() and _overlap(state, state_out):
            raise ValueError("state_out overlaps state without being it")
    _check_written(state_out, "the state that moves on", operands)
    if out is None:
        out = torch.empty((batch, heads, dv), dtype=q.dtype, device=dev)
    else:
        _tensor(out, "out", 3, (q.dtype,), dev)
        if tuple(out.shape) != (batch, heads, dv) or not out.is_contiguous():
            raise ValueError("out must be contiguous %s, got %s, strides %s" % ((batch, heads, dv), tuple(out.shape), out.stride()))
        _check_written(out, "out", operands + (state, state_out))
    q, k, v = _unit(q), _unit(k), _unit(v)
    log_decay = log_decay.contiguous()
    a = FishingDecayAttention()
    a.dtype, a.heads, a.dk, a.dv, a.batch, a.steps = _DTYPES[q.dtype], heads, dk, dv, batch, 1
    a.scale = dk ** -0.5 if scale is None else float(scale)
    a.q, a.k, a.v, a.log_decay = q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr()
    a.state, a.state_out, a.out = state.data_ptr(), state_out.data_ptr(), out.data_ptr()
    for to, x in ((a.q_stride, q), (a.k_stride, k), (a.v_stride, v), (a.out_stride, out)):
        to[0], to[2], _ = x.stride()
    if starts is not None:
        a.starts = starts.data_ptr()
        a.starts_stride[0] = starts.stride(0)
    _call(_capi.lib().fishing_decay_attention_step, dev, ctypes.byref(a))
    # written behind torch's back: a recorded graph that saved them has to notice
    for x in (state_out, out):
        if not x.is_inference():
            torch.autograd.graph.increment_version(x)
    return out


# ---- softmax cross entropy over the levels ------------------------------------------------------------------------------

def _loss(hidden, head, target):
    rows, dim = hidden.shape
    lib, dev = _capi.lib(), hidden.device
    loss = torch.empty(rows, dtype=torch.float32, device=dev)
    lse = torch.empty(rows, dtype=torch.float32, device=dev)
    work = _workspace(lib.fishing_cross_entropy_workspace(_DTYPES[hidden.dtype], rows, head.shape[0], dim, 0), dev)
    _call(lib.fishing_cross_entropy_forward, dev, _DTYPES[hidden.dtype], target.element_size(), rows, head.shape[0], dim, hidden.data_ptr(), _row_stride(hidden),
          head.data_ptr(), _row_stride(head), target.data_ptr(), loss.data_ptr(), lse.data_ptr(), work.data_ptr(), work.numel())
    return loss, lse


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, head, target):
        hidden, head = _rows(hidden), _rows(head)
        loss, lse = _loss(hidden, head, target)
        ctx.save_for_backward(hidden, head, target, lse)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, head, target, lse = ctx.saved_tensors
        _no_tangent(grad, "the gradient")
        rows, dim = hidden.shape
        levels = head.shape[0]
        lib, dev = _capi.lib(), hidden.device
        grad = grad.to(torch.float32).contiguous()
        dhidden, dhead = torch.empty((rows, dim), dtype=hidden.dtype, device=dev), torch.empty((levels, dim), dtype=head.dtype, device=dev)
        work = _workspace(lib.fishing_cross_entropy_workspace(_DTYPES[hidden.dtype], rows, levels, dim, 1), dev)
        _call(lib.fishing_cross_entropy_backward, dev, _DTYPES[hidden.dtype], target.element_size(), rows, levels, dim, hidden.data_ptr(), _row_stride(hidden),
              head.data_ptr(), _row_stride(head), target.data_ptr(), lse.data_ptr(), grad.data_ptr(), dhidden.data_ptr(), dhead.data_ptr(), work.data_ptr(), work.numel())
        return dhidden, dhead, None


def cross_entropy(hidden, head, target):
    """loss[r] = logsumexp_v(hidden[r] . head[v]) - hidden[r] . head[target[r]], float32 [rows]: minus the log probability of the
    level taken.  hidden: [rows, dim], head: [levels, dim], float32 or bfloat16; target: int32 / int64 [rows], one outside
    [0, levels) is padding: loss 0, no gradient, whatever its row of `hidden` or the head hold.  The logits are computed in pieces of the
    levels and never kept.  Differentiable in hidden and head, with any gradient of the rows (weights, advantages); in bfloat16 with one
    rounding more than the result's own (of dz, see above)."""
    _tensor(hidden, "hidden", 2, _DTYPES)
    dev = hidden.device
    _tensor(head, "head", 2, (hidden.dtype,), dev)
    _tensor(target, "target", 1, (torch.int32, torch.int64), dev)
    if head.shape[1] != hidden.shape[1]:
        raise ValueError("head must have hidden's width %d, got %d" % (hidden.shape[1], head.shape[1]))
    if not (1 <= hidden.shape[1] <= 65536 and 1 <= head.shape[0] <= 0x7FFFFFF):
        raise ValueError("hidden [rows, 1 <= dim <= 65536] and head [1 <= levels < 2^27, dim] are needed, got %s and %s" % (tuple(hidden.shape), tuple(head.shape)))
    if target.shape[0] != hidden.shape[0]:
        raise ValueError("target must hold one level for each of %d rows, got %d" % (hidden.shape[0], target.shape[0]))
    target = target.contiguous()
    if torch.is_grad_enabled() and (hidden.requires_grad or head.requires_grad):
        return _CrossEntropy.apply(hidden, head, target)
    return _loss(_rows(hidden), _rows(head), target)[0]
