"""The sequence operators where their forms have to agree with each other, and what they refuse or leave alone."""
import os
import sys

import pytest
import torch
from torch.autograd import forward_ad

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import sequence_reference as ref  # noqa: E402
from test_gpu_sequence import make, rand  # noqa: E402
from gym_fishing_amd import _capi, sequence  # noqa: E402

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


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dk,dv", [(17, 33), (33, 65), (49, 5), (65, 127), (81, 50), (127, 97)])
def test_segments_of_rows_that_are_not_whole_accesses(dk, dv, dtype):
    """Long histories of few rows whose loads cannot be wide: their states are computed in segments too, and dv's walk starts from dk's."""
    steps = 600 if dtype == torch.float32 else 1100
    q, k, v, ld, cut, s0, g, gs = make(1, steps, 2, dk, dv, dtype, dk % 4 == 1, 0.004, True, seed=dk * dv)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, s0)]
    got = sequence.decay_attention(*leaves[:3], ld / 16, starts=cut, state=leaves[3], scale=0.3, return_state=True)
    grads = torch.autograd.grad(got, leaves, [g, gs])
    args = (q, k, v, ld / 16, cut, s0, 0.3, g, gs)
    want, bound = ref.attention(*args), ref.attention_bounds(*args)
    size = ref.attention(*[x.abs() for x in args[:3]], *args[3:5], s0.abs(), 0.3, g.abs(), gs.abs())
    for name, x in zip(("out", "state", "dq", "dk", "dv", "dstate"), list(got) + list(grads)):
        ref.check(x, want[name], bound[name], name)
        if x.dtype == torch.bfloat16:
            ref.check_once_rounded(x, want[name], name)
        elif name.endswith("state"):
            ref.check(x, want[name], ref.state_bound(size[name], steps), name)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dk,dv", [(32, 48), (33, 47), (64, 128)])
def test_nothing_passes_a_start_across_segments(dk, dv, dtype):
    """NaN and infinities in a long history stay in their episode, whichever segment it lies in and however many it spans, in both
    directions of time; and a head whose decay is zero keeps them to their step."""
    steps = 700 if dtype == torch.float32 else 1300
    q, k, v, ld, _, s0, g, gs = make(1, steps, 3, dk, dv, dtype, False, 0.0, True, seed=dk)
    ld = torch.tensor([-0.02, -0.3, float("-inf")], device="cuda")
    cut = torch.zeros((1, steps), dtype=torch.bool, device="cuda")
    cut[:, [20, 300, steps - 250, steps - 90]] = True
    clean = [x.clone() for x in (q, k, v, g)]
    # the first episode (the state carried in), one that spans segments, and the last (the gradient of the state handed out)
    s0[0], gs[0] = float("nan"), float("inf")
    q[0, 200], k[0, 150], v[0, 170], g[0, 280] = float("nan"), float("inf"), float("-inf"), float("nan")
    k[0, steps - 50] = float("nan")
    leaves = [x.detach().requires_grad_() for x in (q, k, v, s0)]
    got = sequence.decay_attention(*leaves[:3], ld, starts=cut, state=leaves[3], return_state=True)
    grads = torch.autograd.grad(got, leaves, [g, gs])
    args = (*clean[:3], torch.nan_to_num(ld, neginf=-200.0), cut, torch.zeros_like(s0), dk ** -0.5, clean[3], torch.zeros_like(gs))
    want, bound = ref.attention(*args), ref.attention_bounds(*args)
    got = dict(zip(("out", "state", "dq", "dk", "dv", "dstate"), list(got) + list(grads)))
    for name in ("out", "dq", "dk", "dv"):
        for at in (slice(300, steps - 250), slice(steps - 250, steps - 90)):
            ref.check(got[name][:, at], want[name][:, at], bound[name][:, at], name)
        dirty = torch.zeros(steps, dtype=torch.bool)         # of the head that forgets: these steps and no other
        dirty[[200, 150, 170, 280, steps - 50]] = True
        if name in ("dk", "dv"):
            dirty[-1] = True
        ref.check(got[name][:, ~dirty, 2], want[name][:, ~dirty, 2], bound[name][:, ~dirty, 2], name + " without memory")
    # forwards what comes later does not reach back, backwards what came before does not reach on
    ref.check(got["out"][:, 20:150, :2], want["out"][:, 20:150, :2], bound["out"][:, 20:150, :2], "out")
    ref.check(got["out"][:, steps - 90:steps - 50], want["out"][:, steps - 90:steps - 50], bound["out"][:, steps - 90:steps - 50], "out")
    ref.check(got["dk"][:, 281:300, :2], want["dk"][:, 281:300, :2], bound["dk"][:, 281:300, :2], "dk")
    assert not torch.isfinite(got["out"][0, :20, :2]).any() and not torch.isfinite(got["out"][0, 170:300, :2]).any()
    assert torch.isnan(got["state"][0]).any() and torch.isfinite(got["state"][0, 2]).all()
    ref.check(got["dstate"][:, 2], want["dstate"][:, 2], bound["dstate"][:, 2], "dstate")


@pytest.mark.parametrize("dtype", BOTH)
def test_the_entry_takes_starts_that_run_backwards(dtype):
    """A negative step stride of `starts`, which the C entry allows: read from the last byte down, never beyond them."""
    q, k, v, ld, cut, s0, _, _ = make(3, 77, 2, 32, 32, dtype, False, 0.1, True, seed=4)
    want = sequence.decay_attention(q, k, v, ld, starts=cut, state=s0)
    back = cut.flip(1).contiguous()
    out = torch.empty_like(v)
    a = sequence._attention_args(q, k, v, ld, back, s0, 32 ** -0.5)
    a.starts += back.shape[1] - 1
    a.starts_stride[1] = -1
    a.out = out.data_ptr()
    a.out_stride[:] = out.stride()[:3]
    lib = _capi.lib()
    work = torch.empty(lib.fishing_decay_attention_workspace(a, 0), dtype=torch.uint8, device="cuda")
    assert lib.fishing_decay_attention_forward(a, work.data_ptr(), work.numel(), torch.cuda.current_stream().cuda_stream) == 0
    bound = ref.attention_bounds(q, k, v, ld, cut, s0, 32 ** -0.5)["out"]
    ref.check(out, want.cpu().double(), 2 * bound, "out")        # (another width of access: the same sums in another order)


def test_the_step_writes_nowhere_it_reads():
    """The state that moves on and `out` may lie neither in q, k, v nor in the decays or the starts: another workgroup may not have read them yet."""
    batch, heads, d = 4, 2, 8
    pool = torch.zeros(4096, device="cuda")
    state = pool[512:512 + batch * heads * d * d].view(batch, heads, d, d)
    end = 512 + state.numel()
    q, k, v = (rand(batch, heads, d, seed=i) for i in range(3))
    ld, starts, other = torch.tensor([-0.1, -0.2], device="cuda"), torch.zeros(batch, dtype=torch.bool, device="cuda"), torch.zeros_like(state)
    inside, bits = pool[600:600 + batch * heads * d].view(batch, heads, d), pool.view(torch.bool)
    fine = dict(q=q, k=k, v=v, log_decay=ld, state=state, starts=starts)
    for bad in (dict(q=inside), dict(k=inside), dict(v=inside), dict(log_decay=pool[end - 1:end + 1]), dict(starts=bits[4 * end - 1:4 * end + 3])):
        for kw in (dict(), dict(state=other, state_out=state)):
            with pytest.raises(ValueError, match="overlaps"):
                sequence.decay_attention_step(**{**fine, **bad, **kw})
        if not set(bad) & {"q", "k", "v"}:                # `out` in the same place
            with pytest.raises(ValueError, match="overlaps"):
                sequence.decay_attention_step(**{**fine, **bad, "state": other, "out": pool[end - batch * heads * d:end].view(batch, heads, d)})
    beside = pool[end:end + batch * heads * d].view(batch, heads, d)         # next to it is not in it
    sequence.decay_attention_step(**{**fine, "q": beside, "out": pool[512 - batch * heads * d:512].view(batch, heads, d)})
    wide = pool[:512].view(batch, 128)[:, 100:116].view(batch, heads, d)       # rows that end before it, with gaps
    sequence.decay_attention_step(**{**fine, "q": wide})


def test_the_step_does_not_write_into_what_requires_a_gradient():
    q, k, v = (rand(2, 1, 8, seed=i) for i in range(3))
    ld, state = torch.tensor([-0.1], device="cuda"), rand(2, 1, 8, 8, seed=4)
    for bad in (dict(out=torch.zeros((2, 1, 8), device="cuda", requires_grad=True)), dict(state_out=torch.zeros_like(state).requires_grad_())):
        with pytest.raises(ValueError, match="no gradient"):
            sequence.decay_attention_step(q, k, v, ld, state, **bad)
        with torch.no_grad():
            sequence.decay_attention_step(q, k, v, ld, state, **bad)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,levels,dim", [(200, 100, 40), (64, 20001, 16), (9, 5, 300)])
def test_padding_takes_no_gradient_whatever_the_head_holds(rows, levels, dim, dtype):
    hidden, head = rand(rows, dim, seed=1, dtype=dtype).requires_grad_(), rand(levels, dim, seed=2, dtype=dtype, scale=dim ** -0.5)
    head[levels // 2, 0], head[levels - 1, dim - 1] = float("nan"), float("inf")
    head.requires_grad_()
    target = torch.arange(rows, device="cuda") % levels
    gone = torch.arange(0, rows, 4, device="cuda")
    target[gone] = torch.tensor([-1, levels], device="cuda")[torch.arange(len(gone), device="cuda") % 2]
    loss = sequence.cross_entropy(hidden, head, target)
    dhidden, dhead = torch.autograd.grad(loss.sum(), (hidden, head))
    assert (loss[gone] == 0).all() and (dhidden[gone] == 0).all()
    there = torch.ones(rows, dtype=torch.bool, device="cuda")
    there[gone] = False
    assert torch.isnan(loss[there]).all() and torch.isnan(dhidden[there]).all()          # and what is not padding does not hide it
