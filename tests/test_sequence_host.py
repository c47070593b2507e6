"""The sequence operators' host side without a GPU: refusals, the C entries' argument checks, the struct's layout, workspace sizes."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT
from gym_fishing_amd import _capi, build, sequence


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(build.LIB_PATH):
        build.build()
    return _capi.lib()


def test_no_cpu_path_and_types_are_checked_first():
    f, i = torch.zeros, torch.zeros(3, dtype=torch.int64)
    gone = sequence.FishingLibraryError
    for call, kind in ((lambda: sequence.embedding(i, f(5, 8)), gone), (lambda: sequence.embedding(i, f(5, 8).half()), TypeError), (lambda: sequence.embedding(i, f(5)), ValueError),
                       (lambda: sequence.embedding(i, None), TypeError), (lambda: sequence.cross_entropy(f(4, 8), f(5, 8), i), gone),
                       (lambda: sequence.cross_entropy(f(4, 8).double(), f(5, 8), i), TypeError), (lambda: sequence.cross_entropy(f(4), f(5, 8), i), ValueError),
                       (lambda: sequence.decay_attention(*[f(1, 2, 1, 4)] * 3, f(1)), gone), (lambda: sequence.decay_attention(*[f(2, 1, 4)] * 3, f(1)), ValueError),
                       (lambda: sequence.decay_attention(*[f(1, 2, 1, 4).half()] * 3, f(1)), TypeError),
                       (lambda: sequence.decay_attention_step(*[f(1, 1, 4)] * 3, f(1), f(1, 1, 4, 4)), gone),
                       (lambda: sequence.decay_attention_step(*[f(1, 1, 4)] * 3, f(1), None), TypeError)):
        with pytest.raises(kind):
            call()


def test_overlap_of_strided_tensors():
    pool = torch.zeros(100)
    a, b = pool[:60].view(6, 10)[:, :5], pool[60:]
    assert not sequence._overlap(a, b) and sequence._overlap(a, pool[54:56]) and not sequence._overlap(a, pool[55:])
    assert not sequence._overlap(pool[:0], pool)


def test_embedding_arguments(lib):
    fwd, bwd = lib.fishing_embedding_forward, lib.fishing_embedding_backward
    assert fwd(2, 4, 8, 5, 8, 64, 8, 64, 1.0, 64, None) == -7 and fwd(0, 2, 8, 5, 8, 64, 8, 64, 1.0, 64, None) == -7
    for n, vocab, dim in ((-1, 5, 8), (2 ** 31, 5, 8), (8, 0, 8), (8, 5, 0), (8, 5, 65537)):
        assert fwd(0, 4, n, vocab, dim, 64, 8, 64, 1.0, 64, None) == -4
        assert lib.fishing_embedding_workspace(0, n, vocab, dim) == -4
    assert fwd(0, 4, 8, 5, 8, 64, 7, 64, 1.0, 64, None) == -4
    assert fwd(0, 4, 8, 5, 8, None, 8, 64, 1.0, 64, None) == -1 and fwd(0, 4, 0, 5, 8, None, 8, None, 1.0, None, None) == 0
    need = lib.fishing_embedding_workspace(0, 8, 5, 8)
    assert need > 0
    assert bwd(0, 4, 8, 5, 8, 64, 8, 64, 1.0, 64, 256, need - 1, None) == -4
    assert bwd(0, 4, 8, 5, 8, 64, 8, 64, 1.0, 64, 260, need, None) == -3
    assert bwd(0, 4, 8, 5, 8, 64, 8, 64, 1.0, None, 256, need, None) == -1


def test_attention_arguments(lib):
    def args(**kw):
        a = _capi.FishingDecayAttention()
        a.heads, a.dk, a.dv, a.batch, a.steps = 2, 8, 8, 3, 4
        for k in ("q", "k", "v", "log_decay", "state", "out", "state_out", "dout", "dq", "dk_out", "dv_out"):
            setattr(a, k, 256)
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)
    step, fwd, bwd, work = lib.fishing_decay_attention_step, lib.fishing_decay_attention_forward, lib.fishing_decay_attention_backward, lib.fishing_decay_attention_workspace
    assert step(None, None) == -1 and fwd(None, 256, 1 << 20, None) == -1
    for kw, rc in ((dict(dtype=2), -7), (dict(dk=129), -4), (dict(dv=0), -4), (dict(heads=0), -4), (dict(batch=-1), -4), (dict(steps=-1), -4), (dict(batch=2 ** 31), -4),
                   (dict(q=None), -1), (dict(log_decay=None), -1)):
        assert step(args(**kw), None) == rc and fwd(args(**kw), 256, 1 << 30, None) == rc and bwd(args(**kw), 256, 1 << 30, None) == rc, kw
        assert work(args(**kw), 0) == rc
    assert step(args(state=None), None) == -1 and fwd(args(out=None), 256, 1 << 30, None) == -1 and bwd(args(dq=None), 256, 1 << 30, None) == -1
    assert step(args(batch=0), None) == 0 and fwd(args(batch=0), None, 0, None) == 0
    need = work(args(), 0)
    assert need > 0 and fwd(args(), 256, need - 1, None) == -4 and fwd(args(), 264, need, None) == -3 and fwd(args(), None, need, None) == -1
    assert work(args(), 1) >= need
    # one long history is cut into segments, whose states live in the workspace; many rows are not
    assert work(args(batch=1, steps=1 << 16, dk=64, dv=64), 0) > 64 * 64 * 4 * 2 * 8
    assert work(args(batch=1 << 14, steps=1 << 10, dk=64, dv=64), 0) < 1 << 20


def test_cross_entropy_arguments(lib):
    fwd, bwd, work = lib.fishing_cross_entropy_forward, lib.fishing_cross_entropy_backward, lib.fishing_cross_entropy_workspace
    for d, r, v, m, rc in ((2, 4, 5, 8, -7), (0, -1, 5, 8, -4), (0, 4, 0, 8, -4), (0, 4, 5, 0, -4), (0, 4, 2 ** 27, 8, -4), (0, 2 ** 31, 5, 8, -4), (0, 4, 5, 65537, -4)):
        assert work(d, r, v, m, 0) == rc and work(d, r, v, m, 1) == rc
        assert fwd(d, 8, r, v, m, 64, m, 64, m, 64, 64, 64, 256, 1 << 40, None) == rc
        assert bwd(d, 8, r, v, m, 64, m, 64, m, 64, 64, 64, 64, 64, 256, 1 << 40, None) == rc
    need = work(0, 4, 5, 8, 0)
    assert fwd(0, 2, 4, 5, 8, 64, 8, 64, 8, 64, 64, 64, 256, need, None) == -7
    assert fwd(0, 8, 4, 5, 8, 64, 7, 64, 8, 64, 64, 64, 256, need, None) == -4
    assert fwd(0, 8, 4, 5, 8, None, 8, 64, 8, 64, 64, 64, 256, need, None) == -1
    assert fwd(0, 8, 4, 5, 8, 64, 8, 64, 8, 64, 64, 64, 256, need - 1, None) == -4
    assert fwd(0, 8, 0, 5, 8, None, 8, None, 8, None, None, None, None, 0, None) == 0
    # every size has a plan, and the backward pass of a large one keeps a piece of the levels, not all of them
    for rows in (0, 1, 17, 5001, 1 << 17):
        for levels in (1, 2, 100, 1009, 65537):
            for dim in (1, 33, 200, 1024):
                for d in (0, 1):
                    assert work(d, rows, levels, dim, 0) > 0 and work(d, rows, levels, dim, 1) > 0
    assert work(1, 8192, 1 << 20, 64, 1) < 8192 * (1 << 20) // 8


def test_the_struct_is_the_headers(tmp_path):
    names = [n for n, _ in _capi.FishingDecayAttention._fields_]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fishing_hip.h"\nint main(void){printf("%%zu", sizeof(FishingDecayAttention));%s return 0;}\n'
                   % "".join('printf(" %%zu", offsetof(FishingDecayAttention, %s));' % n for n in names))
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_capi.FishingDecayAttention)] + [getattr(_capi.FishingDecayAttention, n).offset for n in names]


def test_large_calls_have_a_plan_that_fits(lib):
    """Rows and batches are walked in blocks: workspaces stop growing with them, and what no launch could count is refused."""
    work = lib.fishing_cross_entropy_workspace
    for d, size in ((0, 4), (1, 2)):
        for levels, dim in ((5, 8), (100, 128), (20000, 8), (32771, 1024), (3, 65536)):
            assert work(d, 1 << 23, levels, dim, 1) == work(d, 1 << 30, levels, dim, 1) < 40 << 30
            assert work(d, 1 << 23, levels, dim, 0) == work(d, 1 << 30, levels, dim, 0) < 12 << 30
    assert work(0, 4, 1 << 26, 1024, 0) == -4 and work(1, 4, 1 << 26, 1024, 1) == -4
    a = _capi.FishingDecayAttention()
    a.heads, a.dk, a.dv, a.steps, a.batch, a.log_decay = 2, 4, 4, 2, 1 << 21, 64
    a.q = a.k = a.v = 64
    need = lib.fishing_decay_attention_workspace(a, 1)
    a.batch = 1 << 29
    assert lib.fishing_decay_attention_workspace(a, 1) == need < 1 << 28
    a.heads, a.batch = 65537, 1
    assert lib.fishing_decay_attention_workspace(a, 0) == -4 and lib.fishing_decay_attention_step(a, None) == -4


def test_forward_mode_tangents_are_refused():
    """Before anything else is looked at: a kernel would see the value alone, and the derivative would come out as zero."""
    from torch.autograd import forward_ad
    f, i = torch.ones, torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level():
        def dual(*shape):
            return forward_ad.make_dual(f(*shape), f(*shape))
        seq, one = [f(1, 2, 1, 4)] * 3, [f(1, 1, 4)] * 3
        calls = [lambda: sequence.embedding(i, dual(5, 8)), lambda: sequence.cross_entropy(dual(3, 8), f(5, 8), i)]
        calls += [lambda a=a: sequence.decay_attention(*a, f(1)) for a in ([dual(1, 2, 1, 4)] + seq[1:],)]
        calls += [lambda a=a: sequence.decay_attention_step(*a, f(1), f(1, 1, 4, 4)) for a in ([dual(1, 1, 4)] + one[1:],)]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    sequence._no_tangent(f(3), "x")                       # outside a level, and without a tangent inside one
    with forward_ad.dual_level():
        sequence._no_tangent(f(3), "x")
