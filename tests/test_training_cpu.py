"""The fine-tuning operators without a GPU: what their entry points refuse, the generator's published vectors, and the
tests' own restatements against finite differences."""
import ctypes

import numpy as np
import pytest
import torch

import train_ref as R
from granite_conv_b200 import _lib, training

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(257)


def test_philox_known_answers():
    """The vectors published with the generator: all zeros, all ones."""
    assert [int(v) for v in R.philox([0, 0, 0, 0], (0, 0))] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    assert [int(v) for v in R.philox([f] * 4, (f, f))] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_row_entry_points_refuse_bad_calls():
    L = _lib.lib()

    def fwd(x=P, ld=64, w=P, y=P, M=4, D=64, dtype=0, ptype=2, lens=None, T=0):
        return L.gsn_layer_norm_fwd(x, ld, w, P, y, M, D, 1e-5, dtype, ptype, lens, T, None)

    assert fwd(M=-1) == 1 and fwd(D=0) == 1
    assert fwd(x=None) == 1 and "null x" in _lib.last_error()
    assert fwd(w=None) == 1 and fwd(y=None) == 1
    assert fwd(D=8193, ld=8193) == 2 and "8192" in _lib.last_error()
    assert fwd(ld=63) == 2 and "row stride" in _lib.last_error()
    assert fwd(dtype=3) == 2 and fwd(ptype=1) == 2 and fwd(x=ODD) == 2
    assert fwd(M=1 << 31) == 2
    assert fwd(lens=P, T=3) == 2 and "must divide" in _lib.last_error()
    assert fwd(M=0, x=None, w=None, y=None) == 0

    need = L.gsn_layer_norm_bwd_workspace_bytes(4, 64)
    assert need > 0 and L.gsn_layer_norm_bwd_workspace_bytes(0, 64) == 0

    def bwd(dy=P, x=P, ws=P, nbytes=need, dw=P):
        return L.gsn_layer_norm_bwd(dy, 64, x, 64, P, P, dw, P, 4, 64, 1e-5, 0, 2, None, 0, ws, nbytes, None)

    assert bwd(nbytes=need - 1) == 5 and "workspace" in _lib.last_error()
    assert bwd(ws=None) == 1 and bwd(dy=None) == 1 and bwd(dw=None) == 1 and bwd(x=ODD) == 2

    def drop(p=0.1, rng=P, scale=1.0, M=4, ld_r=64):
        return L.gsn_dropout_add(P, 64, P, ld_r, P, M, 64, 0, rng, 0, p, scale, None, 0, None)

    assert drop(p=-0.1) == 1 and drop(p=1.1) == 1 and drop(p=float("nan")) == 1
    assert drop(rng=None) == 1 and drop(rng=ctypes.c_void_p(260)) == 1
    assert drop(scale=float("inf")) == 1 and drop(ld_r=8) == 2 and drop(M=0) == 0
    assert drop(scale=1e39) == 1 and drop(p=0.99998, scale=1e37) == 1 and "fp32" in _lib.last_error()

    def both(res=P, h=P, p=0.1):
        return L.gsn_dropout_add_layer_norm_fwd(P, 64, res, 64, P, P, P, h, 4, 64, 1e-5, 0, 2, P, 0, p, 1.0, None, 0,
                                                None)

    assert both(res=None) == 1 and both(h=None) == 1 and both(p=2.0) == 1

    def both_bwd(h=P, nbytes=need, dres=P, dh=None, ld_dh=0):
        return L.gsn_dropout_add_layer_norm_bwd(P, 64, dh, ld_dh, h, 64, P, P, dres, P, P, 4, 64, 1e-5, 0, 2, P, 0, 0.1,
                                                1.0, None, 0, P, nbytes, None)

    assert both_bwd(h=None) == 1 and both_bwd(dres=None) == 1 and both_bwd(nbytes=0) == 5
    assert both_bwd(dh=P, ld_dh=3) == 2


def test_ctc_entry_points_refuse_bad_calls():
    L = _lib.lib()

    def fwd(B=2, T=5, V=7, S=3, ld_t=7, blank=0, dtype=0, logits=P, targets=P, ws=None, nbytes=0):
        return L.gsn_ctc_loss_fwd(logits, 35, ld_t, targets, P, P, B, T, V, S, blank, 0, 1, dtype, P, P, 1 << 20, ws,
                                  nbytes, None)

    assert fwd(B=-1) == 1 and fwd(V=0) == 1 and fwd(S=-1) == 1
    assert fwd(blank=7) == 1 and fwd(blank=-1) == 1 and "blank" in _lib.last_error()
    assert fwd(S=2001) == 2 and fwd(T=16385) == 2 and fwd(ld_t=6) == 2 and fwd(dtype=7) == 2
    assert fwd(logits=None) == 1 and fwd(targets=None) == 1 and fwd(logits=ODD) == 2
    need = L.gsn_ctc_loss_workspace_bytes(2, 5, 3, 1)
    assert need > L.gsn_ctc_loss_workspace_bytes(2, 5, 3, 0) > 0 and L.gsn_ctc_loss_workspace_bytes(0, 5, 3, 1) == 0
    assert fwd(ws=P, nbytes=need - 1) == 5
    assert fwd(B=0, logits=None, targets=None) == 0

    state = L.gsn_ctc_loss_state_bytes(2, 5, 3)

    def bwd(dloss=P, out=P, T=5, st=P, nbytes=state):
        return L.gsn_ctc_loss_bwd(dloss, P, 35, 7, P, P, P, 2, T, 7, 3, 0, 0, 0, st, nbytes, out, None)

    assert bwd(dloss=None) == 1 and bwd(out=None) == 1 and bwd(out=ODD) == 2 and bwd(dloss=None, T=0) == 0
    assert bwd(nbytes=state - 1) == 5 and bwd(st=None) == 1 and bwd(st=ctypes.c_void_p(264)) == 1


def test_functions_refuse_cpu_tensors():
    x = torch.zeros(2, 3, 16)
    w = torch.zeros(16)
    rng = torch.zeros(2, dtype=torch.int64)
    i = torch.ones(2, dtype=torch.int32)
    t = torch.zeros(2, 4, dtype=torch.int32)
    for call in (lambda: training.layer_norm(x, w, w), lambda: training.layer_norm_backward(x, x, w),
                 lambda: training.dropout_add(x, rng, 0.1), lambda: training.dropout_add_backward(x, rng, 0.1),
                 lambda: training.dropout_add_layer_norm(x, x, w, w, rng, 0.1),
                 lambda: training.dropout_add_layer_norm_backward(x, None, x, w, rng, 0.1),
                 lambda: training.ctc_loss(x, t, i, i)):
        with pytest.raises(RuntimeError, match="CUDA device"):
            call()


# ---- the restatements the GPU tests compare with, against differences ------------------------------------------------
def _difference(f, x, at, h=1e-5):
    a, b = x.clone(), x.clone()
    a[at] += h
    b[at] -= h
    return (float(f(a)) - float(f(b))) / (2 * h)


def test_layer_norm_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 4, 6, generator=g, dtype=torch.float64)
    w = torch.randn(6, generator=g, dtype=torch.float64)
    b = torch.randn(6, generator=g, dtype=torch.float64)
    dy = torch.randn(2, 4, 6, generator=g, dtype=torch.float64)
    lens = [4, 2]
    dx, dw, db, _, _ = R.layer_norm_backward(dy, x, w, 1e-5, lens)
    for at in [(0, 1, 2), (1, 1, 5), (1, 3, 0)]:
        d = _difference(lambda v: (R.layer_norm(v, w, b, 1e-5, lens)[0] * dy).sum(), x, at)
        assert abs(d - float(dx[at])) < 1e-7          # central differences at h = 1e-5: h^2 and 1e-16 / h
    for k in range(6):
        assert abs(_difference(lambda v: (R.layer_norm(x, v, b, 1e-5, lens)[0] * dy).sum(), w, (k,)) - dw[k]) < 1e-7
        assert abs(_difference(lambda v: (R.layer_norm(x, w, v, 1e-5, lens)[0] * dy).sum(), b, (k,)) - db[k]) < 1e-7


def test_ctc_against_all_paths_and_differences():
    """The recursion against the sum over every frame labelling that collapses to the target, and its gradient against
    differences."""
    import itertools
    import math
    g = torch.Generator().manual_seed(5)
    V, n = 3, 4
    x = torch.randn(n, V, generator=g, dtype=torch.float64)
    for target in ([], [1], [1, 1], [1, 2], [2, 1, 2]):
        logp = torch.log_softmax(x, -1)
        total = 0.0
        for path in itertools.product(range(V), repeat=n):
            if [k for k, _ in itertools.groupby(path) if k != 0] == target:
                total += math.exp(sum(float(logp[t, v]) for t, v in enumerate(path)))
        loss, grad = R.ctc_one(x, target, 0)
        assert abs(loss + math.log(total)) < 1e-12
        for at in [(0, 0), (1, 2), (3, 1)]:
            assert abs(_difference(lambda v: R.ctc_one(v, target, 0)[0], x, at) - grad[at]) < 1e-8
    assert R.ctc_one(x[:2], [1, 1], 0) == (math.inf, None)
    assert R.ctc_one(x[:0], [], 0)[0] == 0.0


def test_keep_mask_probability():
    """The share of kept elements lies within five standard deviations of 1 - p."""
    for p in (0.1, 0.5, 0.9):
        keep = R.keep_mask((64, 1001), 12345, 7, 3, p)
        n = keep.numel()
        assert abs(keep.double().mean().item() - (1 - p)) < 5 * np.sqrt(p * (1 - p) / n) + 2 ** -17
    assert R.keep_mask((3, 9), 1, 0, 0, 0.0).all() and not R.keep_mask((3, 9), 1, 0, 0, 1.0).any()


def test_ctc_workspace_holds_every_lane_reference():
    """A frame's stored states: two words for each of the S + 1 pairs, and one for each lane of the warps that hold them
    (the first 32 lanes of NP pairs, the others less the lanes that repeat the warp below)."""
    lib = _lib.lib()

    def warps(pairs, NP, H):
        halo = -(-H // NP)
        return 1 if pairs <= 32 * NP else 1 - (32 * NP - pairs) // ((32 - halo) * NP)

    for S in range(0, training.MAX_CTC_LABELS + 1):
        shapes = [(1, 16, 4), (2, 16, 4), (3, 16, 4), (4, 8, 8), (4, 4, 99)]
        nw = next(warps(S + 1, NP, H) for NP, H, most in shapes if warps(S + 1, NP, H) <= most)
        frames = 1000
        states = lib.gsn_ctc_loss_workspace_bytes(1, frames, S, 1) - lib.gsn_ctc_loss_workspace_bytes(1, frames, S, 0)
        assert states >= frames * 4 * (2 * (S + 1) + 32 * nw), S


# ---- who takes a call ------------------------------------------------------------------------------------------------
def test_calls_under_a_tracer_go_through_the_dispatcher():
    """A tracer or mode that watches ops has to see the op, not the empty output that the kernel would fill."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, seen = torch.randn(3), []

    def f(a):
        seen.append(training._dispatched(a))
        return a * 1

    f(x)
    assert seen.pop() is False
    with Mode():
        f(x)
    make_fx(f)(x)
    make_fx(f, pre_dispatch=True)(x)
    make_fx(f, tracing_mode="fake")(x)
    torch.jit.trace(f, x, check_trace=False)
    assert len(seen) == 5 and all(seen)
    f(x)
    assert seen.pop() is False


def test_functions_refuse_tangents():
    """A forward-mode tangent is refused, by torch.func.jvp as by a dual tensor, not dropped."""
    from torch.autograd import forward_ad
    x, t = torch.randn(2, 3, 16), torch.ones(2, 3, 16)
    w = torch.ones(16)
    rng = torch.zeros(2, dtype=torch.int64)
    i = torch.ones(2, dtype=torch.int32)
    lab = torch.zeros(2, 4, dtype=torch.int32)
    calls = [lambda a: training.layer_norm(a, w, w), lambda a: training.layer_norm(x, a[0, 0], w),
             lambda a: training.layer_norm_backward(x, a, w), lambda a: training.dropout_add(x, rng, 0.1, residual=a),
             lambda a: training.dropout_add_backward(a, rng, 0.1),
             lambda a: training.dropout_add_layer_norm(x, a, w, w, rng, 0.1),
             lambda a: training.dropout_add_layer_norm_backward(x, a, x, w, rng, 0.1),
             lambda a: training.ctc_loss(a, lab, i, i)]
    for f in calls:
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(f, (x,), (t,))
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, t)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(dual)
            with pytest.raises(RuntimeError, match="CUDA device"):     # other tensors of a dual level are welcome
                f(x)


def test_batches_without_frames_take_lengths():
    """M = 0 with lengths, T = 0 among them, is a call with nothing to do and no error (the backward passes, which write
    dweight and dbias, are launches: on the GPU)."""
    L = _lib.lib()
    for T in (0, 3):
        assert L.gsn_layer_norm_fwd(P, 64, P, P, P, 0, 64, 1e-5, 0, 2, P, T, None) == 0
        assert L.gsn_dropout_add(P, 64, P, 64, P, 0, 64, 0, P, 0, 0.1, 1.0, P, T, None) == 0
        assert L.gsn_dropout_add_layer_norm_fwd(P, 64, P, 64, P, P, P, P, 0, 64, 1e-5, 0, 2, P, 0, 0.1, 1.0, P, T, None) == 0
    assert L.gsn_layer_norm_fwd(P, 64, P, P, P, 4, 64, 1e-5, 0, 2, P, 0, None) == 2


def test_sizes_past_32_bits_are_refused():
    """Widths, classes and utterances that an int does not hold must not come down to their low halves."""
    L = _lib.lib()
    wide = 2 ** 31 - 255
    assert L.gsn_dropout_add(P, wide, None, 0, P, 1, wide, 0, P, 0, 0.1, 1.0, None, 0, None) == 2
    assert "at most" in _lib.last_error()
    big = 2 ** 31 - 1023
    assert L.gsn_ctc_loss_fwd(P, big, big, P, P, P, 1, 1, big, 1, 0, 0, 0, 0, P, P, 1 << 20, P, 1 << 20, None) == 2
    one = torch.zeros(1)
    with pytest.raises(RuntimeError, match="elements expected"):
        training._check_rows("rows", one.expand(2 ** 32 + 5))
    training._check_rows("rows", one.expand(2 ** 31 - 256))


def test_ctc_selftest_refuses_bad_calls():
    L = _lib.lib()

    def call(side=0, half=0, B=2, nbytes=0, S=3):
        return L.gsn_selftest_ctc_withheld(P, 35, 7, P, P, P, B, 5, 7, S, 0, 0, P, P, 1 << 20, P, nbytes, side, half, None)

    assert call(side=2) == 1 and call(side=-1) == 1 and call(half=2) == 1 and call(B=-1) == 1 and call(S=80) == 2
    assert call() == 5 and "gsn_selftest_ctc_withheld: workspace" in _lib.last_error() and call(B=0) == 0
