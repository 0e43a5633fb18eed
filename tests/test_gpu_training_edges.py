"""The fine-tuning operators at the edges of their ranges: where they once were wrong, and where a rule changes sides."""
import math

import numpy as np
import pytest
import torch

import train_ref as R
from granite_conv_b200 import training as tr
from test_gpu_training import (BF, DEV, E, EPS, F32, HF, check_ctc, close, ctc_case, grads_bound, lens_of, param_bounds,
                               rand, rng_of, rounded)

pytestmark = pytest.mark.gpu


# ---- CTC: states that the logits favour in another order than the transcript -------------------------------------------
def run_case(S, at, runs, tail=40):
    """A transcript whose labels at - 1, at and at + 1 are c, a and b of classes of their own, its places in the middle
    of the frames; `runs` of (class, frames, boost) are favoured there, everything else is noise."""
    names = {"blank": 0, "a": 1, "b": 2, "c": 3}
    V = 13
    g = np.random.default_rng(S + at)
    labels = 4 + (np.arange(S) % (V - 4))
    labels[at - 1:at + 2] = (3, 1, 2)
    head = 2 * at + 4
    T = head + sum(r[1] for r in runs) + 2 * (S - at) + tail
    x = g.normal(size=(1, T, V))
    t = head
    for name, n, boost in runs:
        x[0, t:t + n, names[name]] += boost
        t += n
    return (torch.tensor(x, dtype=F32, device=DEV), torch.tensor(labels[None], dtype=torch.int32, device=DEV),
            torch.tensor([T], dtype=torch.int32, device=DEV), torch.tensor([S], dtype=torch.int32, device=DEV))


def backwards(logits, targets, il, tl):
    """The same case with frames and labels reversed: its states are those of the chain from the end."""
    return logits.flip(1).contiguous(), targets.flip(1).contiguous(), il, tl


@pytest.mark.parametrize("S,at,boost,K", [(100, 44, 16.0, 59), (200, 90, 18.0, 55), (300, 60, 12.0, 79),
                                          (300, 150, 14.0, 75), (500, 100, 10.0, 100), (500, 100, 14.0, 75)])
def test_ctc_path_from_a_lane_far_below(S, at, boost, K):
    """b, favoured first, lifts the lane of a and b more than 1000 octaves above the lane of c.  The path that counts
    waits before c through that, goes from c to a and then has a's frames: all of Z crosses between the two lanes."""
    case = run_case(S, at, [("b", K, boost), ("c", 12, boost), ("a", K + 12, boost)])
    for logits, targets, il, tl in (case, backwards(*case)):
        ref, _ = R.ctc(logits, targets, il, tl, 0, False)
        loss = tr.ctc_loss(logits, targets, il, tl).double().cpu()
        # check_ctc's bound: n frames' normalisers and steps, and the loss's own rounding
        assert abs(loss - ref) <= logits.shape[1] * 100 * E + E * ref + 1e-6, (float(loss), float(ref))


def sharp_check(logits, targets, il, tl, blank=0):
    """check_ctc, and the gradient against what the stored words leave: an emission is rounded by 2^-21 of itself, its
    exponent (log2 e in fp32, a difference of logits up to 32) by 2^-20, so a posterior, a share of two products of n
    of them, by less than n 2^-19."""
    _, grad = check_ctc(logits, targets, il, tl, blank, dloss=torch.ones(logits.shape[0], device=DEV))
    ref = R.ctc(logits, targets, il, tl, blank, False)[1]
    d = (grad.double().cpu() - ref).abs()
    bound = rounded(logits.dtype, ref) + logits.shape[1] * 2.0 ** -19 + (logits.shape[2] / 256 + 100) * E
    assert (d <= bound).all(), float(d.max())


@pytest.mark.parametrize("S,at,K,boost,back", [(100, 44, 100, 15.0, 5), (300, 147, 75, 20.0, 5), (300, 150, 40, 30.0, 3),
                                               (500, 240, 60, 25.0, 5), (1200, 600, 90, 25.0, 5)])
def test_ctc_posterior_far_below_its_lane(S, at, K, boost, back):
    """a and b in one lane, b favoured K frames and a behind it: a's states lie up to 3246 octaves below b's and carry
    the posterior; words against the lane's largest would drop them."""
    case = run_case(S, at, [("b", K, boost), ("a", K + back, boost)])
    sharp_check(*case)
    sharp_check(*backwards(*case))


@pytest.mark.parametrize("S,at", [(60, 24), (100, 45), (300, 148), (500, 243)])
def test_ctc_posterior_in_a_blank_far_below_its_label(S, at):
    """The label favoured, then the blank, then the label again: the posterior lies on the blank before it."""
    case = run_case(S, at, [("a", 80, 20.0), ("blank", 80, 20.0), ("a", 85, 20.0)])
    sharp_check(*case)
    sharp_check(*backwards(*case))


def test_ctc_utterances_far_apart_beside_others():
    """Only the utterances that need it are walked with every state's exponent; a captured call does the same."""
    far = [run_case(100, 44, [("b", 100, 15.0), ("a", 105, 15.0)]), run_case(100, 45, [("a", 80, 20.0), ("blank", 80, 20.0),
                                                                                      ("a", 85, 20.0)])]
    plain = ctc_case(31, 3, 560, 13, 100, F32, ([560, 410, 0], [100, 90, 0]))
    T = 560
    logits, targets = [plain[0]], [plain[1]]
    for x, lab, _, _ in far:
        logits.append(torch.cat([x, torch.full((1, T - x.shape[1], 13), float("nan"), device=DEV)], 1))
        targets.append(lab)
    il, tl = (torch.cat([plain[i], *[c[i] for c in far]]) for i in (2, 3))
    order = torch.tensor([3, 0, 4, 1, 2], device=DEV)
    case = [t[order].contiguous() for t in (torch.cat(logits), torch.cat(targets), il, tl)]
    sharp_check(*case)

    def step():
        x = case[0].detach().requires_grad_()
        loss = tr.ctc_loss(x, *case[1:])
        return loss.detach(), torch.autograd.grad(loss, x, torch.ones(5, device=DEV))[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


# ---- CTC: emissions far apart ----------------------------------------------------------------------------------------
def test_ctc_needed_class_far_below():
    """A needed class far below the frame's likeliest has a finite loss by definition, no mask: one frame of 1000
    against 0, single frames of thousands in an utterance, every frame of a long one, and the border at 11000."""
    one = torch.tensor([[[1000.0, 0.0]]], device=DEV)
    i = torch.ones(1, dtype=torch.int32, device=DEV)
    assert tr.ctc_loss(one, i[None], i, i).item() == 1000.0
    check_ctc(one, i[None], i, i)
    check_ctc(one, i[None], i, i, zero_infinity=True)
    g = np.random.default_rng(40)
    for seed, T, V, S, share, gap in ((41, 40, 30, 9, 0.1, 900), (42, 90, 12, 30, 0.3, 5000), (43, 64, 8, 20, 1.0, 10900),
                                      (44, 700, 40, 310, 0.05, 3000), (45, 1100, 40, 500, 0.02, 700)):
        for dtype in (F32, BF, HF):
            case = ctc_case(seed, 2, T, V, S, dtype, ([T, T - 7], [S, S // 2]))
            at = torch.from_numpy(g.random((2, T, V)) < share).to(DEV)
            low = torch.from_numpy(g.uniform(0.5, 1.0, (2, T, V)) * gap).to(DEV)
            logits = (case[0].double() - torch.where(at, low, 0.0)).to(dtype)
            check_ctc(logits, *case[1:])
            check_ctc(logits, *case[1:], zero_infinity=True)
    near, beyond = (torch.tensor([[[0.0, -v]]], device=DEV) for v in (10999.0, 11001.0))
    assert tr.ctc_loss(near, i[None], i, i).item() == 10999.0
    assert tr.ctc_loss(beyond, i[None], i, i).item() == math.inf


def test_ctc_needed_class_far_below_over_the_longest_chain():
    """Every frame of the longest utterance 10000 below: exponents of -2.3e8 in the states."""
    T = tr.MAX_CTC_FRAMES
    logits = torch.zeros(1, T, 3, device=DEV)
    logits[:, :, 1:] = -10000.0
    logits[:, :, 0] = -9000.0
    logits[:, ::2, 0] = 0.0
    logits[:, 1::2, 2] = 0.0                             # not of the transcript
    targets = torch.ones(1, 5, dtype=torch.int32, device=DEV)
    check_ctc(logits, targets, lens_of([T]), lens_of([5]))


# ---- norms: spreads far from 1 ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [40, 1001, 1024])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("spread,eps", [(1e10, EPS), (1e13, EPS), (1e15, EPS), (1e17, EPS), (1e-14, 1e-30)])
def test_layer_norm_gradient_at_far_spreads(spread, eps, dtype, D):
    """Rows whose deviation is far from 1, up to where its square still fits fp32 and down to an eps of 1e-30: the
    gradient is as near as at 1, and a constant row's is that of eps."""
    x, dy = rand(50, (2, 5, D), dtype, spread), rand(51, (2, 5, D), dtype)
    x[0, 1] = x[0, 1, 0]
    w, b = rand(52, (D,), F32, 0.2, 1.0), rand(53, (D,), F32)
    ref, rdw, rdb, r, xh = R.layer_norm_backward(dy, x, w, eps)
    dx, dw, db = tr.layer_norm_backward(dy, x, w, eps)
    even = [i for i in range(10) if i != 1]
    # of the constant row the formula has r of eps alone, 1e15 here: x - m is exactly 0 in neither 64 bits nor fp32
    bound = (grads_bound(dtype, ref, dy, x, w, r, None) - 1e-30 + torch.finfo(dtype).smallest_normal * 2.0 ** -8)
    close(dx.view(10, D)[even], ref.view(10, D)[even], bound.view(10, D)[even], "dx")
    assert torch.isfinite(dx).all()
    fx, fres, fw, fb = tr.dropout_add_layer_norm_backward(dy, None, x, w, rng_of(), 0.0, eps=eps)
    close(fres.view(10, D)[even], ref.view(10, D)[even], bound.view(10, D)[even], "dresidual")
    assert torch.equal(fx, fres) and torch.equal(fw, dw) and torch.equal(fb, db)
    bw, bb = param_bounds(F32, rdw, rdb, dy, x, r, xh, None)
    if spread > 1:
        close(dw, rdw, bw, "dw")
    close(db, rdb, bb, "db")


# ---- tracers ---------------------------------------------------------------------------------------------------------
def test_traced_calls_compute():
    """make_fx and torch.jit.trace record the ops of every function, and their graphs compute on other inputs."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, y = (rand(s, (2, 5, 40), F32) for s in (60, 61))
    w, b, rng = rand(62, (40,), F32, 0.2, 1.0), rand(63, (40,), F32), rng_of()
    logits, targets, il, tl = ctc_case(64, 2, 9, 7, 3, F32)
    other = rand(65, (2, 9, 7), F32)
    rows = [lambda a: tr.layer_norm(a, w, b), lambda a: tr.layer_norm_backward(a, y, w)[0],
            lambda a: tr.dropout_add(a, rng, 0.3, residual=y), lambda a: tr.dropout_add_backward(a, rng, 0.3),
            lambda a: tr.dropout_add_layer_norm(a, y, w, b, rng, 0.3)[0],
            lambda a: tr.dropout_add_layer_norm_backward(a, a, y, w, rng, 0.3)[1]]
    for f, at, to in [(f, x, y) for f in rows] + [(lambda a: tr.ctc_loss(a, targets, il, tl), logits, other)]:
        want = f(to)
        graphs = [make_fx(f)(at), make_fx(f, pre_dispatch=True)(at), torch.jit.trace(f, at, check_trace=False)]
        for g in graphs:
            assert torch.equal(g(to), want)


def test_traced_gradients_compute():
    """A tracer that sees only the backward pass of a call made before it records the ops of that."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, y = (rand(s, (2, 5, 40), F32) for s in (66, 67))
    w, b, rng = rand(68, (40,), F32, 0.2, 1.0), rand(69, (40,), F32), rng_of()
    logits, targets, il, tl = ctc_case(70, 2, 9, 7, 3, F32)
    calls = [(lambda a: tr.layer_norm(a, w, b), x), (lambda a: tr.dropout_add(a, rng, 0.3, residual=y), x),
             (lambda a: tr.dropout_add_layer_norm(a, y, w, b, rng, 0.3)[0], x),
             (lambda a: tr.dropout_add_layer_norm(a, y, w, b, rng, 0.3)[1], x),
             (lambda a: tr.ctc_loss(a, targets, il, tl), logits)]
    for f, at in calls:
        leaf = at.clone().requires_grad_()
        out = f(leaf)
        first, second = (torch.linspace(a, 2.0, out.numel(), device=DEV).reshape(out.shape) for a in (-1.0, 0.5))
        graph = make_fx(lambda d: torch.autograd.grad(out, leaf, d, retain_graph=True)[0])(first)
        assert torch.equal(graph(second), torch.autograd.grad(out, leaf, second, retain_graph=True)[0])


def test_forward_mode_is_refused():
    """Dual tensors are refused by the functions and by the ops behind them."""
    from torch.autograd import forward_ad
    x, w = rand(70, (2, 3, 16), F32), torch.ones(16, device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        for f in (tr.layer_norm, lambda *a: torch.ops.granite.layer_norm(*a, EPS)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(dual, w, w)
            assert torch.equal(f(x, w, w), tr.layer_norm(x, w, w))


# ---- empty batches ---------------------------------------------------------------------------------------------------
def test_batches_without_frames_take_lengths():
    w, rng = torch.ones(32, device=DEV), rng_of()
    for shape, lengths in (((3, 0, 32), [0, 0, 0]), ((0, 5, 32), []), ((0, 0, 32), [])):
        x, lens = torch.empty(shape, dtype=BF, device=DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
        assert tr.layer_norm(x, w, w, lengths=lens).shape == shape
        dx, dw, db = tr.layer_norm_backward(x, x, w, lengths=lens)
        assert dx.shape == shape and not dw.any() and not db.any()
        assert tr.dropout_add(x, rng, 0.1, residual=x, lengths=lens).shape == shape
        y, h = tr.dropout_add_layer_norm(x, x, w, w, rng, 0.1, lengths=lens)
        assert y.shape == h.shape == shape
        dx, dres, dw, db = tr.dropout_add_layer_norm_backward(x, x, x, w, rng, 0.1, lengths=lens)
        assert dres.shape == shape and not dw.any() and not db.any()
        leaf = x.clone().requires_grad_()
        tr.layer_norm(leaf, w, w, lengths=lens).sum().backward()
        assert leaf.grad.shape == shape


# ---- what ran before -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [256, 512, 1024, 2048])
def test_views_keep_the_inference_kernel(D):
    """Views of bf16 rows, off the 16-byte grid among them, have the inference kernel's bits."""
    from granite_conv_b200 import ops
    wide = rand(80, (64, 2 * D + 8), BF, 1.3, 0.7)
    w, b = rand(81, (D,), BF, 0.1, 1.0), rand(82, (D,), BF)
    for x in (wide[:, 3:3 + D], wide[:, 8:8 + D], wide[::2, :D], wide[1:3, 5:5 + D],
              wide[:, 1:1 + D].t().contiguous().t(), wide.view(8, 8, -1)[:, 1:4, 7:7 + D]):
        want = ops.layernorm(x.contiguous().view(-1, D), w, b, EPS).view(x.shape)
        assert torch.equal(torch.ops.granite.layer_norm(x, w, b, EPS), want)
        assert torch.equal(tr.layer_norm(x, w, b, EPS), want)


# ---- sizes that an int does not hold ---------------------------------------------------------------------------------
def test_sizes_past_32_bits_are_refused():
    """Refused before anything is allocated: the tensors are one element, expanded."""
    one, i = torch.zeros(1, dtype=BF, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="elements expected"):
        tr.dropout_add(one.expand(2 ** 32 + 5), rng_of(), 0.1)
    with pytest.raises(RuntimeError, match="classes"):
        tr.ctc_loss(one.expand(1, 1, 2 ** 32 + 5), i[None], i, i)
    with pytest.raises(RuntimeError, match="utterances"):
        tr.ctc_loss(one.expand(2 ** 32 + 1, 0, 5), i.expand(2 ** 32 + 1, 0), i.expand(2 ** 32 + 1), i.expand(2 ** 32 + 1))


# ---- a wait that runs out --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("side,half", [(0, 0), (1, 0), (0, 1), (1, 1)])
def test_ctc_wait_that_runs_out_is_nan(side, half, far):
    """A copy armed and never issued on one side: the status word reads 0x105, that utterance's gradient is NaN, its
    loss too before the sides have met, the other utterance's are what they are, and the next call is as always.  far:
    an utterance that is walked again for its posteriors."""
    from granite_conv_b200 import _lib
    if far:
        case = run_case(60, 24, [("a", 80, 20.0), ("blank", 80, 20.0), ("a", 85, 20.0)])
        logits, targets, il, tl = (torch.cat([t, t]).contiguous() for t in case)
    else:
        logits, targets, il, tl = ctc_case(90, 2, 150, 20, 40, F32, ([150, 141], [40, 39]))
    _, T, V = logits.shape
    S = targets.shape[1]
    L, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    loss = torch.zeros(2, device=DEV)
    state = torch.zeros(L.gsn_ctc_loss_state_bytes(2, T, S), dtype=torch.uint8, device=DEV)
    ws = torch.zeros(L.gsn_ctc_loss_workspace_bytes(2, T, S, 1), dtype=torch.uint8, device=DEV)
    _lib.device_status(stream, clear=True)
    _lib.call("gsn_selftest_ctc_withheld", logits.data_ptr(), T * V, V, targets.data_ptr(), il.data_ptr(), tl.data_ptr(),
              2, T, V, S, 0, 2, loss.data_ptr(), state.data_ptr(), state.numel(), ws.data_ptr(), ws.numel(), side, half,
              stream)
    assert _lib.device_status(stream, clear=True) == 0x105
    want = tr.ctc_loss(logits, targets, il, tl)
    assert loss[1] == want[1] and (torch.isnan(loss[0]) if half == 0 else loss[0] == want[0])
    grad = tr._ctc_loss_backward(torch.ones(2, device=DEV), logits, targets, il, tl, state, 0, False)
    assert torch.isnan(grad[0]).all() and torch.isfinite(grad[1]).all()
    _, good = check_ctc(logits, targets, il, tl, dloss=torch.ones(2, device=DEV))
    assert torch.equal(grad[1], good[1])
    assert _lib.device_status(stream, clear=False) == 0


def test_ctc_transcript_at_the_lowest_value():
    """A frame whose classes of the transcript all have the type's lowest value beside others at 0: the loss is that
    value, and the gradient finite; two such frames are beyond fp32.  Next to a log Z of 3.4e38 the posteriors of a
    64-bit recursion are lost (an ulp of 2^76): they are taken from the same frame with the other classes impossible,
    which scales Z and changes no path's share of it."""
    for dtype in (F32, BF, HF):
        low = torch.finfo(dtype).min
        logits, targets, il, tl = ctc_case(46, 2, 12, 9, 3, dtype, labels=[[1, 2, 3]] * 2)
        logits[:, 5, :4] = low
        logits[1, 6, :4] = low
        shares = logits[:1].clone()
        shares[:, 5, :4], shares[:, 5, 4:] = 0.0, -math.inf
        ref = R.ctc(shares, targets[:1], il[:1], tl[:1], 0, False)[1]
        p, q = (torch.softmax(t.double().cpu(), -1) for t in (logits[:1], shares))
        ref = p - (q - ref)
        for zero_infinity in (False, True):
            x = logits.clone().requires_grad_()
            loss = tr.ctc_loss(x, targets, il, tl, zero_infinity=zero_infinity)
            grad, = torch.autograd.grad(loss.sum(), x)
            assert abs(loss[0].item() + low) <= 2.0 ** -24 * abs(low) + 100
            bound = rounded(dtype, ref) + (9 / 256 + 100 + 12 * 64 + 164) * E        # as in check_ctc
            close(grad[:1], ref, bound, (dtype, zero_infinity))
            if dtype == HF:
                assert abs(loss[1].item() + 2 * low) < 200
            else:
                assert loss[1].item() == (0.0 if zero_infinity else math.inf)


@pytest.mark.parametrize("D", [139, 141, 150, 281, 282])
def test_dropout_on_either_side_of_its_rule(D):
    """Off the 16-byte grid, around the width where blocks of 256 columns take over: the same mask and values."""
    x, res = rand(95, (3, 7, D), BF), rand(96, (3, 7, D), BF)
    keep = R.keep_mask(x.shape, 99, 1, 6, 0.4)
    assert torch.equal(tr.dropout_add(torch.ones_like(x), rng_of(99, 1), 0.4, site=6).cpu() != 0, keep)
    out = tr.dropout_add(x, rng_of(99, 1), 0.4, residual=res, site=6, lengths=lens_of([7, 0, 3]))
    ref = R.dropout_add(x, res, 99, 1, 6, 0.4, 1.0, [7, 0, 3])
    k = R.factor(0.4, 1.0)
    close(out, ref, rounded(BF, ref) + 2 * E * (k * x.double().cpu().abs() + res.double().cpu().abs()))
