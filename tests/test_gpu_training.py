"""The fine-tuning operators on the GPU against plain 64-bit evaluations of their formulas.

Bounds.  rounded(t, v) is one rounding to the output type: finfo(t).eps / 2 relative to the value, and below the normal
range, where the values of t lie smallest_normal * eps apart, half of that (fp16: 2^-14 * 2^-10 / 2 = 2^-25, which a
gradient of 1e-5 meets).  E = 2^-24 is one fp32 rounding.
A row's sums run over at most 32 elements a lane, 5 shuffles and 8 warps, so 64 E covers their roundings; they enter
through the largest magnitudes of the row.  Sums over rows add at most M + 64 roundings of the summed magnitudes.
"""
import math

import numpy as np
import pytest
import torch

import train_ref as R
from granite_conv_b200 import ops
from granite_conv_b200 import training as tr

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24
EPS = 1e-5

# (shape, lengths): one row, the encoder's width, narrow, odd and ragged widths, several warps a row, the widest
SHAPES = [((1, 1, 1), None), ((1, 1, 1024), None), ((2, 37, 1024), [37, 11]), ((3, 5, 160), [5, 0, 1]),
          ((2, 9, 7), None), ((2, 9, 257), [9, 3]), ((1, 33, 1001), None), ((2, 17, 2048), None), ((1, 6, 2051), None),
          ((2, 3, 4096), [3, 1]), ((1, 3, 8192), None), ((1, 2, 8191), None), ((1, 700, 24), None), ((2, 8, 153), [8, 2]), ((2, 8, 155), [3, 8])]


def rand(seed, shape, dtype, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).to(DEV)


def lens_of(lengths, dtype=torch.int32):
    return None if lengths is None else torch.tensor(lengths, dtype=dtype, device=DEV)


def rng_of(seed=0x1234567890ABCDEF, offset=5):
    return torch.tensor([seed, offset], dtype=torch.int64, device=DEV)


def rounded(dtype, ref):
    f = torch.finfo(dtype)
    return (f.eps / 2 * ref.abs()).clamp(min=f.smallest_normal * f.eps / 2)


def close(out, ref, bound, what=""):
    d = (out.double().cpu() - ref).abs()
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(d)
    assert out.shape == ref.shape, what
    worst = (d - bound).max() if d.numel() else torch.tensor(-1.0)
    fine = not torch.isnan(d).any().item() and (d <= bound).all().item()
    assert fine, f"{what}: {float(worst):.3e} beyond the bound"


def row_max(x):
    return x.double().cpu().abs().amax(-1, keepdim=True)


def norm_bound(dtype, ref, x, w, b, r):
    return rounded(dtype, ref) + 64 * E * (w.double().cpu().abs() * r * 2 * row_max(x) + b.double().cpu().abs()) + 1e-30


def grads_bound(dtype, ref, dy, x, w, r, lengths):
    """Of dx: xh is off by 64 E * 2 X with X = r max|x|, and enters twice with the row's largest g."""
    X = r * row_max(x.double().cpu().masked_fill(R.padding(x.shape, lengths), 0.0))
    G = row_max(dy.double().cpu() * w.double().cpu())
    return rounded(dtype, ref) + 64 * E * r * G * 2 * (1 + X) ** 2 + 1e-30


def param_bounds(wtype, dw, db, dy, x, r, xh, lengths):
    pad = R.padding(x.shape, lengths)
    rows = tuple(range(x.dim() - 1))
    M = x.numel() // x.shape[-1]
    a = dy.double().cpu().masked_fill(pad, 0.0).abs()
    X = r * row_max(x.double().cpu().masked_fill(pad, 0.0))
    return (rounded(wtype, dw) + ((M + 64) * E * a * xh.abs() + 128 * E * a * X).sum(rows) + 1e-30,
            rounded(wtype, db) + (M + 64) * E * a.sum(rows) + 1e-30)


# ---- layer norm ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,wtype", [(BF, F32), (BF, BF), (HF, HF), (F32, F32)])
@pytest.mark.parametrize("shape,lengths", SHAPES)
def test_layer_norm(shape, lengths, dtype, wtype):
    D = shape[-1]
    x, dy = rand(1, shape, dtype, 1.3, 0.7), rand(2, shape, dtype)
    w, b = rand(3, (D,), wtype, 0.2, 1.0), rand(4, (D,), wtype, 0.3)
    lens = lens_of(lengths)
    if lengths is not None:             # what padding holds does not matter
        pad = R.padding(shape, lengths).to(DEV)
        x, dy = x.masked_fill(pad, float("nan")), dy.masked_fill(pad, float("inf"))
    y = tr.layer_norm(x, w, b, EPS, lens)
    clean = x.masked_fill(R.padding(shape, lengths).to(DEV), 0.0)
    ref, r = R.layer_norm(clean, w, b, EPS, lengths)
    close(y, ref, norm_bound(dtype, ref, clean, w, b, r), "y")
    dx, dw, db = tr.layer_norm_backward(dy, x, w, EPS, lens)
    gclean = dy.masked_fill(R.padding(shape, lengths).to(DEV), 0.0)
    rdx, rdw, rdb, r, xh = R.layer_norm_backward(gclean, clean, w, EPS, lengths)
    close(dx, rdx, grads_bound(dtype, rdx, gclean, clean, w, r, lengths), "dx")
    bw, bb = param_bounds(wtype, rdw, rdb, gclean, clean, r, xh, lengths)
    close(dw, rdw, bw, "dw")
    close(db, rdb, bb, "db")
    assert dw.dtype == wtype and dx.dtype == dtype


def test_layer_norm_many_rows():
    """More rows than the grid has places, ragged: every row group takes several."""
    B, T, D = 6, 1531, 1024
    lengths = [1531, 1, 1530, 700, 0, 64]
    x, dy, w, b = rand(1, (B, T, D), BF), rand(2, (B, T, D), BF), rand(3, (D,), F32, 0.2, 1.0), rand(4, (D,), F32)
    ref, r = R.layer_norm(x, w, b, EPS, lengths)
    close(tr.layer_norm(x, w, b, EPS, lens_of(lengths)), ref, norm_bound(BF, ref, x, w, b, r))
    out = tr.layer_norm_backward(dy, x, w, EPS, lens_of(lengths, torch.int64))
    rdx, rdw, rdb, r, xh = R.layer_norm_backward(dy, x, w, EPS, lengths)
    close(out[0], rdx, grads_bound(BF, rdx, dy, x, w, r, lengths))
    for o, v, bound in zip(out[1:], (rdw, rdb), param_bounds(F32, rdw, rdb, dy, x, r, xh, lengths)):
        close(o, v, bound)
    again = tr.layer_norm_backward(dy, x, w, EPS, lens_of(lengths))
    assert all(torch.equal(a, c) for a, c in zip(out, again))


def test_many_utterances():
    """More utterances than a walk takes at once, lengths from zero up and out of range, both operators and directions."""
    B, T, D = 2500, 3, 40
    g = np.random.default_rng(5)
    given = g.integers(-1, T + 2, B)
    given[:3] = (0, T, 2 ** 31 - 1)
    lengths = np.clip(given, 0, T).tolist()
    lens = torch.tensor(given, dtype=torch.int32, device=DEV)
    x, dy, res = rand(1, (B, T, D), BF), rand(2, (B, T, D), BF), rand(5, (B, T, D), BF)
    w, b = rand(3, (D,), F32, 0.2, 1.0), rand(4, (D,), F32)
    ref, r = R.layer_norm(x, w, b, EPS, lengths)
    close(tr.layer_norm(x, w, b, EPS, lens), ref, norm_bound(BF, ref, x, w, b, r))
    rdx, rdw, rdb, r, xh = R.layer_norm_backward(dy, x, w, EPS, lengths)
    bw, bb = param_bounds(F32, rdw, rdb, dy, x, r, xh, lengths)
    dx, dw, db = tr.layer_norm_backward(dy, x, w, EPS, lens)
    close(dx, rdx, grads_bound(BF, rdx, dy, x, w, r, lengths))
    close(dw, rdw, bw)
    close(db, rdb, bb)
    y, h = tr.dropout_add_layer_norm(x, res, w, b, rng_of(), 0.2, lengths=lens)
    assert torch.equal(h, tr.dropout_add(x, rng_of(), 0.2, residual=res, lengths=lens))
    pad = R.padding(x.shape, lengths).to(DEV)
    assert torch.equal(h.masked_select(pad), res.masked_select(pad)) and not y.masked_select(pad).any()
    out = tr.dropout_add_layer_norm_backward(dy, res, h, w, rng_of(), 0.2, lengths=lens)
    assert torch.equal(out[1].masked_select(pad), res.masked_select(pad)) and not out[0].masked_select(pad).any()


def test_layer_norm_keeps_the_inference_kernel():
    """What granite::layer_norm took before keeps its kernel and its bits, with and without a gradient to record."""
    x, w, b = rand(1, (2, 37, 1024), BF), rand(2, (1024,), BF, 0.1, 1.0), rand(3, (1024,), BF)
    old = ops.layernorm(x.view(-1, 1024), w, b, EPS).view(x.shape)
    assert torch.equal(torch.ops.granite.layer_norm(x, w, b, EPS), old)
    assert torch.equal(tr.layer_norm(x, w, b), old)
    assert torch.equal(tr.layer_norm(x.requires_grad_(), w, b).detach(), old)


def test_strides_and_alignment():
    """Row strides, a tensor off the 16-byte grid, transposed and broadcast inputs, a zero-stride weight.  Rows off the
    grid are added up in another order than those on it: within the bounds, not the same bits."""
    B, T, D = 2, 5, 64
    w, b = rand(3, (D,), F32, 0.2, 1.0), rand(4, (D,), F32)
    wide = rand(1, (B, T, 2 * D), BF)
    off = rand(2, (B * T * D + 1,), BF)[1:].view(B, T, D)
    cases = [wide[..., :D], wide[..., D:], wide[..., 3:3 + D], off, rand(5, (T, B, D), BF).transpose(0, 1),
             rand(6, (B, D, T), BF).transpose(1, 2), rand(7, (1, 1, D), BF).expand(B, T, D), wide[:, ::2, :D]]
    for i, x in enumerate(cases):
        dense = x.contiguous().clone()
        dy, rng = rand(8, x.shape, BF), rng_of()
        ref, r = R.layer_norm(x, w, b, EPS)
        close(tr.layer_norm(x, w, b), ref, norm_bound(BF, ref, x, w, b, r), i)
        for g, at in ((dy, x), (x, dy)):
            rdx, rdw, rdb, r, xh = R.layer_norm_backward(g, at, w, EPS)
            dx, dw, db = tr.layer_norm_backward(g, at, w)
            close(dx, rdx, grads_bound(BF, rdx, g, at, w, r, None), i)
            bw, bb = param_bounds(F32, rdw, rdb, g, at, r, xh, None)
            close(dw, rdw, bw, i)
            close(db, rdb, bb, i)
            fx, fres, fw, fb = tr.dropout_add_layer_norm_backward(g, at, at, w, rng, 0.3)
            total = rdx + at.double().cpu()
            bound = rounded(BF, total) + grads_bound(F32, rdx, g, at, w, r, None) + E * total.abs()
            close(fres, total, bound, i)
            want = torch.where(R.keep_mask(x.shape, int(rng[0]), int(rng[1]), 0, 0.3), total * R.factor(0.3, 1.0), 0.0)
            close(fx, want, R.factor(0.3, 1.0) * bound + rounded(BF, want), i)
            assert torch.equal(fw, dw) and torch.equal(fb, db), i
        assert torch.equal(tr.dropout_add(x, rng, 0.3, residual=x), tr.dropout_add(dense, rng, 0.3, residual=dense)), i
        y, h = tr.dropout_add_layer_norm(x, x, w, b, rng, 0.3)
        assert torch.equal(h, tr.dropout_add(x, rng, 0.3, residual=x)), i
        rh = R.dropout_add(x, x, int(rng[0]), int(rng[1]), 0, 0.3, 1.0)
        ry, r = R.layer_norm(rh, w, b, EPS)
        extra = 8 * E * row_max(rh) * r * w.double().cpu().abs() * (2 + r * row_max(rh))
        close(y, ry, norm_bound(BF, ry, rh, w, b, r) + extra, i)
    one = torch.ones(1, device=DEV).expand(D)
    assert torch.equal(tr.layer_norm(wide[..., :D], one, one), tr.layer_norm(wide[..., :D], one.clone(), one.clone()))


def test_layer_norm_special_rows():
    """A constant row, the type's largest values, and rows with inf and NaN, which must not reach other rows."""
    D = 1024
    x = rand(1, (1, 5, D), F32)
    w, b = rand(2, (D,), F32, 0.1, 1.0), rand(3, (D,), F32)
    x[0, 1] = 3.25
    x[0, 2, 7] = float("inf")
    x[0, 3, 9] = float("nan")
    y = tr.layer_norm(x, w, b)
    assert torch.equal(y[0, 1], b)                       # x - m is exactly zero
    assert torch.isnan(y[0, 2]).all() and torch.isnan(y[0, 3]).all()
    good = [0, 4]
    ref, r = R.layer_norm(x[:, good], w, b, EPS)
    close(y[:, good], ref, norm_bound(F32, ref, x[:, good], w, b, r))
    big = torch.full((1, 1, D), torch.finfo(HF).max, dtype=HF, device=DEV)
    assert torch.equal(tr.layer_norm(big, w, b), b.to(HF)[None, None])


def test_empty_rows():
    w, rng = torch.ones(32, device=DEV), rng_of()
    for shape in ((0, 5, 32), (3, 0, 32), (0, 32)):
        x = torch.empty(shape, dtype=BF, device=DEV)
        assert tr.layer_norm(x, w, w).shape == shape
        dx, dw, db = tr.layer_norm_backward(x, x, w)
        assert dx.shape == shape and not dw.any() and not db.any()
        assert tr.dropout_add(x, rng, 0.1).shape == shape
        y, h = tr.dropout_add_layer_norm(x, x, w, w, rng, 0.1)
        assert y.shape == h.shape == shape
        dx, dres, dw, db = tr.dropout_add_layer_norm_backward(x, None, x, w, rng, 0.1)
        assert dres.shape == shape and not dw.any() and not db.any()
    x = torch.randn(2, 3, 32, device=DEV)                # every utterance empty
    none = lens_of([0, 0])
    assert not tr.layer_norm(x, w, w, lengths=none).any()
    dx, dw, db = tr.layer_norm_backward(x, x, w, lengths=none)
    assert not dx.any() and not dw.any() and not db.any()


# ---- dropout ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("shape,lengths", SHAPES)
def test_dropout_add(shape, lengths, dtype):
    x, res = rand(1, shape, dtype), rand(2, shape, dtype)
    seed, offset, site, p, scale = -3, 2 ** 33 + 9, 2 ** 32 - 1, 0.27, 0.5
    rng, lens = rng_of(seed, offset), lens_of(lengths)
    k = R.factor(p, scale)
    clean = x
    if lengths is not None:
        x = x.masked_fill(R.padding(shape, lengths).to(DEV), float("nan"))
    out = tr.dropout_add(x, rng, p, residual=res, scale=scale, site=site, lengths=lens)
    ref = R.dropout_add(clean, res, seed, offset, site, p, scale, lengths)
    close(out, ref, rounded(dtype, ref) + 2 * E * (k * clean.double().cpu().abs() + res.double().cpu().abs()))
    dx = tr.dropout_add_backward(x, rng, p, scale=scale, site=site, lengths=lens)
    ref = R.dropout_add(clean, None, seed, offset, site, p, scale, lengths)
    close(dx, ref, rounded(dtype, ref) + 2 * E * ref.abs())
    assert torch.equal(dx != 0, (ref != 0).to(DEV) & (dx != 0)) and not dx[(ref == 0).to(DEV)].any()


def test_dropout_probabilities():
    x, rng = rand(1, (64, 1000), F32) + 10, rng_of()
    assert torch.equal(tr.dropout_add(x, rng, 0.0), x)
    assert not tr.dropout_add(x, rng, 1.0).any()
    bad = x.clone()
    bad[3] = float("inf")
    assert not tr.dropout_add(bad, rng, 1.0).any()       # dropped, not multiplied by zero
    assert torch.equal(tr.dropout_add(bad, rng, 1.0, residual=x), x)
    a, b = tr.dropout_add(x, rng, 0.5, site=1), tr.dropout_add(x, rng, 0.5, site=2)
    assert not torch.equal(a != 0, b != 0)
    rng2 = rng.clone()
    rng2[1] += 1
    assert not torch.equal(a != 0, tr.dropout_add(x, rng2, 0.5, site=1) != 0)


def test_dropout_mask_is_the_same_everywhere():
    """One mask for a seed, offset and site, whatever the type, operator or direction."""
    shape, rng, p = (3, 50, 264), rng_of(99, 1), 0.4
    keep = R.keep_mask(shape, 99, 1, 6, p).to(DEV)
    w = torch.ones(264, device=DEV)
    for dtype in (BF, HF, F32):
        one = torch.ones(shape, dtype=dtype, device=DEV)
        zero = torch.zeros(shape, dtype=dtype, device=DEV)
        assert torch.equal(tr.dropout_add(one, rng, p, site=6) != 0, keep)
        assert torch.equal(tr.dropout_add_layer_norm(one, zero, w, w, rng, p, site=6)[1] != 0, keep)
        dx, dres, _, _ = tr.dropout_add_layer_norm_backward(zero, one, one, w, rng, p, site=6)
        assert torch.equal(dx != 0, keep) and torch.equal(dres, one)


# ---- dropout, residual and norm together -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,wtype", [(BF, F32), (HF, HF), (F32, F32)])
@pytest.mark.parametrize("shape,lengths", SHAPES)
def test_dropout_add_layer_norm(shape, lengths, dtype, wtype):
    D = shape[-1]
    x, res = rand(1, shape, dtype), rand(2, shape, dtype, 1.0, 0.4)
    w, b = rand(3, (D,), wtype, 0.2, 1.0), rand(4, (D,), wtype, 0.3)
    rng, lens, p, scale, site = rng_of(7, 8), lens_of(lengths), 0.2, 0.5, 3
    pad = R.padding(shape, lengths).to(DEV)
    k = R.factor(p, scale)
    y, h = tr.dropout_add_layer_norm(x.masked_fill(pad, float("nan")), res, w, b, rng, p, scale, site, EPS, lens)
    rh = R.dropout_add(x, res, 7, 8, site, p, scale, lengths)
    close(h, rh, rounded(dtype, rh) + 2 * E * (k * x.double().cpu().abs() + res.double().cpu().abs()), "h")
    ry, r = R.layer_norm(rh, w, b, EPS, lengths)
    # h itself is off by 2 E of its terms, which the row's deviation magnifies
    extra = 4 * E * (k * row_max(x) + row_max(res)) * r * w.double().cpu().abs() * (2 + r * row_max(rh))
    close(y, ry, norm_bound(dtype, ry, rh, w, b, r) + extra, "y")

    dy, dh = rand(5, shape, dtype), rand(6, shape, dtype, 0.3)
    for side in (dh, None):
        dx, dres, dw, db = tr.dropout_add_layer_norm_backward(
            dy.masked_fill(pad, float("nan")), side, h.masked_fill(pad, float("nan")), w, rng, p, scale, site, EPS, lens)
        g, rdw, rdb, r, xh = R.layer_norm_backward(dy, h, w, EPS, lengths)
        bound = grads_bound(F32, g, dy, h, w, r, lengths)
        if side is not None:
            g = g + side.double().cpu()
            bound = bound + E * g.abs()
        close(dres, g, rounded(dtype, g) + bound, "dres")
        keep = R.keep_mask(shape, 7, 8, site, p) & ~R.padding(shape, lengths)
        rdx = torch.where(keep, g * k, 0.0)
        close(dx, rdx, rounded(dtype, rdx) + k * bound + 2 * E * rdx.abs(), "dx")
        bw, bb = param_bounds(wtype, rdw, rdb, dy, h, r, xh, lengths)
        close(dw, rdw, bw, "dw")
        close(db, rdb, bb, "db")


# ---- CTC -------------------------------------------------------------------------------------------------------------
def ctc_case(seed, B, T, V, S, dtype, lengths=None, labels=None, blank=0, spread=2.0):
    g = np.random.default_rng(seed)
    logits = rand(seed, (B, T, V), dtype, spread)
    targets = g.integers(0, V, (B, S)) if labels is None else np.asarray(labels).reshape(B, S)
    if labels is None and V > 1:
        targets = np.where(targets == blank, (targets + 1) % V, targets)
    il, tl = lengths if lengths is not None else ([T] * B, [S] * B)
    return (logits, torch.tensor(targets, dtype=torch.int32, device=DEV), torch.tensor(il, dtype=torch.int32, device=DEV),
            torch.tensor(tl, dtype=torch.int32, device=DEV))


def check_ctc(logits, targets, il, tl, blank=0, zero_infinity=False, dloss=None):
    """The loss adds n frames' normalisers (a sum over V in threads of 256, an exponential within 2 + 1.16 |x| ulp that
    weighs at most log V) and n steps of the chain; the posteriors carry the chain's roundings from both sides."""
    B, T, V = logits.shape
    rl, rg = R.ctc(logits, targets, il, tl, blank, zero_infinity)
    x = logits.detach().requires_grad_()           # as it lies, strides and alignment
    loss = tr.ctc_loss(x, targets, il, tl, blank=blank, zero_infinity=zero_infinity)
    d = torch.linspace(0.5, 2.0, B, device=DEV) if dloss is None else dloss
    grad, = torch.autograd.grad(loss, x, d)
    alone = tr.ctc_loss(logits, targets, il, tl, blank=blank, zero_infinity=zero_infinity)
    assert torch.equal(alone, loss) or torch.isnan(alone).any()
    assert loss.dtype == F32 and grad.dtype == logits.dtype and grad.shape == logits.shape
    n = max(1, T)
    per_frame = (V / 256 + 100) * E
    fin = torch.isfinite(rl)
    got = loss.detach().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(rl)) and torch.equal(got == math.inf, rl == math.inf)
    assert ((got - rl).abs()[fin] <= (n * per_frame + E * rl.abs() + 1e-6)[fin]).all(), (got, rl)
    dd = d.double().cpu()[:, None, None]
    ref = rg * dd
    out = grad.double().cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    ok = ~torch.isnan(ref)
    # p and the posteriors are at most 1 and off by these shares
    bound = rounded(logits.dtype, ref) + dd.abs() * ((V / 256 + 100) * E + (n * 64 + 164) * E)
    assert ((out - ref).abs()[ok] <= bound[ok]).all(), float(((out - ref).abs() - bound)[ok].max())
    return loss, grad


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("B,T,V,S", [(1, 1, 5, 0), (1, 1, 5, 1), (2, 2, 7, 1), (3, 37, 348, 9), (2, 64, 29, 31),
                                     (1, 90, 2, 40), (2, 20, 1001, 7), (1, 50, 17, 25), (1, 9, 4099, 4), (1, 75, 40, 70)])
def test_ctc_loss(B, T, V, S, dtype):
    check_ctc(*ctc_case(B * 1000 + T, B, T, V, S, dtype))


@pytest.mark.parametrize("S", [79, 80, 207, 208, 329, 330, 368, 489, 499, 615, 740, 860, 900, 967, 968])
def test_ctc_label_counts(S):
    """Around the counts where a lane holds more of them or a block fewer frames; long and short chains beside them."""
    il, tl = [2 * S + 40, S + 30, 17], [S, S // 3, 5]
    check_ctc(*ctc_case(100 + S, 3, 2 * S + 40, 50, S, BF, (il, tl)))


def test_ctc_ragged_batch_and_padding():
    """Lengths from zero up, with garbage behind them, and the blank inside the vocabulary."""
    il, tl = [40, 13, 1, 0, 25, 0], [12, 6, 1, 0, 0, 2]
    logits, targets, il, tl = ctc_case(3, 6, 40, 50, 12, BF, (il, tl), blank=31)
    for b in range(6):
        logits[b, int(il[b]):] = float("nan")
        targets[b, int(tl[b]):] = 10 ** 6
    loss, grad = check_ctc(logits, targets, il, tl, blank=31)
    assert loss[3] == 0 and loss[5] == math.inf
    for b in range(6):
        assert not grad[b, int(il[b]):].any()


def test_ctc_repeats_and_infeasible():
    """Repeated labels need a blank between them: exactly enough frames, one too few; the blank as a label."""
    labels = [[1, 1, 1, 2], [1, 1, 1, 2], [2, 2, 2, 2], [1, 0, 2, 1]]
    case = ctc_case(4, 4, 7, 6, 4, F32, ([6, 5, 6, 7], [4, 4, 4, 4]), labels)
    check_ctc(*case)
    loss, grad = check_ctc(*case, zero_infinity=True)
    assert loss[1] == 0 and not grad[1].any()
    loss = tr.ctc_loss(*case)
    assert loss[1] == math.inf and loss[2] == math.inf and torch.isfinite(loss[0])


def test_ctc_long_repeats():
    """One label two hundred times, and few classes: many places of the transcript add into one class."""
    check_ctc(*ctc_case(5, 1, 260, 3, 120, F32, labels=[[1] * 120]))
    check_ctc(*ctc_case(6, 1, 260, 4, 200, F32, ([260], [180])))


def test_ctc_masked_classes():
    """Classes masked with -inf and with the type's lowest value: no gradient there, the others as without them; a
    needed label masked leaves no alignment."""
    for dtype, low in ((F32, -math.inf), (BF, -math.inf), (F32, torch.finfo(F32).min), (BF, torch.finfo(BF).min),
                       (HF, torch.finfo(HF).min)):
        logits, targets, il, tl = ctc_case(7, 2, 30, 40, 6, dtype, labels=[[1, 2, 3, 4, 5, 6]] * 2)
        logits[:, :, 20:] = low
        _, grad = check_ctc(logits, targets, il, tl)
        assert not grad[:, :, 20:].any()
        logits[1, :, 3] = low
        loss = tr.ctc_loss(logits, targets, il, tl)
        assert torch.isfinite(loss[0]) and loss[1] == math.inf


def test_ctc_confident_and_wrong():
    """A model sure of another transcript: the states that carry the posterior lie thousands of octaves below the
    frame's best."""
    B, T, V, S = 2, 300, 30, 60
    logits, targets, il, tl = ctc_case(8, B, T, V, S, F32)
    logits[:, :, 0] += 60.0
    logits[1, :, 7] += 120.0
    loss, _ = check_ctc(logits, targets, il, tl)
    assert (loss > 2000).all()


def test_ctc_bad_input_is_nan():
    """Labels outside the classes, lengths outside the tensors and NaN logits make their own utterance NaN."""
    logits, targets, il, tl = ctc_case(9, 6, 12, 9, 4, F32)
    targets[1, 2] = 9
    targets[2, 0] = -1
    il[3] = 13
    tl[4] = 5
    logits[5, 3, 3] = float("nan")
    x = logits.clone().requires_grad_()
    loss = tr.ctc_loss(x, targets, il, tl, zero_infinity=True)
    grad, = torch.autograd.grad(loss.sum(), x)
    assert torch.isfinite(loss[0]) and torch.isnan(loss[1:]).all()
    assert torch.isfinite(grad[0]).all() and torch.isnan(grad[1:]).all()


def test_ctc_strides_and_index_types():
    """Frames first, a padded class axis, classes outermost, each within the bounds (a row's sum begins at its own
    16-byte boundary, so its order is the alignment's); int64 indices and a broadcast batch, the same bits."""
    logits, targets, il, tl = ctc_case(10, 3, 21, 40, 5, BF)
    base = check_ctc(logits, targets, il, tl)
    wide = torch.zeros(3, 21, 47, dtype=BF, device=DEV)
    wide[..., 3:43] = logits
    for x in (logits.transpose(0, 1).contiguous().transpose(0, 1), wide[..., 3:43],
              logits.transpose(1, 2).contiguous().transpose(1, 2)):
        check_ctc(x, targets, il, tl)
    x = logits.clone().requires_grad_()
    loss = tr.ctc_loss(x, targets.long(), il.long(), tl.long())
    grad, = torch.autograd.grad(loss, x, torch.linspace(0.5, 2.0, 3, device=DEV))
    assert torch.equal(loss, base[0]) and torch.equal(grad, base[1])
    one = logits[:1].expand(3, -1, -1)
    same = tr.ctc_loss(one, targets[:1].expand(3, -1), il, tl)
    assert torch.equal(same, tr.ctc_loss(logits[:1], targets[:1], il[:1], tl[:1]).expand(3))
    assert tr.ctc_loss(logits[:0], targets[:0], il[:0], tl[:0]).shape == (0,)
    empty = tr.ctc_loss(logits[:, :0], targets, torch.zeros_like(il), tl)
    assert (empty == math.inf).all()


def test_ctc_most_labels():
    """The most labels that are taken, on as many frames as they need and a few more."""
    S = tr.MAX_CTC_LABELS
    V, T = 5, S + 40
    labels = [[1 + i % 4 for i in range(S)]]
    check_ctc(*ctc_case(11, 1, T, V, S, F32, labels=labels))


def test_ctc_gradient_against_differences():
    """The kernel's gradient against central differences of the 64-bit loss: h = 1e-4 leaves h^2 / 6 of a third
    derivative below 1, beside the gradient's own bound."""
    logits, targets, il, tl = ctc_case(12, 1, 12, 6, 4, F32)
    _, grad = check_ctc(logits, targets, il, tl, dloss=torch.ones(1, device=DEV))
    x, lab = logits[0].double().cpu(), targets[0].tolist()
    for t in range(0, 12, 3):
        for v in range(6):
            a, b = x.clone(), x.clone()
            a[t, v] += 1e-4
            b[t, v] -= 1e-4
            d = (R.ctc_one(a, lab, 0)[0] - R.ctc_one(b, lab, 0)[0]) / 2e-4
            assert abs(d - float(grad[0, t, v])) < 1e-8 + (12 * 64 + 300) * E


# ---- as they are used ------------------------------------------------------------------------------------------------
def tail_parameters(D, V, seed=20):
    return {"w": rand(seed, (D,), F32, 0.1, 1.0), "b": rand(seed + 1, (D,), F32, 0.1),
            "head": rand(seed + 2, (V, D), F32, D ** -0.5), "hb": rand(seed + 3, (V,), F32, 0.1)}


def tail_loss(ff, x, par, rng, targets, il, tl, p):
    """A block's tail and the character head: half-step residual with dropout, post norm, dropout, head, loss."""
    y, h = tr.dropout_add_layer_norm(ff, x, par["w"], par["b"], rng, p, scale=0.5, site=0, lengths=il)
    y = tr.dropout_add(y, rng, p, site=1, lengths=il)
    logits = y.float() @ par["head"].t() + par["hb"]
    loss = tr.ctc_loss(logits, targets, il, tl)
    return (loss / tl.clamp(min=1)).mean() + 1e-3 * h.float().square().mean()


def tail_case(seed=30, B=3, T=24, D=160, V=30, S=6):
    ff, x = rand(seed, (B, T, D), F32), rand(seed + 1, (B, T, D), F32)
    g = np.random.default_rng(seed)
    targets = torch.tensor(g.integers(1, V, (B, S)), dtype=torch.int32, device=DEV)
    il = torch.tensor([T, T - 5, T // 2], dtype=torch.int32, device=DEV)
    tl = torch.tensor([S, S - 1, 3], dtype=torch.int32, device=DEV)
    return ff, x, targets, il, tl


def test_training_step_against_formulas():
    """Loss and every gradient of the run above, against the same step in 64 bits with torch's own autograd."""
    ff, x, targets, il, tl = tail_case()
    B, T, D = ff.shape
    par = tail_parameters(D, 30)
    p, rng = 0.2, rng_of(41, 2)
    leaves = [t.clone().requires_grad_() for t in (ff, x, *par.values())]
    named = dict(zip(par, leaves[2:]))
    before = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        loss = tail_loss(leaves[0], leaves[1], named, rng, targets, il, tl, p)
        grads = torch.autograd.grad(loss, leaves)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = before

    ref = [t.detach().double().cpu().requires_grad_() for t in leaves]
    pad = R.padding(ff.shape, il)
    k0 = torch.where(R.keep_mask(ff.shape, 41, 2, 0, p) & ~pad, R.factor(p, 0.5), 0.0)
    k1 = torch.where(R.keep_mask(ff.shape, 41, 2, 1, p) & ~pad, R.factor(p, 1.0), 0.0)
    h = ref[1] + ref[0] * k0
    d = h - h.mean(-1, keepdim=True)
    y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS) * ref[2] + ref[3]
    logits = (y * k1) @ ref[4].t() + ref[5]
    rl, rg = R.ctc(logits.detach(), targets, il, tl, 0, False)
    share = 1.0 / (tl.double().cpu().clamp(min=1) * B)
    value = (rl * share).sum() + 1e-3 * h.square().mean()
    rgrads = torch.autograd.grad([logits, h], ref, [rg * share[:, None, None], 2e-3 * h.detach() / h.numel()])
    assert abs(float(loss.detach()) - float(value.detach())) < 1e-4 * abs(float(value.detach()))
    for name, got, want in zip(("ff", "x", *par), grads, rgrads):
        # fp32 throughout: chain, norm and products leave about (64 T + D) roundings of the largest entry
        bound = (64 * T + 4 * D + 300) * E * want.abs().max() * 8
        assert ((got.double().cpu() - want).abs() <= bound).all(), name


def test_training_step_captured():
    """The step in a CUDA graph: a replay gives the bits of the eager step, and new masks once the offset moved."""
    ff, x, targets, il, tl = tail_case(60)
    par = tail_parameters(ff.shape[-1], 30)
    rng = rng_of(5, 0)

    def step():
        leaves = [t.detach().requires_grad_() for t in (ff, x, *par.values())]
        loss = tail_loss(leaves[0], leaves[1], dict(zip(par, leaves[2:])), rng, targets, il, tl, 0.3)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        rng[1] += 1
    seen = []
    for i in range(3):
        rng.copy_(rng_of(5, i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert int(rng[1]) == i + 1
        rng.copy_(rng_of(5, i))
        want = step()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), i
        seen.append(got[0].item())
    assert len(set(seen)) == 3


def test_two_streams():
    """Calls on two streams at once keep to their own stream and buffers."""
    ff, x, targets, il, tl = tail_case(70)
    par = tail_parameters(ff.shape[-1], 30)
    logits = rand(1, (3, 24, 30), F32)
    w = par["w"]

    def both():
        return (*tr.layer_norm_backward(ff, x, w), tr.ctc_loss(logits, targets, il, tl))

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(5):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(both())
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_compiled_graph_sees_one_node_each():
    ff, x, targets, il, tl = tail_case(80)
    par = tail_parameters(ff.shape[-1], 30)
    rng = rng_of(6, 1)

    def f(a, r):
        y, h = tr.dropout_add_layer_norm(a, r, par["w"], par["b"], rng, 0.1, scale=0.5, lengths=il)
        return tr.layer_norm(tr.dropout_add(y, rng, 0.1, site=1), par["w"], par["b"]) + h

    got = torch.compile(f, fullgraph=True, backend="aot_eager")(ff, x)
    assert torch.equal(got, f(ff, x))


def test_registered_ops_are_consistent():
    """torch's own checks of the ops: schema, fake outputs, autograd registration."""
    ff, x, targets, il, tl = tail_case(90, B=3, T=8, D=24)
    w = rand(1, (24,), F32)
    rng = rng_of(2, 3)
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    check = torch.library.opcheck
    check(torch.ops.granite.layer_norm, (x.requires_grad_(), w, w, EPS, il), test_utils=tests)
    check(torch.ops.granite.layer_norm_backward, (ff, x.detach(), w, EPS, None), test_utils=tests)
    check(torch.ops.granite.dropout_add, (ff, None, rng, 0.1, 1.0, 0, il), test_utils=tests)
    check(torch.ops.granite.dropout_add_layer_norm, (ff, x.detach(), w, w, rng, 0.1, 1.0, 0, EPS, il), test_utils=tests)
    check(torch.ops.granite.dropout_add_layer_norm_backward,
          (ff, None, x.detach(), w, rng, 0.1, 1.0, 0, EPS, il), test_utils=tests)
    logits = rand(4, (3, 8, 30), F32)
    check(torch.ops.granite.ctc_loss, (logits.requires_grad_(), targets, il.clamp(max=8), tl, 0, False),
          test_utils=tests)


def test_functions_refuse_mismatched_tensors():
    x, w, rng = rand(1, (2, 3, 16), BF), torch.ones(16, device=DEV), rng_of()
    i = torch.ones(2, dtype=torch.int32, device=DEV)
    for call in (lambda: tr.layer_norm(x, w.half(), w.half()), lambda: tr.layer_norm(x, w, w.bfloat16()),
                 lambda: tr.layer_norm(x, w[:8], w), lambda: tr.layer_norm(x.double(), w, w),
                 lambda: tr.layer_norm(x, w, w, lengths=i[:1]), lambda: tr.layer_norm(x[0], w, w, lengths=i),
                 lambda: tr.layer_norm(x, w, w, lengths=i.float()), lambda: tr.layer_norm(x, w, w, lengths=i.cpu()),
                 lambda: tr.layer_norm(torch.zeros(1, 8200, device=DEV), torch.ones(8200, device=DEV),
                                       torch.ones(8200, device=DEV)),
                 lambda: tr.layer_norm_backward(x.float(), x, w), lambda: tr.layer_norm_backward(x[:1], x, w),
                 lambda: tr.dropout_add(x, rng, 1.5), lambda: tr.dropout_add(x, rng.int(), 0.1),
                 lambda: tr.dropout_add(x, rng, 0.1, site=-1), lambda: tr.dropout_add(x, rng, 0.1, residual=x[:1]),
                 lambda: tr.dropout_add(x, rng.cpu(), 0.1),
                 lambda: tr.ctc_loss(x, i[:, None], i, i, blank=16), lambda: tr.ctc_loss(x, i, i, i),
                 lambda: tr.ctc_loss(x[0], i[:, None], i, i), lambda: tr.ctc_loss(x, i[:, None].float(), i, i),
                 lambda: tr.ctc_loss(x, i[:, None], i[:1], i)):
        with pytest.raises(RuntimeError):
            call()


def test_functions_record_what_the_ops_record():
    """The functions' gradients are the dispatcher ops' bit for bit; dropout's gradient has a gradient of its own, those
    of the norms and of the loss refuse to be differentiated."""
    ff, x, targets, il, tl = tail_case(80)
    w, b, rng = rand(81, (x.shape[-1],), F32), rand(82, (x.shape[-1],), F32), rng_of(9, 2)
    logits = rand(83, (3, 24, 30), BF)
    o = torch.ops.granite
    pairs = [
        (lambda u: tr.layer_norm(u, w, b, EPS, il), lambda u: o.layer_norm(u, w, b, EPS, il), x),
        (lambda u: tr.dropout_add(u, rng, 0.2, x, 0.5, 3, il), lambda u: o.dropout_add(u, x, rng, 0.2, 0.5, 3, il), ff),
        (lambda u: tr.dropout_add_layer_norm(ff, u, w, b, rng, 0.2, 0.5, 1, EPS, il),
         lambda u: o.dropout_add_layer_norm(ff, u, w, b, rng, 0.2, 0.5, 1, EPS, il), x),
        (lambda u: tr.ctc_loss(u, targets, il, tl), lambda u: o.ctc_loss(u, targets, il, tl, 0, False)[0], logits),
    ]
    for function, op, at in pairs:
        got = []
        for f in (function, op):
            u = at.clone().requires_grad_()
            out = f(u)
            first = out[0] if isinstance(out, tuple) else out
            d = torch.linspace(-1.0, 1.0, first.numel(), device=DEV).reshape(first.shape).to(first.dtype)
            got.append((first.detach(), *torch.autograd.grad(first, u, d)))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    u = ff.clone().requires_grad_()
    d = x.clone().requires_grad_()
    du, = torch.autograd.grad(tr.dropout_add(u, rng, 0.2), u, d, create_graph=True)
    dd, = torch.autograd.grad(du, d, ff)
    assert torch.equal(dd, tr.dropout_add(ff, rng, 0.2))
    for function, _, at in (pairs[0], pairs[2], pairs[3]):
        u = at.clone().requires_grad_()
        out = function(u)
        first = out[0] if isinstance(out, tuple) else out
        du, = torch.autograd.grad(first.float().square().sum(), u, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(du.float().sum(), u)


# ---- the ends of the ranges ------------------------------------------------------------------------------------------
def test_ctc_wide_integers():
    """int64 labels and lengths that int32 does not hold are outside, not what their low halves say."""
    logits, targets, il, tl = ctc_case(200, 4, 12, 9, 4, F32)
    targets, il, tl = targets.long(), il.long(), tl.long()
    targets[1, 2] += 2 ** 32
    il[2] += 2 ** 32
    tl[3] -= 2 ** 33
    loss = tr.ctc_loss(logits, targets, il, tl)
    assert torch.isfinite(loss[0]) and torch.isnan(loss[1:]).all()
    x, w = rand(201, (2, 3, 16), BF), torch.ones(16, device=DEV)
    lengths = torch.tensor([2 ** 32 + 1, -2 ** 32 + 1], device=DEV)
    y = tr.layer_norm(x, w, w, EPS, lengths)
    assert torch.equal(y[0], tr.layer_norm(x, w, w, EPS, torch.tensor([3, 0], device=DEV))[0]) and not y[1].any()


def test_ctc_one_class():
    """A vocabulary of the blank alone: the loss is 0 without labels; as a label the blank needs one frame of its own."""
    logits, targets, il, tl = ctc_case(202, 3, 4, 1, 2, F32, ([4, 4, 1], [0, 2, 2]), labels=[[0, 0]] * 3)
    check_ctc(logits, targets, il, tl)


def test_ctc_more_utterances_than_a_grid_holds():
    B = 65535 + 9
    logits, targets, il, tl = ctc_case(203, 7, 3, 5, 2, BF, ([3, 2, 1, 3, 0, 3, 2], [2, 1, 1, 0, 0, 2, 2]))
    base, grad = check_ctc(logits, targets, il, tl, dloss=torch.ones(7, device=DEV))
    many = [t.repeat(-(-B // 7), *[1] * (t.dim() - 1))[:B] for t in (logits, targets, il, tl)]
    x = many[0].requires_grad_()
    loss = tr.ctc_loss(x, *many[1:])
    got, = torch.autograd.grad(loss, x, torch.ones(B, device=DEV))
    # rows of five bf16 logits begin at every alignment, and a row's sum at its first 16-byte boundary: its order, so not
    # its bits, is the utterance's own.  Both sides lie within check_ctc's bounds (T = 3, V = 5) of the same number.
    want, wgrad = base.repeat(-(-B // 7))[:B].detach().double(), grad.repeat(-(-B // 7), 1, 1)[:B].double()
    per_frame = (5 / 256 + 100) * E
    fin = torch.isfinite(want)
    assert torch.equal(fin, torch.isfinite(loss)) and torch.equal(want == math.inf, loss == math.inf)
    assert ((loss.double() - want).abs()[fin] <= (2 * (3 * per_frame + E * want.abs() * (1 + E) + 1e-6))[fin]).all()
    ok = ~torch.isnan(wgrad)
    assert torch.equal(ok, ~torch.isnan(got))
    bound = 2 * (rounded(BF, wgrad) * (1 + 2 ** -8) + per_frame + (3 * 64 + 164) * E)
    assert ((got.double() - wgrad).abs()[ok] <= bound[ok]).all()


def test_ctc_longest_chain():
    check_ctc(*ctc_case(204, 2, tr.MAX_CTC_FRAMES, 5, 20, F32, ([tr.MAX_CTC_FRAMES, 9001], [20, 13])))


def test_elements_past_32_bits():
    """More elements than an int counts: the last rows and the last utterance as they are alone."""
    M, D = 2 ** 21 + 104, 1024
    g = torch.Generator(device=DEV).manual_seed(205)
    x = torch.randn(M, D, device=DEV, generator=g, dtype=BF)
    res = torch.randn(M, D, device=DEV, generator=g, dtype=BF)
    w, b, rng = rand(206, (D,), F32, 0.1, 1.0), rand(207, (D,), F32, 0.1), rng_of(3, 4)
    last = slice(M - 40, M)
    y, h = tr.dropout_add_layer_norm(x, res, w, b, rng, 0.0)
    y1, h1 = tr.dropout_add_layer_norm(x[last], res[last], w, b, rng, 0.0)
    assert torch.equal(y[last], y1) and torch.equal(h[last], h1)
    del y, h
    dx, dres, _, _ = tr.dropout_add_layer_norm_backward(x, res, x, w, rng, 0.0)
    dx1, dres1, _, _ = tr.dropout_add_layer_norm_backward(x[last], res[last], x[last], w, rng, 0.0)
    assert torch.equal(dx[last], dx1) and torch.equal(dres[last], dres1)
    del dx, dres
    out = tr.dropout_add(x, rng, 0.25, res)
    kept = out[M - 2:].double().cpu() != res[M - 2:].double().cpu()
    groups = np.arange((M - 2) * (D // 8), M * (D // 8), dtype=np.uint64)
    r = R.philox((groups & np.uint64(0xFFFFFFFF), groups >> np.uint64(32), np.full(groups.shape, 4, np.uint64),
                  np.zeros(groups.shape, np.uint64)), (3, 0))
    halves = np.stack([(v >> np.uint64(16 * i)) & np.uint64(0xFFFF) for v in r for i in (0, 1)], -1).reshape(2, D)
    keep = torch.from_numpy(halves >= 16384)
    # a kept element is the sum rounded, the residual itself only where x is lost beside it
    assert not (kept & ~keep).any() and (keep & ~kept).sum() < 16
    del x, res, out
    B, T, V = 2, 10800, 100352
    logits = torch.randn(B, T, V, device=DEV, generator=g, dtype=BF).requires_grad_()
    targets = torch.randint(1, V, (B, 30), device=DEV, generator=g, dtype=torch.int32)
    il, tl = lens_of([T, T - 7]), lens_of([30, 29])
    loss = tr.ctc_loss(logits, targets, il, tl)
    grad, = torch.autograd.grad(loss.sum(), logits)
    alone = logits[1:].detach().requires_grad_()
    loss1 = tr.ctc_loss(alone, targets[1:], il[1:], tl[1:])
    grad1, = torch.autograd.grad(loss1.sum(), alone)
    assert torch.equal(loss[1:], loss1) and torch.equal(grad[1:], grad1)
