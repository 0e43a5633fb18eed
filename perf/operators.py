"""The operators for fine-tuning the encoder, as they are measured: layer norm and its backward pass, dropout with a
residual (the mask regenerated from a counter), the residual step fused with the layer norm after it, and the CTC loss
with its gradient.

A case is one pass through one operator: ``run`` in plain torch operations where ``own`` is false, through the
package's own calls where it is true.  ``exact`` evaluates the same definitions in 64 bits, separately written.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


# ---- the cases ------------------------------------------------------------------------------------------------------
# Row operators: B utterances of T frames of D channels; `fill` < 1 pads: the lengths run evenly from fill * T to T, and
# fill = 1 passes no lengths.  `wtype` is the type of the layer norm's weight and bias (fp32 master weights, or the
# activations' own type).
def listed():
    def row(name, op, B, T, D, dtype="bf16", wtype="fp32", fill=1.0, p=0.0, scale=1.0, residual=False):
        return dict(name=name, op=op, B=B, T=T, D=D, dtype=dtype, wtype=wtype, fill=fill, p=p, scale=scale,
                    residual=residual)

    def ctc(name, op, B, T, V, S, dtype, fill=1.0):
        return dict(name=name, op=op, B=B, T=T, V=V, S=S, dtype=dtype, fill=fill)

    return [
        # one short utterance through a norm with fp32 master weights: launch latency
        row("ln_fwd_short", "ln_fwd", 1, 37, 1024),
        # the padded execution batch of 48 utterances at the encoder's width
        row("ln_fwd_batch", "ln_fwd", 48, 1536, 1024, fill=0.25),
        # its gradient, the weight's and bias' reduced over all valid frames
        row("ln_bwd_batch", "ln_bwd", 48, 1536, 1024, fill=0.25),
        # a width off the vector grid, in fp16 throughout
        row("ln_bwd_odd", "ln_bwd", 48, 237, 1001, dtype="fp16", wtype="fp16"),
        # full-precision training at the convolution module's inner width
        row("ln_bwd_fp32", "ln_bwd", 48, 261, 2048, dtype="fp32"),
        # the half-step residual of one short utterance
        row("drop_fwd_short", "drop_fwd", 1, 37, 1024, p=0.1, scale=0.5, residual=True),
        # dropout behind the feed-forward activation (4 x the width), backward
        row("drop_bwd_ff", "drop_bwd", 48, 1024, 4096, p=0.1),
        # the tail of a block: half-step residual of the second feed-forward, then the post norm
        row("dropln_fwd_tail", "dropln_fwd", 48, 1024, 1024, p=0.1, scale=0.5, residual=True),
        # its backward pass on the padded batch
        row("dropln_bwd_tail", "dropln_bwd", 48, 1536, 1024, p=0.1, scale=0.5, residual=True, fill=0.25),
        # validation loss of one utterance at the character head
        ctc("ctc_loss_short", "ctc_fwd", 1, 237, 348, 40, "fp32"),
        # a training step's loss and gradient at the character head, the padded batch
        ctc("ctc_char_batch", "ctc_train", 48, 1536, 348, 300, "bf16", fill=0.25),
        # the BPE head's loss and gradient: pooled frames over the whole vocabulary
        ctc("ctc_bpe", "ctc_train", 8, 384, 100352, 96, "bf16", fill=0.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "drop_fwd", "drop_bwd", "dropln_fwd", "dropln_bwd", "ctc_fwd", "ctc_train"])
    B = _log_int(rng, 1, 48)
    T = _log_int(rng, 1, 1536)
    fill = rng.choice([1.0, rng.uniform(0.05, 1.0)])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if op.startswith("ctc"):
        V = _log_int(rng, 4, 100352)
        B = max(1, min(B, 300_000_000 // (T * V)))
        S = rng.randint(0, max(1, min(300, T // 2)))
        return dict(op=op, B=B, T=T, V=V, S=S, dtype=dtype, fill=fill)
    D = _log_int(rng, 16, 4096)
    if rng.random() < 0.5:
        D = (D + 7) // 8 * 8
    limit = 75_000_000 // (2 if dtype == "fp32" else 1)
    B = max(1, min(B, limit // (T * D)))
    return dict(op=op, B=B, T=T, D=D, dtype=dtype, wtype=rng.choice(["fp32", dtype]), fill=fill,
                p=0.0 if op.startswith("ln") else rng.choice([0.05, 0.1, 0.3, rng.uniform(0.01, 0.9)]),
                scale=1.0 if op.startswith("ln") else rng.choice([1.0, 0.5]),
                residual=op.startswith("dropln") or (op == "drop_fwd" and rng.random() < 0.7))


def _lengths(B, T, fill):
    """B lengths running evenly from fill * T to T (the longest is T)."""
    lo = max(1, math.ceil(fill * T))
    return [T - (T - lo) * i // max(1, B - 1) for i in range(B)]


def _ctc_sizes(case):
    """(input length, target length) of every utterance: targets in the proportion S / T of the frames."""
    T, S = case["T"], case["S"]
    return [(n, S * n // T) for n in _lengths(case["B"], T, case["fill"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)
    dt = DTYPES[case["dtype"]]
    B, T = case["B"], case["T"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    st = dict(case=case)
    order = host.permutation(B)
    if case["op"].startswith("ctc"):
        V, S = case["V"], case["S"]
        sizes = [_ctc_sizes(case)[i] for i in order]
        blank = V - 1 if V > 1000 else 0         # the BPE head's blank lies inside its vocabulary, the character head's is 0
        targets = host.integers(0, V - 1, (B, S))
        targets[targets >= blank] += 1
        # logits of a model part way through training: blank likely, the labels peaked along some alignment
        logits = torch.randn((B, T, V), generator=g, device="cuda").mul_(1.5)
        logits[:, :, blank] += 5.0
        for b, (n, s) in enumerate(sizes):
            if s:
                at = np.sort(host.choice(n, s, replace=False))
                t = torch.from_numpy(at).cuda()
                v = torch.from_numpy(targets[b, :s]).cuda()
                logits[b, t, blank] -= 4.0
                logits[b, t, v] += 6.0
        st["logits"] = logits.to(dt)
        st["targets"] = torch.from_numpy(targets.astype(np.int32)).cuda()
        st["in_len"] = torch.tensor([n for n, _ in sizes], dtype=torch.int32, device="cuda")
        st["tg_len"] = torch.tensor([s for _, s in sizes], dtype=torch.int32, device="cuda")
        st["blank"] = blank
        # the gradient that a mean over the batch, each utterance by its number of labels, sends back
        st["dloss"] = torch.tensor([1.0 / (B * max(1, s)) for _, s in sizes], device="cuda")
        return st
    D = case["D"]
    wt = DTYPES[case["wtype"]]
    st["lengths"] = None
    if case["fill"] < 1.0:
        n = np.asarray(_lengths(B, T, case["fill"]), dtype=np.int32)[order]
        st["lengths"] = torch.from_numpy(n).cuda()
    st["rng"] = torch.tensor([int(host.integers(0, 2 ** 62)), int(host.integers(0, 2 ** 31))], device="cuda")
    st["site"] = int(host.integers(0, 64))
    st["weight"] = (1.0 + 0.1 * normal(D)).to(wt)
    st["bias"] = (0.1 * normal(D)).to(wt)
    channel = torch.exp(0.5 * normal(D))         # a residual stream: channels of unlike spread and offset
    offset = normal(D)
    if case["op"] in ("ln_fwd", "ln_bwd"):
        st["x"] = (normal(B, T, D) * channel + offset).to(dt)
    elif case["op"] in ("drop_fwd", "dropln_fwd"):
        st["x"] = normal(B, T, D).to(dt)
        st["residual"] = (normal(B, T, D) * channel + offset).to(dt) if case["residual"] else None
    if case["op"] == "dropln_bwd":
        st["h"] = (normal(B, T, D) * channel + offset).to(dt)
        st["dh"] = (0.1 * normal(B, T, D)).to(dt)
    if case["op"].endswith("bwd"):
        st["dout"] = (0.1 * normal(B, T, D)).to(dt)
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _training():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "granite-speech-4.1-2b-nar-turbo_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from granite_conv_b200 import training
    return training


def _run_own(st):
    tr = _training()
    c = st["case"]
    op = c["op"]
    if op == "ln_fwd":
        return tr.layer_norm(st["x"], st["weight"], st["bias"], EPS, lengths=st["lengths"])
    if op == "ln_bwd":
        return tr.layer_norm_backward(st["dout"], st["x"], st["weight"], EPS, lengths=st["lengths"])
    if op == "drop_fwd":
        return tr.dropout_add(st["x"], st["rng"], c["p"], residual=st["residual"], scale=c["scale"], site=st["site"],
                              lengths=st["lengths"])
    if op == "drop_bwd":
        return tr.dropout_add_backward(st["dout"], st["rng"], c["p"], scale=c["scale"], site=st["site"],
                                       lengths=st["lengths"])
    if op == "dropln_fwd":
        return tr.dropout_add_layer_norm(st["x"], st["residual"], st["weight"], st["bias"], st["rng"], c["p"],
                                         scale=c["scale"], site=st["site"], eps=EPS, lengths=st["lengths"])
    if op == "dropln_bwd":
        return tr.dropout_add_layer_norm_backward(st["dout"], st["dh"], st["h"], st["weight"], st["rng"], c["p"],
                                                  scale=c["scale"], site=st["site"], eps=EPS, lengths=st["lengths"])
    if op == "ctc_fwd":
        return tr.ctc_loss(st["logits"], st["targets"], st["in_len"], st["tg_len"], blank=st["blank"],
                           zero_infinity=True)
    logits = st["logits"].detach().requires_grad_()
    loss = tr.ctc_loss(logits, st["targets"], st["in_len"], st["tg_len"], blank=st["blank"], zero_infinity=True)
    return loss.detach(), torch.autograd.grad(loss, logits, st["dloss"])[0]


def _valid(st, like):
    """[B, T, 1] truth values of the frames inside their utterance, or None."""
    if st["lengths"] is None:
        return None
    return (torch.arange(like.shape[1], device=like.device)[None, :] < st["lengths"][:, None])[:, :, None]


def _where(valid, a, b):
    return a if valid is None else torch.where(valid, a, b)


def _philox(rng, site, groups):
    """Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011) for the counters
    (group, group >> 32, offset, site) and the 64-bit seed as key: int64 [groups, 8], eight 16-bit numbers each."""
    mask = 0xFFFFFFFF
    i = torch.arange(groups, dtype=torch.int64, device=rng.device)
    c0, c1 = i & mask, i >> 32
    c2 = (rng[1] & mask).expand_as(i)
    c3 = torch.full_like(i, site)
    k0, k1 = rng[0] & mask, (rng[0] >> 32) & mask
    for _ in range(10):
        a = c0 * 0xD2511F53              # the low 64 bits of a 32 x 32 bit product are exact in wrapping int64
        b = c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & mask) ^ c1 ^ k0, b & mask, ((a >> 32) & mask) ^ c3 ^ k1, a & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], 1)


def _keep(st, shape):
    """Truth values of the kept elements; groups of eight columns, every row starting a new group."""
    B, T, D = shape
    per_row = (D + 7) // 8
    u = _philox(st["rng"], st["site"], B * T * per_row)
    return (u >= round(65536 * st["case"]["p"])).view(B, T, per_row * 8)[:, :, :D]


def _factor(c):
    """What a kept element is multiplied with: scale over the probability of being kept."""
    kept = 65536 - round(65536 * c["p"])
    return c["scale"] * 65536 / kept if kept else 0.0


def _norm(x):
    D = x.shape[-1]
    mean = x.sum(-1, keepdim=True) / D
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).sum(-1, keepdim=True) / D + EPS)
    return d * rstd, rstd


def _norm_backward(dy, x, weight, valid):
    D = x.shape[-1]
    if valid is not None:
        dy, x = torch.where(valid, dy, 0.0), torch.where(valid, x, 0.0)
    xh, rstd = _norm(x)
    g = dy * weight
    dx = rstd * (g - g.sum(-1, keepdim=True) / D - xh * ((g * xh).sum(-1, keepdim=True) / D))
    dw = (dy * xh).sum((0, 1), dtype=torch.float64)
    db = dy.sum((0, 1), dtype=torch.float64)
    return _where(valid, dx, torch.zeros_like(dx)), dw, db


def _run_plain(st):
    c = st["case"]
    op = c["op"]
    if op.startswith("ctc"):
        return _plain_ctc(st, gradient=op == "ctc_train")
    dt = DTYPES[c["dtype"]]
    w, b = st["weight"].float(), st["bias"].float()
    if op == "ln_fwd":
        valid = _valid(st, st["x"])
        y = _norm(st["x"].float())[0] * w + b
        return _where(valid, y, torch.zeros_like(y)).to(dt)
    if op == "ln_bwd":
        dx, dw, db = _norm_backward(st["dout"].float(), st["x"].float(), w, _valid(st, st["x"]))
        return dx.to(dt), dw.to(st["weight"].dtype), db.to(st["weight"].dtype)
    if op in ("drop_fwd", "dropln_fwd"):
        x = st["x"].float()
        valid = _valid(st, x)
        kept = _keep(st, x.shape)
        if valid is not None:
            kept = kept & valid
        h = torch.where(kept, x * _factor(c), 0.0)
        if st["residual"] is not None:
            h = h + st["residual"].float()
        if op == "drop_fwd":
            return h.to(dt)
        y = _norm(h)[0] * w + b
        return _where(valid, y, torch.zeros_like(y)).to(dt), h.to(dt)
    g = st["dout"].float()
    valid = _valid(st, g)
    kept = _keep(st, g.shape)
    if valid is not None:
        kept = kept & valid
    if op == "drop_bwd":
        return torch.where(kept, g * _factor(c), 0.0).to(dt)
    dh, dw, db = _norm_backward(g, st["h"].float(), w, valid)
    dh = dh + st["dh"].float()
    return (torch.where(kept, dh * _factor(c), 0.0).to(dt), dh.to(dt), dw.to(st["weight"].dtype),
            db.to(st["weight"].dtype))


def _add_logs(*parts):
    top = parts[0]
    for a in parts[1:]:
        top = torch.maximum(top, a)
    base = torch.where(top == -math.inf, 0.0, top)
    total = torch.exp(parts[0] - base)
    for a in parts[1:]:
        total = total + torch.exp(a - base)
    return base + torch.log(total)


def _states(st):
    """Labels of the 2 S + 1 states (int64 [B, 2 S + 1], blank at the even ones) and where a state may be entered from
    two states before it."""
    targets = st["targets"].long()
    B, S = targets.shape
    labels = torch.full((B, 2 * S + 1), st["blank"], dtype=torch.int64, device=targets.device)
    labels[:, 1::2] = targets
    skip = torch.zeros_like(labels, dtype=torch.bool)
    skip[:, 3::2] = targets[:, 1:] != targets[:, :-1]
    return labels, skip


def _plain_ctc(st, gradient):
    x = st["logits"].float()
    B, T, V = x.shape
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    labels, skip = _states(st)
    L = labels.shape[1]
    # the sums over paths are long: the chain of T steps is kept in 64 bits, on the logarithms
    index = labels[:, None, :].expand(B, T, L)
    lp = x.gather(2, index).double() - top.double() - torch.log(total.double())
    n, s = st["in_len"].long(), st["tg_len"].long()
    none = torch.full((B, L), -math.inf, dtype=torch.float64, device=x.device)
    pos = torch.arange(L, device=x.device)[None, :]
    ends = (pos == 2 * s[:, None]) | (pos == 2 * s[:, None] - 1)
    alphas = []
    a = torch.where(pos <= 1, lp[:, 0], none)
    alphas.append(a)
    for t in range(1, T):
        one = torch.cat([none[:, :1], a[:, :-1]], 1)
        two = torch.where(skip, torch.cat([none[:, :2], a[:, :-2]], 1)[:, :L], none)
        a = _add_logs(a, one, two) + lp[:, t]
        alphas.append(a)
    alpha = torch.stack(alphas, 1)
    last = alpha[torch.arange(B, device=x.device), n - 1]
    logz = _add_logs(*torch.where(ends, last, none).unbind(1))
    feasible = logz > -math.inf
    loss = torch.where(feasible, -logz, 0.0).float()
    if not gradient:
        return loss
    jump = torch.cat([skip[:, 2:], torch.zeros_like(skip[:, :2])], 1)[:, :L]
    start = torch.where(ends, 0.0, none)
    betas = [None] * T
    nxt = none
    for t in range(T - 1, -1, -1):
        if t + 1 < T:
            q = nxt + lp[:, t + 1]
            one = torch.cat([q[:, 1:], none[:, :1]], 1)
            two = torch.where(jump, torch.cat([q[:, 2:], none[:, :2]], 1)[:, :L], none)
            nxt = _add_logs(q, one, two)
        nxt = torch.where((n == t + 1)[:, None], start, nxt)
        betas[t] = nxt
    inside = (torch.arange(T, device=x.device)[None, :] < n[:, None]) & feasible[:, None]
    gamma = torch.exp(alpha + torch.stack(betas, 1) - torch.where(feasible, logz, 0.0)[:, None, None]).float()
    # states behind an utterance's own last one take no part
    gamma = torch.where(pos[:, None, :] <= 2 * s[:, None, None], gamma, 0.0)
    grad = e / total
    grad.scatter_add_(2, index, -gamma)
    grad = torch.where(inside[:, :, None], grad * st["dloss"][:, None, None], 0.0)
    return loss, grad.to(st["logits"].dtype)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _mul32(a, m):
    """High and low word of a 32 x 32 bit product from 16-bit parts (int64 tensors, no wrapping)."""
    al, ah, ml, mh = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    mid = ah * ml + ((al * ml) >> 16)
    mid2 = al * mh + (mid & 0xFFFF)
    return ah * mh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((al * ml) & 0xFFFF)


def _exact_keep(st, rows, D):
    seed, offset = (int(v) for v in st["rng"].tolist())
    G = -(-D // 8)
    ctr = torch.arange(rows * G, dtype=torch.int64, device="cuda")
    word = [ctr % 2 ** 32, ctr // 2 ** 32, torch.zeros_like(ctr) + offset % 2 ** 32, torch.zeros_like(ctr) + st["site"]]
    key = [seed % 2 ** 32, (seed >> 32) % 2 ** 32]
    for r in range(10):
        h0, l0 = _mul32(word[0], 0xD2511F53)
        h1, l1 = _mul32(word[2], 0xCD9E8D57)
        word = [h1 ^ word[1] ^ ((key[0] + r * 0x9E3779B9) % 2 ** 32), l1,
                h0 ^ word[3] ^ ((key[1] + r * 0xBB67AE85) % 2 ** 32), l0]
    limit = round(65536 * st["case"]["p"])
    keep = torch.empty((rows * G, 8), dtype=torch.bool, device="cuda")
    for j in range(8):
        keep[:, j] = ((word[j // 2] >> (16 * (j % 2))) % 65536) >= limit
    return keep.view(rows, G * 8)[:, :D]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op.startswith("ctc"):
        return _exact_ctc(st, op == "ctc_train")
    B, T, D = case["B"], case["T"], case["D"]
    rows = B * T
    inside = torch.ones(rows, dtype=torch.bool, device="cuda")
    if st["lengths"] is not None:
        frame = torch.arange(rows, device="cuda")
        inside = frame % T < st["lengths"].long()[frame // T]
    inside = inside[:, None]

    def rows64(name):
        return None if st.get(name) is None else st[name].double().view(rows, D)

    w, b = st["weight"].double(), st["bias"].double()
    keep = 1.0 - round(65536 * case["p"]) / 65536
    k = case["scale"] / keep if keep > 0 else 0.0

    def drop(v):
        return (v * k).masked_fill_(~(_exact_keep(st, rows, D) & inside), 0.0)

    def centred(v):
        u = v - v.mean(1, keepdim=True)
        sd = (u.square().mean(1, keepdim=True) + EPS).sqrt()
        return u / sd, sd

    def norm_gradient(dy, v):
        dy = dy.masked_fill(~inside, 0.0)
        z, sd = centred(v.masked_fill(~inside, 0.0))
        q = dy * w
        dx = (q - q.mean(1, keepdim=True) - z * (q * z).mean(1, keepdim=True)) / sd
        return dx.masked_fill_(~inside, 0.0), (dy * z).sum(0), dy.sum(0)

    shape = (B, T, D)
    if op == "ln_fwd":
        y = torch.addcmul(b, centred(rows64("x"))[0], w)
        return y.masked_fill_(~inside, 0.0).view(shape)
    if op == "ln_bwd":
        dx, dw, db = norm_gradient(rows64("dout"), rows64("x"))
        return dx.view(shape), dw, db
    if op == "drop_bwd":
        return drop(rows64("dout")).view(shape)
    if op == "dropln_bwd":
        dx, dw, db = norm_gradient(rows64("dout"), rows64("h"))
        total = dx + rows64("dh")
        return drop(total).view(shape), total.view(shape), dw, db
    h = drop(rows64("x"))
    if st["residual"] is not None:
        h += rows64("residual")
    if op == "drop_fwd":
        return h.view(shape)
    y = torch.addcmul(b, centred(h)[0], w).masked_fill_(~inside, 0.0)
    return y.view(shape), h.view(shape)


def _walk(lp, may_skip):
    """Log sums over the paths into every state, emissions included: lp [B, T, L], the paths beginning in the first two
    states."""
    B, T, L = lp.shape
    out = torch.full_like(lp, -math.inf)
    out[:, 0, :2] = lp[:, 0, :2]
    pad = torch.full((B, L + 2), -math.inf, dtype=lp.dtype, device=lp.device)
    for t in range(1, T):
        pad[:, 2:] = out[:, t - 1]
        three = torch.stack([pad[:, 2:], pad[:, 1:-1], pad[:, :-2].masked_fill(~may_skip, -math.inf)])
        out[:, t] = torch.logsumexp(three, 0) + lp[:, t]
    return out


def _exact_ctc(st, gradient):
    x = st["logits"].double()
    B, T, V = x.shape
    norm = torch.logsumexp(x, -1)
    labels, skip = _states(st)
    L = labels.shape[1]
    lp = x.gather(2, labels[:, None].expand(B, T, L)) - norm[:, :, None]
    n, s = st["in_len"].long(), st["tg_len"].long()
    fwd = _walk(lp, skip)
    bi = torch.arange(B, device=x.device)
    tail = fwd[bi, n - 1]
    before = torch.where(s > 0, tail[bi, (2 * s - 1).clamp(min=0)], -math.inf)
    logz = torch.logaddexp(tail[bi, 2 * s], before)
    ok = torch.isfinite(logz)
    loss = torch.where(ok, -logz, 0.0)
    if not gradient:
        return loss
    # the same walk from the end: frames and states of every utterance in reverse order
    t_rev = (n[:, None] - 1 - torch.arange(T, device=x.device)[None, :]) % T
    s_rev = (2 * s[:, None] - torch.arange(L, device=x.device)[None, :]) % L
    lp_rev = lp[bi[:, None, None], t_rev[:, :, None], s_rev[:, None, :]]
    lab_rev = labels.gather(1, s_rev)
    skip_rev = torch.zeros_like(skip)
    skip_rev[:, 2:] = (lab_rev[:, 2:] != st["blank"]) & (lab_rev[:, 2:] != lab_rev[:, :-2])
    # a reversed order's states behind the last one wrap round: shut them
    lp_rev = lp_rev.masked_fill((torch.arange(L, device=x.device)[None, :] > 2 * s[:, None])[:, None, :], -math.inf)
    bwd = _walk(lp_rev, skip_rev)[bi[:, None, None], t_rev[:, :, None], s_rev[:, None, :]]
    inside = torch.arange(T, device=x.device)[None, :] < n[:, None]
    own_state = torch.arange(L, device=x.device)[None, :] <= 2 * s[:, None]
    use = inside[:, :, None] & own_state[:, None, :] & ok[:, None, None] & torch.isfinite(lp)
    gamma = torch.where(use, torch.exp(fwd + bwd - lp - logz[:, None, None]), 0.0)
    grad = torch.exp_(x.sub_(norm[:, :, None]))
    grad.scatter_add_(2, labels[:, None].expand(B, T, L), -gamma)
    grad *= st["dloss"].double()[:, None, None]
    grad.masked_fill_(~(inside & ok[:, None])[:, :, None], 0.0)
    return loss, grad


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    op, B, T = case["op"], case["B"], case["T"]
    if op.startswith("ctc"):
        V = case["V"]
        sizes = _ctc_sizes(case)
        frames = sum(n for n, _ in sizes)
        cells = sum(n * (2 * s + 1) for n, s in sizes)
        small = B * case["S"] * 4 + 12 * B
        if op == "ctc_fwd":
            return {"bytes": frames * V * size + small, "flops": 4 * frames * V + 6 * cells}
        return {"bytes": frames * V * size + B * T * V * size + small + 4 * B, "flops": 7 * frames * V + 16 * cells}
    D = case["D"]
    wsize = 4 if case["wtype"] == "fp32" else 2
    every = B * T * D
    n = D * (sum(_lengths(B, T, case["fill"])) if case["fill"] < 1.0 else B * T)
    rand = 10 * n                       # ten rounds of the generator over eight elements, about ten operations each
    if op == "ln_fwd":
        return {"bytes": (n + every) * size + 2 * D * wsize, "flops": 8 * n}
    if op == "ln_bwd":
        return {"bytes": (2 * n + every) * size + 3 * D * wsize, "flops": 18 * n}
    if op == "drop_fwd":
        reads = n + (every if case["residual"] else 0)
        return {"bytes": (reads + every) * size, "flops": 2 * n + rand}
    if op == "drop_bwd":
        return {"bytes": (n + every) * size, "flops": n + rand}
    if op == "dropln_fwd":
        return {"bytes": (n + 3 * every) * size + 2 * D * wsize, "flops": 10 * n + rand}
    return {"bytes": (2 * n + 3 * every) * size + 3 * D * wsize, "flops": 20 * n + rand}
