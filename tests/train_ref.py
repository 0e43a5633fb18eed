"""Plain 64-bit restatements of the fine-tuning operators (numpy and torch on the CPU), for the tests."""
from __future__ import annotations

import math

import numpy as np
import torch


# ---- Philox4x32-10 ---------------------------------------------------------------------------------------------------
def philox(counter, key):
    """counter: four uint32 arrays, key: two ints -> four uint32 arrays."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(key[0]), int(key[1])]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a = c[0] * np.uint64(0xD2511F53)
        b = c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]),
             a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [v.astype(np.uint32) for v in c]


def keep_mask(shape, seed, offset, site, p):
    """Truth values of the kept elements of rows [..., D]."""
    D = shape[-1]
    rows = int(np.prod(shape[:-1], dtype=np.int64))
    G = -(-D // 8)
    g = np.arange(rows * G, dtype=np.uint64)
    seed &= 2 ** 64 - 1
    w = philox([g & np.uint64(0xFFFFFFFF), g >> np.uint64(32), np.full_like(g, offset & 0xFFFFFFFF),
                np.full_like(g, site)], (seed & 0xFFFFFFFF, seed >> 32))
    u = np.stack([h for v in w for h in (v & np.uint32(0xFFFF), v >> np.uint32(16))], 1)
    keep = u >= round(65536 * p)
    return torch.from_numpy(keep.reshape(rows, G * 8)[:, :D].reshape(shape))


def factor(p, scale):
    kept = 65536 - round(65536 * p)
    return scale * 65536 / kept if kept else 0.0


# ---- rows ------------------------------------------------------------------------------------------------------------
def padding(shape, lengths):
    """Truth values [B, T, 1] (or all false) of the padding frames."""
    if lengths is None:
        return torch.zeros([1] * len(shape), dtype=torch.bool)
    return (torch.arange(shape[1])[None, :] >= torch.as_tensor(lengths).cpu()[:, None])[:, :, None]


def layer_norm(x, w, b, eps, lengths=None):
    pad = padding(x.shape, lengths)
    x = x.double().cpu().masked_fill(pad, 0.0)
    d = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    return (d * r * w.double().cpu() + b.double().cpu()).masked_fill(pad, 0.0), r


def layer_norm_backward(dy, x, w, eps, lengths=None):
    """dx, dw, db and, for the bounds, the reciprocal deviation and the normed x."""
    pad = padding(x.shape, lengths)
    x = x.double().cpu().masked_fill(pad, 0.0)
    dy = dy.double().cpu().masked_fill(pad, 0.0)
    d = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    xh = d * r
    g = dy * w.double().cpu()
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    rows = tuple(range(x.dim() - 1))
    return dx.masked_fill(pad, 0.0), (dy * xh).sum(rows), dy.sum(rows), r, xh


def dropout_add(x, residual, seed, offset, site, p, scale, lengths=None):
    keep = keep_mask(x.shape, seed, offset, site, p) & ~padding(x.shape, lengths)
    h = torch.where(keep, x.double().cpu() * factor(p, scale), 0.0)
    return h if residual is None else h + residual.double().cpu()


# ---- CTC -------------------------------------------------------------------------------------------------------------
def _logsum(values):
    top = max(values)
    if top == -math.inf:
        return top
    return top + math.log(sum(math.exp(v - top) for v in values))


def ctc_one(logits, target, blank):
    """(loss, gradient) of one utterance: logits [n, V] float64, target a list of labels.  The gradient of an utterance
    without an alignment is None."""
    n, V = logits.shape
    x = logits.double().numpy()
    states = [blank]
    for v in target:
        states += [int(v), blank]
    L = len(states)
    if n == 0:
        return (0.0 if L == 1 else math.inf), np.zeros((0, V))
    top = x.max(1, keepdims=True)
    logp = x - top - np.log(np.exp(x - top).sum(1, keepdims=True))
    lab = np.asarray(states)
    em = logp[:, lab]
    skip = np.zeros(L, dtype=bool)
    skip[2:] = (lab[2:] != blank) & (lab[2:] != lab[:-2])

    def shifted(v, by, keep):
        """v moved up (by > 0) or down the states, -inf coming in; only where `keep`."""
        out = np.full(L, -math.inf)
        if by > 0:
            out[by:] = v[:-by] if L > by else []
        else:
            out[:by] = v[-by:] if L > -by else []
        return np.where(keep, out, -math.inf)

    alpha = np.full((n, L), -math.inf)
    alpha[0, :2] = em[0, :2]
    for t in range(1, n):
        a = alpha[t - 1]
        alpha[t] = em[t] + np.logaddexp(np.logaddexp(a, shifted(a, 1, True)), shifted(a, 2, skip))
    logz = _logsum([alpha[-1, -1]] + ([alpha[-1, -2]] if L > 1 else []))
    if logz == -math.inf:
        return math.inf, None
    beta = np.full((n, L), -math.inf)
    beta[-1, -2:] = 0.0
    jump = np.append(skip[2:], [False] * min(2, L))[:L]
    for t in range(n - 2, -1, -1):
        q = beta[t + 1] + em[t + 1]
        beta[t] = np.logaddexp(np.logaddexp(q, shifted(q, -1, True)), shifted(q, -2, jump))
    gamma = np.exp(alpha + beta - logz)
    grad = np.exp(logp)
    for s in range(L):
        grad[:, states[s]] -= gamma[:, s]
    return -logz, grad


def ctc(logits, targets, input_lengths, target_lengths, blank, zero_infinity):
    """(loss [B], gradient [B, T, V] for dloss = 1), float64."""
    B, T, V = logits.shape
    x = logits.double().cpu()
    losses, grads = torch.zeros(B, dtype=torch.float64), torch.zeros((B, T, V), dtype=torch.float64)
    for b in range(B):
        n, s = int(input_lengths[b]), int(target_lengths[b])
        loss, grad = ctc_one(x[b, :n], [int(v) for v in targets[b, :s]], blank)
        if grad is None:
            losses[b] = 0.0 if zero_infinity else loss
            grads[b, :n] = 0.0 if zero_infinity else math.nan
        else:
            losses[b] = loss if loss < math.inf or not zero_infinity else 0.0
            grads[b, :n] = torch.from_numpy(grad)
    return losses, grads
