"""Operators for fine-tuning the encoder: the layer norm with its backward pass, dropout with a residual (the mask
regenerated from a counter, never stored), the residual step fused with the norm behind it (a Conformer block's tail,
``models/granite_speech_nar/conformer.py:208-209``), and the CTC loss of the heads (``:240-252``) with its gradient.

The functions here take plain tensors and are differentiable (the ``*_backward`` ones, for gradients by hand, record
nothing); without a gradient to record they launch the kernel directly.  Each is also a ``torch.library`` op, so
``torch.compile(fullgraph=True)`` and other tracers see one node:

* ``granite::layer_norm(x, weight, bias, eps, lengths?)``, ``granite::layer_norm_backward``
* ``granite::dropout_add(x, residual?, rng, p, scale, site, lengths?)``
* ``granite::dropout_add_layer_norm(x, residual, weight, bias, rng, p, scale, site, eps, lengths?) -> (y, h)``,
  ``granite::dropout_add_layer_norm_backward``
* ``granite::ctc_loss(logits, targets, input_lengths, target_lengths, blank, zero_infinity)``,
  ``granite::ctc_loss_backward``

Tensors are bf16, fp16 or fp32 on one CUDA device, parameters fp32 or of the activations' type; work runs on that
device's current stream.  Results repeat bit for bit.  Tensors with a forward-mode tangent are refused (by the bare
ops as dual tensors only: under ``torch.func.jvp`` torch hands a custom op the values alone).  ``lengths`` (int [B], with
x [B, T, D]) marks the frames t >= lengths[b] as padding: nothing of them is read, normed outputs and gradients there are
zero, they join no weight gradient, and a residual passes through.

``rng`` is an int64 tensor of two on the device, (seed, offset), which the kernels read when they run: a captured graph
draws new masks when it holds ``rng[1] += 1`` after its backward pass.  ``site`` tells apart the dropouts of one step.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_HERE = contextlib.nullcontext()
MAX_NORM_WIDTH = 8192
MAX_ROW_ELEMENTS = 2 ** 31 - 256
INFERENCE_WIDTHS = (256, 512, 1024, 2048)       # of gsn_layernorm_bf16
MAX_CTC_LABELS = 2000
MAX_CTC_FRAMES = 16384
MAX_CTC_CLASSES = 2 ** 31 - 1024


def _on(device: torch.device):
    """The launches go to the current device: make the tensors' device that."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)       # current_stream() without its object: 2 us less


def _dense(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _int32(t: torch.Tensor) -> torch.Tensor:
    """Dense int32; what int64 holds beyond it stays out of every range."""
    if t.dtype == torch.int64:
        t = t.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def _check_device(name: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    if forward_ad._current_level >= 0:             # inside a dual_level: a tangent would be lost without a word
        for t in (first, *others):
            if t is not None and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name}: no forward-mode derivative; use the backward pass")
    if not first.is_cuda:
        raise RuntimeError(f"{name}: every tensor must be on a CUDA device (got {first.device}); the kernels have no "
                           "CPU path")
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{name}: tensors on {first.device} and {t.device}")


def _check_rows(name: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    if first.dim() < 1 or not 0 < first.shape[-1] <= MAX_ROW_ELEMENTS:
        raise RuntimeError(f"{name}: rows of 1 to {MAX_ROW_ELEMENTS} elements expected, got {tuple(first.shape)}")
    if first.dtype not in _TYPES:
        raise RuntimeError(f"{name}: bf16, fp16 or fp32 tensors expected, got {first.dtype}")
    for t in others:
        if t is not None and (t.dtype != first.dtype or t.shape != first.shape):
            raise RuntimeError(f"{name}: {first.dtype} {tuple(first.shape)} against {t.dtype} {tuple(t.shape)}")


def _check_params(name: str, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> None:
    D = x.shape[-1]
    if D > MAX_NORM_WIDTH:
        raise RuntimeError(f"{name}: width {D}, at most {MAX_NORM_WIDTH}")
    if weight.shape != (D,) or (bias is not None and bias.shape != (D,)):
        raise RuntimeError(f"{name}: weight and bias must be [{D}]")
    if weight.dtype not in (torch.float32, x.dtype) or (bias is not None and bias.dtype != weight.dtype):
        raise RuntimeError(f"{name}: weight and bias must both be fp32 or {x.dtype}")


def _check_dropout(name: str, rng: torch.Tensor, p: float, site: int) -> None:
    if rng.dtype != torch.int64 or rng.shape != (2,):
        raise RuntimeError(f"{name}: rng must be int64 [2] (seed, offset), got {rng.dtype} {tuple(rng.shape)}")
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"{name}: p={p} is not a probability")
    if not 0 <= site < 2 ** 32:
        raise RuntimeError(f"{name}: site={site} outside [0, 2^32)")


def _check_lengths(name: str, x: torch.Tensor, lengths: Optional[torch.Tensor]) -> Tuple[Optional[torch.Tensor], int]:
    if lengths is None:
        return None, 0
    if x.dim() != 3 or lengths.shape != x.shape[:1] or lengths.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{name}: lengths must be int [B] beside [B, T, D], got {lengths.dtype} "
                           f"{tuple(lengths.shape)} beside {tuple(x.shape)}")
    return _int32(lengths), x.shape[1]


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """(tensor, row stride): t itself where its rows are dense and evenly spaced, else a copy."""
    D = t.shape[-1]
    if t.is_contiguous():
        return t, D
    if t.stride(-1) == 1 or D == 1:
        try:
            r = t.view(-1, D)
        except RuntimeError:
            return t.contiguous(), D
        if r.shape[0] <= 1:
            return t, D
        if r.stride(0) >= D:
            return t, r.stride(0)
    return t.contiguous(), D


# ---- layer norm ------------------------------------------------------------------------------------------------------
def _layer_norm(x, weight, bias, eps, lengths):
    name = "granite::layer_norm"
    _check_device(name, x, weight, bias, lengths)
    _check_rows(name, x)
    _check_params(name, x, weight, bias)
    lens, T = _check_lengths(name, x, lengths)
    D = x.shape[-1]
    y = _dense(x)
    with _on(x.device):
        xr, ld = _rows(x)
        w, b = weight.contiguous(), bias.contiguous()
        if (lens is None and x.dtype == w.dtype == torch.bfloat16 and D in INFERENCE_WIDTHS
                and not (w.data_ptr() | b.data_ptr()) & 15
                and (not x.is_contiguous() or not xr.data_ptr() & 15)):
            # what the inference path's norm takes keeps its kernel, and its bits: views off its 16-byte grid as a copy
            if ld % 8 or xr.data_ptr() & 15:
                xr, ld = x.contiguous(), D
            _lib.call("gsn_layernorm_bf16", xr.data_ptr(), ld, w.data_ptr(), b.data_ptr(), y.data_ptr(), D,
                      y.numel() // D, D, eps, None, 0, _stream(x.device))
            return y
        _lib.call("gsn_layer_norm_fwd", xr.data_ptr(), ld, w.data_ptr(), b.data_ptr(), y.data_ptr(), y.numel() // D, D,
                  eps, _TYPES[x.dtype], _TYPES[w.dtype], _ptr(lens), T, _stream(x.device))
    return y


def _layer_norm_backward(dy, x, weight, eps, lengths):
    name = "granite::layer_norm_backward"
    _check_device(name, x, dy, weight, lengths)
    _check_rows(name, x, dy)
    _check_params(name, x, weight, None)
    lens, T = _check_lengths(name, x, lengths)
    D = x.shape[-1]
    dx = _dense(x)
    M = dx.numel() // D
    dw, db = _dense(weight), _dense(weight)
    with _on(x.device):
        xr, ld_x = _rows(x)
        gr, ld_g = _rows(dy)
        w = weight.contiguous()
        nbytes = _lib.lib().gsn_layer_norm_bwd_workspace_bytes(M, D)
        ws = x.new_empty((nbytes,), dtype=torch.uint8)
        _lib.call("gsn_layer_norm_bwd", gr.data_ptr(), ld_g, xr.data_ptr(), ld_x, w.data_ptr(), dx.data_ptr(),
                  dw.data_ptr(), db.data_ptr(), M, D, eps, _TYPES[x.dtype], _TYPES[w.dtype], _ptr(lens), T,
                  ws.data_ptr(), nbytes, _stream(x.device))
    return dx, dw, db


@torch.library.custom_op("granite::layer_norm_backward", mutates_args=(), device_types="cuda")
def layer_norm_backward_op(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, eps: float,
                           lengths: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) of granite::layer_norm."""
    return _layer_norm_backward(dy, x, weight, eps, lengths)


@layer_norm_backward_op.register_fake
def _(dy, x, weight, eps, lengths):
    return (torch.empty_like(x, memory_format=torch.contiguous_format), weight.new_empty(weight.shape),
            weight.new_empty(weight.shape))


_PLAIN = (torch.Tensor, torch.nn.Parameter)
_compiling = torch.compiler.is_compiling
_tracing = torch._C._is_tracing
_modes = torch._C._len_torch_dispatch_stack
_early_modes = torch._ops.mode_stack_state_for_pre_dispatch().count


def _dispatched(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a call has to go through the dispatcher: a graph being compiled or traced (whatever watches the ops that
    are called would see an empty output and no kernel), another mode that takes them, or a tensor subclass."""
    if _compiling() or _tracing() or _modes() or _early_modes():
        return True
    for t in tensors:
        if t is not None and type(t) not in _PLAIN:
            return True
    return False


def _recorded(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a call has a gradient to record.  It is then an autograd.Function around the direct launches: 95 to 127
    us of the CPU for a call and its gradient instead of 152 to 206 through the dispatcher's op (137 to 160 with
    setup_context as a function of its own; torch.func transforms, which want that, take neither form)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, lengths):
        ctx.eps = eps
        ctx.save_for_backward(x, weight, lengths)
        return _layer_norm(x, weight, bias, eps, lengths)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, lengths = ctx.saved_tensors
        return (*layer_norm_backward(dy, x, weight, ctx.eps, lengths), None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5,
               lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """nn.LayerNorm over the last dim, differentiable in x, weight and bias."""
    if _dispatched(x, weight, bias):
        return torch.ops.granite.layer_norm(x, weight, bias, eps, lengths)
    if _recorded(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps, lengths)
    return _layer_norm(x, weight, bias, eps, lengths)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                        lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) of layer_norm at x for the gradient dy of its output."""
    if _dispatched(dy, x, weight):
        return torch.ops.granite.layer_norm_backward(dy, x, weight, eps, lengths)
    return _layer_norm_backward(dy, x, weight, eps, lengths)


# ---- dropout with a residual -----------------------------------------------------------------------------------------
def _dropout_add(x, residual, rng, p, scale, site, lengths):
    name = "granite::dropout_add"
    _check_device(name, x, residual, rng, lengths)
    _check_rows(name, x, residual)
    _check_dropout(name, rng, p, site)
    lens, T = _check_lengths(name, x, lengths)
    D = x.shape[-1]
    out = _dense(x)
    with _on(x.device):
        xr, ld_x = _rows(x)
        rr, ld_r = (None, 0) if residual is None else _rows(residual)
        _lib.call("gsn_dropout_add", xr.data_ptr(), ld_x, _ptr(rr), ld_r, out.data_ptr(), out.numel() // D, D,
                  _TYPES[x.dtype], rng.contiguous().data_ptr(), site, p, scale, _ptr(lens), T, _stream(x.device))
    return out


@torch.library.custom_op("granite::dropout_add", mutates_args=(), device_types="cuda")
def dropout_add_op(x: torch.Tensor, residual: Optional[torch.Tensor], rng: torch.Tensor, p: float, scale: float,
                   site: int, lengths: Optional[torch.Tensor]) -> torch.Tensor:
    """residual + scale * dropout(x) (scale * dropout(x) without a residual)."""
    return _dropout_add(x, residual, rng, p, scale, site, lengths)


@dropout_add_op.register_fake
def _(x, residual, rng, p, scale, site, lengths):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _dropout_add_setup(ctx, inputs, output):
    _, residual, rng, ctx.p, ctx.scale, ctx.site, lengths = inputs
    ctx.save_for_backward(rng, lengths)
    ctx.with_residual = residual is not None


def _dropout_add_grad(ctx, dout):
    rng, lengths = ctx.saved_tensors
    dx = None
    if ctx.needs_input_grad[0]:
        dx = torch.ops.granite.dropout_add(dout, None, rng, ctx.p, ctx.scale, ctx.site, lengths)
    return dx, dout if ctx.with_residual else None, None, None, None, None, None


dropout_add_op.register_autograd(_dropout_add_grad, setup_context=_dropout_add_setup)


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        _dropout_add_setup(ctx, inputs, None)
        return _dropout_add(*inputs)

    @staticmethod
    def backward(ctx, dout):                       # linear in x: its gradient is the same call, with a gradient of its own
        rng, lengths = ctx.saved_tensors
        dx = dropout_add(dout, rng, ctx.p, None, ctx.scale, ctx.site, lengths) if ctx.needs_input_grad[0] else None
        return dx, dout if ctx.with_residual else None, None, None, None, None, None


def dropout_add(x: torch.Tensor, rng: torch.Tensor, p: float, residual: Optional[torch.Tensor] = None,
                scale: float = 1.0, site: int = 0, lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + scale * dropout(x, p), differentiable in x and residual; p to the nearest 1 / 65536."""
    if _dispatched(x, residual):
        return torch.ops.granite.dropout_add(x, residual, rng, p, scale, site, lengths)
    if _recorded(x, residual):
        return _DropoutAdd.apply(x, residual, rng, p, scale, site, lengths)
    return _dropout_add(x, residual, rng, p, scale, site, lengths)


def dropout_add_backward(dout: torch.Tensor, rng: torch.Tensor, p: float, scale: float = 1.0, site: int = 0,
                         lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of dropout_add's x for the gradient dout of its output (the residual's is dout itself)."""
    if _dispatched(dout):
        return torch.ops.granite.dropout_add(dout, None, rng, p, scale, site, lengths)
    return _dropout_add(dout, None, rng, p, scale, site, lengths)


# ---- dropout, residual and layer norm in one pass --------------------------------------------------------------------
def _dropout_add_layer_norm(x, residual, weight, bias, rng, p, scale, site, eps, lengths):
    name = "granite::dropout_add_layer_norm"
    _check_device(name, x, residual, weight, bias, rng, lengths)
    _check_rows(name, x, residual)
    _check_params(name, x, weight, bias)
    _check_dropout(name, rng, p, site)
    lens, T = _check_lengths(name, x, lengths)
    D = x.shape[-1]
    y = _dense(x)
    h = _dense(x)
    with _on(x.device):
        xr, ld_x = _rows(x)
        rr, ld_r = _rows(residual)
        w, b = weight.contiguous(), bias.contiguous()
        _lib.call("gsn_dropout_add_layer_norm_fwd", xr.data_ptr(), ld_x, rr.data_ptr(), ld_r, w.data_ptr(),
                  b.data_ptr(), y.data_ptr(), h.data_ptr(), y.numel() // D, D, eps, _TYPES[x.dtype], _TYPES[w.dtype],
                  rng.contiguous().data_ptr(), site, p, scale, _ptr(lens), T, _stream(x.device))
    return y, h


def _dropout_add_layer_norm_backward(dy, dh, h, weight, rng, p, scale, site, eps, lengths):
    name = "granite::dropout_add_layer_norm_backward"
    _check_device(name, h, dy, dh, weight, rng, lengths)
    _check_rows(name, h, dy, dh)
    _check_params(name, h, weight, None)
    _check_dropout(name, rng, p, site)
    lens, T = _check_lengths(name, h, lengths)
    D = h.shape[-1]
    dx = _dense(h)
    dres = _dense(h)
    M = dx.numel() // D
    dw, db = _dense(weight), _dense(weight)
    with _on(h.device):
        hr, ld_h = _rows(h)
        gr, ld_g = _rows(dy)
        sr, ld_s = (None, 0) if dh is None else _rows(dh)
        w = weight.contiguous()
        nbytes = _lib.lib().gsn_layer_norm_bwd_workspace_bytes(M, D)
        ws = h.new_empty((nbytes,), dtype=torch.uint8)
        _lib.call("gsn_dropout_add_layer_norm_bwd", gr.data_ptr(), ld_g, _ptr(sr), ld_s, hr.data_ptr(), ld_h,
                  w.data_ptr(), dx.data_ptr(), dres.data_ptr(), dw.data_ptr(), db.data_ptr(), M, D, eps,
                  _TYPES[h.dtype], _TYPES[w.dtype], rng.contiguous().data_ptr(), site, p, scale, _ptr(lens), T,
                  ws.data_ptr(), nbytes, _stream(h.device))
    return dx, dres, dw, db


@torch.library.custom_op("granite::dropout_add_layer_norm", mutates_args=(), device_types="cuda")
def dropout_add_layer_norm_op(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
                              rng: torch.Tensor, p: float, scale: float, site: int, eps: float,
                              lengths: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = residual + scale * dropout(x), y = layer_norm(h) of the fp32 sum."""
    return _dropout_add_layer_norm(x, residual, weight, bias, rng, p, scale, site, eps, lengths)


@dropout_add_layer_norm_op.register_fake
def _(x, residual, weight, bias, rng, p, scale, site, eps, lengths):
    dense = torch.contiguous_format
    return torch.empty_like(x, memory_format=dense), torch.empty_like(x, memory_format=dense)


@torch.library.custom_op("granite::dropout_add_layer_norm_backward", mutates_args=(), device_types="cuda")
def dropout_add_layer_norm_backward_op(
        dy: torch.Tensor, dh: Optional[torch.Tensor], h: torch.Tensor, weight: torch.Tensor, rng: torch.Tensor,
        p: float, scale: float, site: int, eps: float, lengths: Optional[torch.Tensor]
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dresidual, dweight, dbias) of granite::dropout_add_layer_norm from its stored h."""
    return _dropout_add_layer_norm_backward(dy, dh, h, weight, rng, p, scale, site, eps, lengths)


@dropout_add_layer_norm_backward_op.register_fake
def _(dy, dh, h, weight, rng, p, scale, site, eps, lengths):
    dense = torch.contiguous_format
    return (torch.empty_like(h, memory_format=dense), torch.empty_like(h, memory_format=dense),
            weight.new_empty(weight.shape), weight.new_empty(weight.shape))


def _dropout_add_layer_norm_setup(ctx, inputs, output):
    _, _, weight, _, rng, ctx.p, ctx.scale, ctx.site, ctx.eps, lengths = inputs
    ctx.save_for_backward(output[1], weight, rng, lengths)
    ctx.set_materialize_grads(False)               # an unused output sends nothing back, and nothing is read for it


def _dropout_add_layer_norm_grad(ctx, dy, dh):
    h, weight, rng, lengths = ctx.saved_tensors
    rest = (None,) * 6
    if dy is None and dh is None:
        return (None,) * 10
    if dy is None:
        dx = torch.ops.granite.dropout_add(dh, None, rng, ctx.p, ctx.scale, ctx.site, lengths)
        return (dx, dh, None, None, *rest)
    grads = torch.ops.granite.dropout_add_layer_norm_backward(dy, dh, h, weight, rng, ctx.p, ctx.scale, ctx.site,
                                                              ctx.eps, lengths)
    return (*grads, *rest)


dropout_add_layer_norm_op.register_autograd(_dropout_add_layer_norm_grad, setup_context=_dropout_add_layer_norm_setup)


class _DropoutAddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        out = _dropout_add_layer_norm(*inputs)
        _dropout_add_layer_norm_setup(ctx, inputs, out)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        h, weight, rng, lengths = ctx.saved_tensors
        rest = (None,) * 6
        if dy is None and dh is None:
            return (None,) * 10
        if dy is None:
            return (dropout_add_backward(dh, rng, ctx.p, ctx.scale, ctx.site, lengths), dh, None, None, *rest)
        return (*dropout_add_layer_norm_backward(dy, dh, h, weight, rng, ctx.p, ctx.scale, ctx.site, ctx.eps, lengths),
                *rest)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
                           rng: torch.Tensor, p: float, scale: float = 1.0, site: int = 0, eps: float = 1e-5,
                           lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = residual + scale * dropout(x, p), y = layer_norm(h); differentiable in x, residual, weight, bias."""
    if _dispatched(x, residual, weight, bias):
        return torch.ops.granite.dropout_add_layer_norm(x, residual, weight, bias, rng, p, scale, site, eps, lengths)
    if _recorded(x, residual, weight, bias):
        return _DropoutAddLayerNorm.apply(x, residual, weight, bias, rng, p, scale, site, eps, lengths)
    return _dropout_add_layer_norm(x, residual, weight, bias, rng, p, scale, site, eps, lengths)


def dropout_add_layer_norm_backward(dy: torch.Tensor, dh: Optional[torch.Tensor], h: torch.Tensor,
                                    weight: torch.Tensor, rng: torch.Tensor, p: float, scale: float = 1.0,
                                    site: int = 0, eps: float = 1e-5, lengths: Optional[torch.Tensor] = None
                                    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dresidual, dweight, dbias) for the gradients dy of y and dh of h (None: nothing comes back to h)."""
    if _dispatched(dy, dh, h, weight):
        return torch.ops.granite.dropout_add_layer_norm_backward(dy, dh, h, weight, rng, p, scale, site, eps, lengths)
    return _dropout_add_layer_norm_backward(dy, dh, h, weight, rng, p, scale, site, eps, lengths)


# ---- CTC loss --------------------------------------------------------------------------------------------------------
def _ctc_check(name, logits, targets, input_lengths, target_lengths, blank):
    _check_device(name, logits, targets, input_lengths, target_lengths)
    if logits.dim() != 3 or logits.dtype not in _TYPES or logits.shape[2] == 0:
        raise RuntimeError(f"{name}: logits must be bf16, fp16 or fp32 [B, T, V], got {logits.dtype} "
                           f"{tuple(logits.shape)}")
    B, T, V = logits.shape
    ints = (torch.int32, torch.int64)
    if targets.dim() != 2 or targets.shape[0] != B or targets.dtype not in ints:
        raise RuntimeError(f"{name}: targets must be int [{B}, S], got {targets.dtype} {tuple(targets.shape)}")
    for t in (input_lengths, target_lengths):
        if t.shape != (B,) or t.dtype not in ints:
            raise RuntimeError(f"{name}: lengths must be int [{B}], got {t.dtype} {tuple(t.shape)}")
    if B >= 2 ** 31 or V > MAX_CTC_CLASSES:
        raise RuntimeError(f"{name}: {B} utterances of {V} classes, at most 2^31 - 1 and {MAX_CTC_CLASSES}")
    if not 0 <= blank < V:
        raise RuntimeError(f"{name}: blank={blank} outside the {V} classes")
    if targets.shape[1] > MAX_CTC_LABELS or T > MAX_CTC_FRAMES:
        raise RuntimeError(f"{name}: {targets.shape[1]} labels and {T} frames, at most {MAX_CTC_LABELS} and "
                           f"{MAX_CTC_FRAMES}")


def _ctc_operands(logits, targets, input_lengths, target_lengths):
    B, T, V = logits.shape
    sb, st, sv = logits.stride()
    if (sv != 1 and V > 1) or (st < V and T > 1):
        logits = logits.contiguous()
        sb, st, _ = logits.stride()
    i32 = [_int32(t) for t in (targets, input_lengths, target_lengths)]
    return logits, sb, st if T > 1 else V, i32


def _ctc_loss(logits, targets, input_lengths, target_lengths, blank, zero_infinity, gradient):
    name = "granite::ctc_loss"
    _ctc_check(name, logits, targets, input_lengths, target_lengths, blank)
    B, T, V = logits.shape
    S = targets.shape[1]
    dev = logits.device
    with _on(dev):
        x, sb, st, (tg, il, tl) = _ctc_operands(logits, targets, input_lengths, target_lengths)
        L = _lib.lib()
        state_bytes, nbytes = L.gsn_ctc_loss_state_bytes(B, T, S), L.gsn_ctc_loss_workspace_bytes(B, T, S, int(gradient))
        loss = logits.new_empty((B,), dtype=torch.float32)
        state = logits.new_empty((state_bytes,), dtype=torch.uint8)
        ws = logits.new_empty((nbytes,), dtype=torch.uint8)
        _lib.call("gsn_ctc_loss_fwd", x.data_ptr(), sb, st, tg.data_ptr(), il.data_ptr(), tl.data_ptr(), B, T, V, S,
                  blank, int(zero_infinity), int(gradient), _TYPES[x.dtype], loss.data_ptr(), state.data_ptr(),
                  state_bytes, ws.data_ptr(), nbytes, _stream(dev))
    return loss, state


def _ctc_loss_backward(dloss, logits, targets, input_lengths, target_lengths, state, blank, zero_infinity):
    name = "granite::ctc_loss_backward"
    _ctc_check(name, logits, targets, input_lengths, target_lengths, blank)
    _check_device(name, logits, dloss, state)
    B, T, V = logits.shape
    S = targets.shape[1]
    if dloss.shape != (B,):
        raise RuntimeError(f"{name}: dloss must be [{B}], got {tuple(dloss.shape)}")
    if state.dtype != torch.uint8 or not state.is_contiguous():
        raise RuntimeError(f"{name}: state must be the one of granite::ctc_loss")
    dev = logits.device
    with _on(dev):
        x, sb, st, (tg, il, tl) = _ctc_operands(logits, targets, input_lengths, target_lengths)
        dx = logits.new_empty((B, T, V))
        d = dloss.to(torch.float32).contiguous()
        _lib.call("gsn_ctc_loss_bwd", d.data_ptr(), x.data_ptr(), sb, st, tg.data_ptr(), il.data_ptr(), tl.data_ptr(),
                  B, T, V, S, blank, int(zero_infinity), _TYPES[x.dtype], state.data_ptr(), state.numel(),
                  dx.data_ptr(), _stream(dev))
    return dx


@torch.library.custom_op("granite::ctc_loss", mutates_args=(), device_types="cuda")
def ctc_loss_op(logits: torch.Tensor, targets: torch.Tensor, input_lengths: torch.Tensor,
                target_lengths: torch.Tensor, blank: int, zero_infinity: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss [B] fp32, and the bytes that its gradient needs)."""
    return _ctc_loss(logits, targets, input_lengths, target_lengths, blank, zero_infinity, True)


@ctc_loss_op.register_fake
def _(logits, targets, input_lengths, target_lengths, blank, zero_infinity):
    B, T, _ = logits.shape
    S = targets.shape[1]
    pitch = (S + 6) // 4 * 4                       # as gsn_ctc_loss_state_bytes
    sizes = (4 * B, 4 * B, 8 * B * T, 8 * B * pitch, 4 * B * T * pitch)
    nbytes = sum((n + 255) // 256 * 256 for n in sizes)
    return logits.new_empty((B,), dtype=torch.float32), logits.new_empty((nbytes,), dtype=torch.uint8)


@torch.library.custom_op("granite::ctc_loss_backward", mutates_args=(), device_types="cuda")
def ctc_loss_backward_op(dloss: torch.Tensor, logits: torch.Tensor, targets: torch.Tensor,
                         input_lengths: torch.Tensor, target_lengths: torch.Tensor, state: torch.Tensor, blank: int,
                         zero_infinity: bool) -> torch.Tensor:
    """The gradient of granite::ctc_loss's logits for the gradient dloss [B] of its loss."""
    return _ctc_loss_backward(dloss, logits, targets, input_lengths, target_lengths, state, blank, zero_infinity)


@ctc_loss_backward_op.register_fake
def _(dloss, logits, targets, input_lengths, target_lengths, state, blank, zero_infinity):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def _ctc_loss_setup(ctx, inputs, output):
    logits, targets, input_lengths, target_lengths, ctx.blank, ctx.zero_infinity = inputs
    ctx.save_for_backward(logits, targets, input_lengths, target_lengths, output[1])
    ctx.set_materialize_grads(False)


def _ctc_loss_grad(ctx, dloss, _):
    dx = None
    if dloss is not None:
        dx = torch.ops.granite.ctc_loss_backward(dloss, *ctx.saved_tensors, ctx.blank, ctx.zero_infinity)
    return dx, None, None, None, None, None


ctc_loss_op.register_autograd(_ctc_loss_grad, setup_context=_ctc_loss_setup)


class _CtcLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        out = _ctc_loss(*inputs, True)
        _ctc_loss_setup(ctx, inputs, out)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss, _):
        dx = None
        if dloss is not None:
            backward = torch.ops.granite.ctc_loss_backward if _dispatched(dloss) else _ctc_loss_backward
            dx = backward(dloss, *ctx.saved_tensors, ctx.blank, ctx.zero_infinity)
        return dx, None, None, None, None, None


def ctc_loss(logits: torch.Tensor, targets: torch.Tensor, input_lengths: torch.Tensor, target_lengths: torch.Tensor,
             blank: int = 0, zero_infinity: bool = False) -> torch.Tensor:
    """CTC loss [B] (fp32, one value an utterance, no reduction) of logits [B, T, V], any strides with V innermost, for
    targets int [B, S] with input_lengths and target_lengths int [B]; the softmax is part of it.  Differentiable in the
    logits.  An utterance without an alignment has the loss inf and a NaN gradient, or 0 and 0 with zero_infinity.  A
    class of the transcript, the blank among them, counts as masked in a frame (impossible there, as with -inf) where its
    logit lies more than 11000 below the largest of the transcript's classes; fp16's, bf16's and fp32's lowest values do."""
    if _dispatched(logits):
        return torch.ops.granite.ctc_loss(logits, targets, input_lengths, target_lengths, blank, zero_infinity)[0]
    if _recorded(logits):
        return _CtcLoss.apply(logits, targets, input_lengths, target_lengths, blank, zero_infinity)[0]
    return _ctc_loss(logits, targets, input_lengths, target_lengths, blank, zero_infinity, False)[0]
