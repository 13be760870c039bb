"""Layer normalisation on the CUDA library, with the sum of a residual stream in front.

``layer_norm(x, weight, bias, eps, residual)`` normalises the last dimension of
``s = x + residual`` (``s = x`` without one) in one pass over the rows each way::

    s = x + residual, rounded to the residual's type;  y = (s - mean) / sqrt(variance + eps) * weight + bias

x is FP32 or bf16; the residual and the weights are FP32 or of x's type.
Statistics, sums over rows and the arithmetic are FP32 (sums of the weights'
gradients FP64 at the end); y is the norm of s as it is returned, so that the
gradient, which reads s again, sees the numbers that were normalised.  The last
dimension may have 1 to 16384 elements.  Shape problems raise ``ValueError``,
device and dtype problems and CUDA failures ``RuntimeError``; there is no CPU
fallback.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib
from .gru import is_b200_available

MAX_NORM_WIDTH = 16384

_DTYPES = {torch.float32: _lib.GRU_F32, torch.bfloat16: _lib.GRU_BF16}
_supported: dict = {}  # device index -> whether it is a B200


def _check_plain(name, *tensors):
    """Numbers are read as they lie in memory."""
    if any(t is not None and t.is_neg() for t in tensors):
        raise RuntimeError(f"{name}: a tensor has a pending negation; give its resolve_neg().")


def _check_device(name, dev, *tensors):
    """All tensors on CUDA device ``dev``, a B200."""
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name}: all tensors must be on the same CUDA device.")
    if dev < 0:
        raise RuntimeError(f"{name} requires CUDA tensors.")
    ok = _supported.get(dev)
    if ok is None:
        ok = _supported[dev] = is_b200_available(dev)
    if not ok:
        raise RuntimeError("rnn_kernel_b200 requires a B200-class (sm_100) GPU.")


class _NoSecondDerivative(torch.autograd.Function):
    """Passes gradients on; their own derivative raises, where without it they would count as constants."""

    @staticmethod
    def forward(ctx, anchor, name, *grads):
        ctx.name = name
        return tuple(None if g is None else g.clone() for g in grads)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no second derivative.")


def _first_derivatives(name, grads):
    """What a backward returns: with create_graph=True, gradients that raise when they are differentiated."""
    if torch.is_grad_enabled():
        return _NoSecondDerivative.apply(torch.empty(0, requires_grad=True), name, *grads)
    return tuple(grads)


def _differentiated(*tensors):
    """Whether a call has to go through autograd: gradients asked for, a level of forward mode (which the Functions refuse), or a
    trace (whose replay calls the Function again)."""
    return forward_ad._current_level >= 0 or _lib.traced() or (
        torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


def _no_tangents(name, *tensors):
    """For calls without a derivative, which are no autograd functions and change a state in place."""
    if _lib.traced():
        raise RuntimeError(f"{name} cannot be traced: it updates its state in place.")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no derivative.")


def _check(x, weight, bias, residual, eps):
    name = "layer_norm"
    D = x.shape[-1] if x.dim() else 0
    if x.dim() < 1 or not 1 <= D <= MAX_NORM_WIDTH:
        raise ValueError(f"{name}: x's last dimension must have 1 to {MAX_NORM_WIDTH} elements.")
    if weight.shape != (D,) or (bias is not None and bias.shape != (D,)):
        raise ValueError(f"{name}: weight and bias must have shape ({D},).")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"{name}: the residual must have x's shape.")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"{name}: eps must be finite and not negative.")
    dev = x.get_device()
    if weight.get_device() != dev or (bias is not None and bias.get_device() != dev) or \
            (residual is not None and residual.get_device() != dev):
        raise ValueError(f"{name}: all tensors must be on the same CUDA device.")
    dtype = x.dtype
    if x.is_cuda:
        if dtype not in _DTYPES:
            raise RuntimeError(f"{name}: x must be float32 or bfloat16.")
        if weight.dtype not in (dtype, torch.float32) or (bias is not None and bias.dtype != weight.dtype):
            raise RuntimeError(f"{name}: weight and bias must both be float32 or both of x's type.")
        if residual is not None and residual.dtype not in (dtype, torch.float32):
            raise RuntimeError(f"{name}: the residual must be float32 or of x's type.")
    _check_device(name, dev)
    _check_plain(name, x, weight, bias, residual)
    return dev


def _rows(t):
    """t as rows: a view where its leading dimensions allow one and the last is dense, else a copy."""
    r = t.reshape(-1, t.shape[-1])
    return r if r.stride(-1) == 1 or r.shape[-1] == 1 else r.contiguous()


def _forward(dev, x, weight, bias, residual, eps, train):
    """out, the sum (or None), x's or the sum's rows, and the rows' statistics to train."""
    rows, res = _rows(x), None if residual is None else _rows(residual)
    weight, bias = weight.contiguous(), None if bias is None else bias.contiguous()
    R, D = rows.shape
    kept = x.dtype if residual is None else residual.dtype
    with _lib.on_device(dev):
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        s = None if residual is None else torch.empty(x.shape, dtype=kept, device=x.device)
        stats = torch.empty((3, R), dtype=torch.float32, device=x.device) if train else None
        a = _lib.NORM_ARGS.pack(_DTYPES[x.dtype], _DTYPES[kept], _DTYPES[weight.dtype], D, eps, R, rows.stride(0),
                                D if res is None else res.stride(0))
        _lib.check(_lib.load().gru_layer_norm_forward(
            a, rows.data_ptr(), 0 if res is None else res.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
            out.data_ptr(), 0 if s is None else s.data_ptr(), stats.data_ptr() if train else 0, _lib.raw_stream(dev)),
            "gru_layer_norm_forward")
    return out, s, rows, weight, stats


@functools.lru_cache(maxsize=4096)
def _workspace(code, kept, wcode, D, R):
    return _lib.load().gru_layer_norm_workspace_bytes(_lib.NORM_ARGS.pack(code, kept, wcode, D, 0.0, R, D, D))


class LayerNormFunction(torch.autograd.Function):
    """``(x, weight, bias or None, residual or None, eps) -> (out, sum or None)``; first derivatives, by backward only."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        dev = _check(x, weight, bias, residual, eps)
        out, s, rows, weight, stats = _forward(dev, x, weight, bias, residual, eps, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(rows if s is None else s, weight, stats)
        ctx.shape, ctx.dtype, ctx.summed, ctx.biased = x.shape, x.dtype, s is not None, bias is not None
        return out, s

    @staticmethod
    def backward(ctx, dout, dsum):
        s, weight, stats = ctx.saved_tensors
        rows = s.reshape(-1, ctx.shape[-1])
        R, D = rows.shape
        dev = rows.get_device()
        codes = (_DTYPES[ctx.dtype], _DTYPES[rows.dtype], _DTYPES[weight.dtype])
        with _lib.on_device(dev):
            dout = torch.zeros(ctx.shape, dtype=ctx.dtype, device=rows.device) if dout is None else dout.contiguous()
            dsum = None if dsum is None else dsum.contiguous()
            # a sum hands the same gradient to both of its terms, as torch's addition does, if they have one type
            both = ctx.summed and rows.dtype != ctx.dtype
            dx = torch.empty(ctx.shape, dtype=ctx.dtype, device=rows.device)
            dres = torch.empty(ctx.shape, dtype=rows.dtype, device=rows.device) if both else None
            dw = torch.empty_like(weight)
            db = torch.empty_like(weight) if ctx.biased else None
            ws_bytes = _workspace(*codes, D, R)
            ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=rows.device)
            a = _lib.NORM_ARGS.pack(*codes, D, 0.0, R, rows.stride(0), D)
            _lib.check(_lib.load().gru_layer_norm_backward(
                a, rows.data_ptr(), weight.data_ptr(), stats.data_ptr(), dout.data_ptr(),
                0 if dsum is None else dsum.data_ptr(), dx.data_ptr(), 0 if dres is None else dres.data_ptr(), dw.data_ptr(),
                0 if db is None else db.data_ptr(), ws.data_ptr(), ws_bytes, _lib.raw_stream(dev)), "gru_layer_norm_backward")
        dx, dw, db, dres = _first_derivatives("layer_norm", (dx, dw, db, dres))
        return dx, dw, db, (dres if both else dx) if ctx.summed else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None):
    """The norm of x over its last dimension; with a ``residual`` of x's shape, ``(norm of x + residual, x + residual)``."""
    eps = float(eps)
    fast = _lib.operators()
    if fast is not None and forward_ad._current_level < 0:
        got = fast.layer_norm(x, weight, bias, eps, residual)
        if got is not None:
            return got
    if _differentiated(x, weight, bias, residual):
        out, s = LayerNormFunction.apply(x, weight, bias, residual, eps)
    else:
        dev = _check(x, weight, bias, residual, eps)
        out, s = _forward(dev, x, weight, bias, residual, eps, False)[:2]
    return out if residual is None else (out, s)


class LayerNorm(nn.Module):
    """:func:`layer_norm` with its weights: ``norm(x)``, or ``norm(x, residual) -> (out, sum)``."""

    def __init__(self, width: int, eps: float = 1e-5, bias: bool = True) -> None:
        super().__init__()
        if not 1 <= width <= MAX_NORM_WIDTH:
            raise ValueError(f"LayerNorm: width must be in [1, {MAX_NORM_WIDTH}].")
        self.width, self.eps = width, eps
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width)) if bias else None

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return layer_norm(x, self.weight, self.bias, self.eps, residual)
