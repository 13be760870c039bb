"""The selective state space scan and the short causal convolution in front of it, on the CUDA library.

Each batch row and channel d keeps N numbers ``h``; group ``g = d // (D / G)``
shares B and C.  Token t does, with ``step = softplus(dt + dt_bias)`` (or
``dt + dt_bias``)::

    h[n] = exp(step A[d, n]) h[n] + step x B[g, n];   out = (sum_n C[g, n] h[n] + skip x) silu(z)

* :func:`selective_scan` runs all tokens and has gradients for every input;
* :func:`selective_step` runs one token and updates the state in place;
* :func:`causal_conv` and :func:`causal_conv_step` are the same two for the
  convolution of every channel with its own 2 to 8 weights;
* :class:`SelectiveScan` is the layer around them, with :class:`GRU`'s calling
  convention, and :class:`RecurrentStack` puts layers with a norm before each
  on a residual stream.

x, dt, B, C and z are all FP32 or all bf16; A, skip, dt_bias and states are FP32.
The convolution's weights are FP32 or of x's type, its state of x's type.  All
arithmetic is FP32 (the convolution's weight gradients end in FP64 sums) and
results are rounded to bf16 once.  ``step * A`` must not be positive: states
decay.  Decays below 2^-126 count as 0.  A state that has become infinite stays
so.  Shape problems raise ``ValueError``, device and dtype problems and CUDA
failures ``RuntimeError``; there is no CPU fallback.
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib
from .norm import LayerNorm, _check_device, _check_plain, _differentiated, _first_derivatives, _no_tangents

MAX_STATES = 64
CONV_SIZES = range(2, 9)

_DTYPES = {torch.float32: _lib.GRU_F32, torch.bfloat16: _lib.GRU_BF16}
_ACTIVATIONS = {None: 0, "silu": 1}


def _fast(name, *args):
    """The call by the module in C++, or None where it leaves it to Python."""
    module = _lib.operators()
    return None if module is None or forward_ad._current_level >= 0 else getattr(module, name)(*args)


def _dense_last(t):
    """t itself if its last dimension is dense (other strides are free), else a contiguous copy."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _near(t):
    """_dense_last of [B, T, ...], with tokens less than 2^31 bytes apart, as the scan asks for."""
    t = _dense_last(t)
    return t if t is None or t.stride(1) * t.element_size() < 1 << 31 else t.contiguous()


def _check_counts(name, x):
    if any(n >= 1 << 31 for n in x.shape):
        raise ValueError(f"{name}: each of x's sizes must be below 2^31.")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _dense(t):
    return None if t is None else t.contiguous()


# ---- selective scan ----------------------------------------------------------


def _check(name, x, dt, A, B, C, skip, z, dt_bias, state, lead):
    """Sizes, types and devices of one call; ``lead`` is the number of leading dimensions."""
    if x.dim() != lead + 1 or B.dim() != lead + 2 or A.dim() != 2:
        dims = "batch" if lead == 1 else "batch, tokens"
        raise ValueError(f"{name}: x and dt must have shape [{dims}, channels], A [channels, states] and B and C [{dims}, groups, states].")
    D = x.shape[-1]
    G, N = B.shape[-2:]
    if dt.shape != x.shape or (z is not None and z.shape != x.shape):
        raise ValueError(f"{name}: dt and z must have x's shape.")
    if B.shape[:lead] != x.shape[:lead] or C.shape != B.shape:
        raise ValueError(f"{name}: B and C must have x's leading dimensions and the same groups and states.")
    if D < 1 or G < 1 or D % G:
        raise ValueError(f"{name}: the channels must be a multiple of the groups.")
    if not 1 <= N <= MAX_STATES:
        raise ValueError(f"{name}: the states must be in [1, {MAX_STATES}].")
    if A.shape != (D, N):
        raise ValueError(f"{name}: A must have shape {(D, N)}.")
    if (skip is not None and skip.shape != (D,)) or (dt_bias is not None and dt_bias.shape != (D,)):
        raise ValueError(f"{name}: skip and dt_bias must have shape ({D},).")
    if state is not None and state.shape != (x.shape[0], D, N):
        raise ValueError(f"{name}: the state must have shape {(x.shape[0], D, N)}.")
    _check_counts(name, x)
    dev = x.get_device()
    rest = [t for t in (skip, dt_bias, state) if t is not None]
    _check_device(name, dev, dt, A, B, C, z, *rest)
    _check_plain(name, x, dt, A, B, C, z, *rest)
    code = _DTYPES.get(x.dtype)
    if code is None or any(t is not None and t.dtype != x.dtype for t in (dt, B, C, z)):
        raise RuntimeError(f"{name}: x, dt, B, C and z must all be float32 or all bfloat16.")
    if any(t.dtype != torch.float32 for t in (A, *rest)):
        raise RuntimeError(f"{name}: A, skip, dt_bias and the state must be float32.")
    return code, dev


@functools.lru_cache(maxsize=4096)
def _sizes(code, B, T, D, N, G, gated):
    """Bytes of the stash, the forward's workspace and the backward's."""
    lib = _lib.load()
    a = _lib.SCAN_ARGS.pack(code, B, T, D, N, G, 0, 0, 0, 0, 0, 16 * gated, *[0] * 16)  # a gate's address, which is not read
    return lib.gru_scan_stash_bytes(a), lib.gru_scan_workspace_bytes(a, 0), lib.gru_scan_workspace_bytes(a, 1)


def _args(code, softplus, x, dt, A, B, C, skip, z, dt_bias, state):
    """The C struct for [B, T, ...] tensors."""
    zs = (0, 0) if z is None else z.stride()[:2]
    return _lib.SCAN_ARGS.pack(code, x.shape[0], x.shape[1], *A.shape, B.shape[2], int(softplus), x.data_ptr(), dt.data_ptr(),
                               B.data_ptr(), C.data_ptr(), _ptr(z), A.data_ptr(), _ptr(skip), _ptr(dt_bias), _ptr(state),
                               *x.stride()[:2], *dt.stride()[:2], *zs, *B.stride()[:3], *C.stride()[:3])


def _scan_forward(code, dev, x, dt, A, B, C, skip, z, dt_bias, softplus, state, train):
    """out, the last state, the inputs as they were read and, to train, what the gradient needs besides them."""
    x, dt, B, C, z = (_near(t) for t in (x, dt, B, C, z))
    A, skip, dt_bias, state = (_dense(t) for t in (A, skip, dt_bias, state))
    (b, T, D), (_, N) = x.shape, A.shape
    with _lib.on_device(dev):
        out, last = x.new_empty((b, T, D)), A.new_empty((b, D, N))
        stash_bytes, ws_bytes, _ = _sizes(code, b, T, D, N, B.shape[2], z is not None)
        stash = A.new_empty(stash_bytes // 4) if train else None
        ws = A.new_empty(ws_bytes // 4) if ws_bytes else None
        _lib.check(_lib.load().gru_scan_forward(_args(code, softplus, x, dt, A, B, C, skip, z, dt_bias, state), out.data_ptr(),
                                                last.data_ptr(), _ptr(stash), stash_bytes if train else 0, _ptr(ws), ws_bytes,
                                                _lib.raw_stream(dev)), "gru_scan_forward")
    return out, last, (x, dt, A, B, C, skip, z, dt_bias, stash)


class SelectiveScanFunction(torch.autograd.Function):
    """``(x, dt, A, B, C, skip, z, dt_bias, softplus, state) -> (out, last state)``; first derivatives, by backward only."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, skip, z, dt_bias, softplus, state):
        code, dev = _check("selective_scan", x, dt, A, B, C, skip, z, dt_bias, state, 2)
        out, last, kept = _scan_forward(code, dev, x, dt, A, B, C, skip, z, dt_bias, softplus, state, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*kept)
        ctx.code, ctx.softplus = code, softplus
        return out, last

    @staticmethod
    def backward(ctx, dout, dlast):
        x, dt, A, B, C, skip, z, dt_bias, stash = ctx.saved_tensors
        (b, T, D), (_, N), G = x.shape, A.shape, B.shape[2]
        dev = x.get_device()
        stash_bytes, _, ws_bytes = _sizes(ctx.code, b, T, D, N, G, z is not None)
        with _lib.on_device(dev):
            dout, dlast = _dense(dout), _dense(dlast)
            dx, ddt = x.new_empty((b, T, D)), x.new_empty((b, T, D))
            dz = None if z is None else x.new_empty((b, T, D))
            dB, dC = x.new_empty((b, T, G, N)), x.new_empty((b, T, G, N))
            dA = A.new_empty((D, N))
            dskip, dbias = (None if t is None else A.new_empty(D) for t in (skip, dt_bias))
            ds = A.new_empty((b, D, N)) if ctx.needs_input_grad[9] else None
            ws = A.new_empty(ws_bytes // 4)
            _lib.check(_lib.load().gru_scan_backward(
                _args(ctx.code, ctx.softplus, x, dt, A, B, C, skip, z, dt_bias, None), _ptr(dout), _ptr(dlast), _ptr(stash),
                stash_bytes, dx.data_ptr(), ddt.data_ptr(), dA.data_ptr(), dB.data_ptr(), dC.data_ptr(), _ptr(dskip), _ptr(dz),
                _ptr(dbias), _ptr(ds), ws.data_ptr(), ws_bytes, _lib.raw_stream(dev)), "gru_scan_backward")
        dx, ddt, dA, dB, dC, dskip, dz, dbias, ds = _first_derivatives(
            "selective_scan", (dx, ddt, dA, dB, dC, dskip, dz, dbias, ds))
        return dx, ddt, dA, dB, dC, dskip, dz, dbias, None, ds


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   skip: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                   initial_state: Optional[torch.Tensor] = None):
    """All tokens of a batch: ``(out [B, T, D], last state [B, D, N])``.

    ``x``, ``dt``, ``z``: [B, T, D]; ``A``: [D, N], negative in use; ``B``, ``C``: [B, T, G, N]
    with D a multiple of G; ``skip``, ``dt_bias``: [D].  The strides of all but the
    last dimension are free.
    """
    softplus = bool(dt_softplus)
    got = _fast("selective_scan", x, dt, A, B, C, skip, z, dt_bias, softplus, initial_state)
    if got is not None:
        return got
    if _differentiated(x, dt, A, B, C, skip, z, dt_bias, initial_state):
        return SelectiveScanFunction.apply(x, dt, A, B, C, skip, z, dt_bias, softplus, initial_state)
    code, dev = _check("selective_scan", x, dt, A, B, C, skip, z, dt_bias, initial_state, 2)
    return _scan_forward(code, dev, x, dt, A, B, C, skip, z, dt_bias, softplus, initial_state, False)[:2]


def selective_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, state: torch.Tensor,
                   skip: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False) -> torch.Tensor:
    """One token: ``out [B, D]``; ``state`` [B, D, N] (contiguous) is updated in place.

    ``x``, ``dt``, ``z``: [B, D]; ``B``, ``C``: [B, G, N].  No gradient.
    """
    got = _fast("selective_step", x, dt, A, B, C, state, skip, z, dt_bias, bool(dt_softplus))
    if got is not None:
        return got
    code, dev = _check("selective_step", x, dt, A, B, C, skip, z, dt_bias, state, 1)
    _no_tangents("selective_step", x, dt, A, B, C, skip, z, dt_bias, state)
    if not state.is_contiguous():
        raise ValueError("selective_step: the state is updated in place and must be contiguous.")
    x, dt, B, C, z = (_dense_last(t) for t in (x, dt, B, C, z))
    A, skip, dt_bias = _dense(A), _dense(skip), _dense(dt_bias)
    b, D = x.shape
    (Bb, Bg, _), (Cb, Cg, _) = B.stride(), C.stride()
    a = _lib.SCAN_ARGS.pack(code, b, 1, D, A.shape[1], B.shape[1], int(bool(dt_softplus)), x.data_ptr(), dt.data_ptr(),
                            B.data_ptr(), C.data_ptr(), _ptr(z), A.data_ptr(), _ptr(skip), _ptr(dt_bias), 0, x.stride(0), 0,
                            dt.stride(0), 0, 0 if z is None else z.stride(0), 0, Bb, 0, Bg, Cb, 0, Cg)
    with _lib.on_device(dev):
        out = x.new_empty((b, D))
        _lib.check(_lib.load().gru_scan_step(a, state.data_ptr(), out.data_ptr(), _lib.raw_stream(dev)), "gru_scan_step")
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return out


# ---- causal convolution --------------------------------------------------------


def _check_conv(name, x, weight, bias, state, activation, lead):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{name}: activation must be None or 'silu'.")
    if x.dim() != lead + 1 or weight.dim() != 2:
        dims = "batch" if lead == 1 else "batch, tokens"
        raise ValueError(f"{name}: x must have shape [{dims}, channels] and weight [channels, size].")
    D, W = weight.shape
    if x.shape[-1] != D or D < 1 or (bias is not None and bias.shape != (D,)):
        raise ValueError(f"{name}: x, weight and bias must have the same channels.")
    if W not in CONV_SIZES:
        raise ValueError(f"{name}: the weight's size must be in [{CONV_SIZES[0]}, {CONV_SIZES[-1]}].")
    if state is not None and state.shape != (x.shape[0], W - 1, D):
        raise ValueError(f"{name}: the state must have shape {(x.shape[0], W - 1, D)}.")
    _check_counts(name, x)
    dev = x.get_device()
    _check_device(name, dev, weight, bias, state)
    _check_plain(name, x, weight, bias, state)
    code = _DTYPES.get(x.dtype)
    if code is None or (state is not None and state.dtype != x.dtype):
        raise RuntimeError(f"{name}: x and the state must both be float32 or both bfloat16.")
    if weight.dtype not in (x.dtype, torch.float32) or (bias is not None and bias.dtype != weight.dtype):
        raise RuntimeError(f"{name}: weight and bias must both be float32 or both of x's type.")
    return code, dev


def _conv_args(code, activation, x, weight, bias, state):
    return _lib.CONV_ARGS.pack(code, _DTYPES[weight.dtype], x.shape[0], x.shape[1], *weight.shape, _ACTIVATIONS[activation],
                               x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(state), *x.stride()[:2])


def _conv_forward(code, dev, x, weight, bias, activation, state):
    x, weight, bias, state = _dense_last(x), weight.contiguous(), _dense(bias), _dense(state)
    b, T, D = x.shape
    with _lib.on_device(dev):
        out, last = x.new_empty((b, T, D)), x.new_empty((b, weight.shape[1] - 1, D))
        _lib.check(_lib.load().gru_conv_forward(_conv_args(code, activation, x, weight, bias, state), out.data_ptr(),
                                                last.data_ptr(), _lib.raw_stream(dev)), "gru_conv_forward")
    return out, last, (x, weight, bias, state)


class CausalConvFunction(torch.autograd.Function):
    """``(x, weight, bias, activation, state) -> (out, last state)``; first derivatives, by backward only."""

    @staticmethod
    def forward(ctx, x, weight, bias, activation, state):
        code, dev = _check_conv("causal_conv", x, weight, bias, state, activation, 2)
        out, last, kept = _conv_forward(code, dev, x, weight, bias, activation, state)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*kept)
        ctx.code, ctx.activation = code, activation
        return out, last

    @staticmethod
    def backward(ctx, dout, dlast):
        x, weight, bias, state = ctx.saved_tensors
        dev = x.get_device()
        with _lib.on_device(dev):
            dout, dlast = _dense(dout), _dense(dlast)
            dx, dw = x.new_empty(x.shape), torch.empty_like(weight)
            db = None if bias is None else torch.empty_like(bias)
            ds = torch.empty_like(state) if ctx.needs_input_grad[4] else None
            a = _conv_args(ctx.code, ctx.activation, x, weight, bias, state)
            ws_bytes = _lib.load().gru_conv_workspace_bytes(a)
            ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=x.device)
            _lib.check(_lib.load().gru_conv_backward(a, _ptr(dout), _ptr(dlast), dx.data_ptr(), dw.data_ptr(), _ptr(db),
                                                     _ptr(ds), ws.data_ptr(), ws_bytes, _lib.raw_stream(dev)),
                       "gru_conv_backward")
        dx, dw, db, ds = _first_derivatives("causal_conv", (dx, dw, db, ds))
        return dx, dw, db, None, ds


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                initial_state: Optional[torch.Tensor] = None):
    """``out_t = act(bias + sum_j weight[:, j] x_(t - W + 1 + j))`` and the state after it: ``([B, T, D], [B, W - 1, D])``.

    ``x``: [B, T, D], strides free but the last; ``weight``: [D, W], 2 <= W <= 8; ``activation``: None or
    "silu"; ``initial_state``: the W - 1 inputs before the first, oldest first (default zeros).
    """
    got = _fast("causal_conv", x, weight, bias, activation, initial_state)
    if got is not None:
        return got
    if _differentiated(x, weight, bias, initial_state):
        return CausalConvFunction.apply(x, weight, bias, activation, initial_state)
    code, dev = _check_conv("causal_conv", x, weight, bias, initial_state, activation, 2)
    return _conv_forward(code, dev, x, weight, bias, activation, initial_state)[:2]


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, state: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     activation: Optional[str] = None) -> torch.Tensor:
    """One token, ``x`` [B, D] -> [B, D]; ``state`` [B, W - 1, D] (contiguous) is moved on in place.  No gradient."""
    got = _fast("causal_conv_step", x, weight, state, bias, activation)
    if got is not None:
        return got
    code, dev = _check_conv("causal_conv_step", x, weight, bias, state, activation, 1)
    _no_tangents("causal_conv_step", x, weight, bias, state)
    if not state.is_contiguous():
        raise ValueError("causal_conv_step: the state is updated in place and must be contiguous.")
    x, weight, bias = _dense_last(x), weight.contiguous(), _dense(bias)
    a = _lib.CONV_ARGS.pack(code, _DTYPES[weight.dtype], x.shape[0], 1, *weight.shape, _ACTIVATIONS[activation], x.data_ptr(),
                            weight.data_ptr(), _ptr(bias), 0, x.stride(0), 0)
    with _lib.on_device(dev):
        out = x.new_empty(x.shape)
        _lib.check(_lib.load().gru_conv_step(a, state.data_ptr(), out.data_ptr(), _lib.raw_stream(dev)), "gru_conv_step")
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return out


# ---- layers ----------------------------------------------------------------------


class SelectiveScan(nn.Module):
    """A selective scan layer: ``(input [B, T, input_size], state) -> (output [B, T, output], state)``.

    One projection makes the channels (``inner_size``, default twice the input's)
    and their gates; after the causal convolution another makes every token's B, C
    and, through ``dt_rank`` numbers, step sizes; the scan's gated output goes
    through an output projection.  A state is a pair: the convolution's
    [B, conv_size - 1, inner] and the scan's [B, inner, state_size].
    """

    def __init__(self, input_size: int, inner_size: Optional[int] = None, state_size: int = 16, conv_size: int = 4,
                 num_groups: int = 1, dt_rank: Optional[int] = None, output_size: Optional[int] = None) -> None:
        super().__init__()
        inner = 2 * input_size if inner_size is None else inner_size
        rank = max(1, math.ceil(input_size / 16)) if dt_rank is None else dt_rank
        if input_size < 1 or rank < 1 or num_groups < 1 or inner < 1 or inner % num_groups:
            raise ValueError("SelectiveScan: sizes must be positive and inner_size a multiple of num_groups.")
        if not 1 <= state_size <= MAX_STATES or conv_size not in CONV_SIZES:
            raise ValueError(f"SelectiveScan: state_size must be in [1, {MAX_STATES}], conv_size in "
                             f"[{CONV_SIZES[0]}, {CONV_SIZES[-1]}].")
        self.input_size, self.inner_size, self.state_size, self.conv_size = input_size, inner, state_size, conv_size
        self.num_groups, self.output_size = num_groups, input_size if output_size is None else output_size
        self._split = (rank, num_groups * state_size, num_groups * state_size)
        self.in_proj = nn.Linear(input_size, 2 * inner, bias=False)
        self.conv_weight = nn.Parameter(torch.empty(inner, conv_size).uniform_(-conv_size ** -0.5, conv_size ** -0.5))
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        self.x_proj = nn.Linear(inner, sum(self._split), bias=False)
        self.dt_proj = nn.Linear(rank, inner, bias=False)
        # steps that remember from ten tokens to a thousand; decay rates 1 to N
        start = torch.exp(torch.linspace(math.log(1e-3), math.log(1e-1), inner))
        self.dt_bias = nn.Parameter(torch.log(torch.expm1(start)))
        self.log_rate = nn.Parameter(torch.log(torch.arange(1, state_size + 1, dtype=torch.float32)).repeat(inner, 1))
        self.skip = nn.Parameter(torch.ones(inner))
        self.out_proj = nn.Linear(inner, self.output_size, bias=False)

    def init_state(self, batch: int, dtype: Optional[torch.dtype] = None):
        """Zeros; ``dtype`` is the convolution's (default: that of the projection's output, which autocast sets)."""
        like = self.in_proj.weight
        kind = like.device.type
        if dtype is None:
            cast = torch.amp.is_autocast_available(kind) and torch.is_autocast_enabled(kind)
            dtype = torch.get_autocast_dtype(kind) if cast else like.dtype
        return (torch.zeros(batch, self.conv_size - 1, self.inner_size, dtype=dtype, device=like.device),
                torch.zeros(batch, self.inner_size, self.state_size, dtype=torch.float32, device=like.device))

    def _inputs(self, x, z):
        """Everything that the scan takes beside the state, from the convolution's output."""
        low, b, c = self.x_proj(x).split(self._split, dim=-1)
        groups = (self.num_groups, self.state_size)
        dt = self.dt_proj(low)
        # one type, which under autocast is the projections'
        return dict(x=x.to(dt.dtype), dt=dt, A=-self.log_rate.float().exp(), B=b.unflatten(-1, groups), C=c.unflatten(-1, groups),
                    skip=self.skip.float(), z=z.to(dt.dtype), dt_bias=self.dt_bias.float(), dt_softplus=True)

    def forward(self, x: torch.Tensor, state=None):
        if x.dim() != 3 or x.shape[-1] != self.input_size:
            raise ValueError(f"x must have shape [batch, seq, {self.input_size}].")
        conv, scan = (None, None) if state is None else state
        u, z = self.in_proj(x).chunk(2, dim=-1)
        u, conv = causal_conv(u, self.conv_weight, self.conv_bias, "silu", conv)
        y, scan = selective_scan(**self._inputs(u, z), initial_state=scan)
        return self.out_proj(y), (conv, scan)

    @torch.no_grad()
    def step(self, x: torch.Tensor, state) -> torch.Tensor:
        """One token of every sequence, [batch, input_size]; both states are updated in place."""
        if x.dim() != 2 or x.shape[-1] != self.input_size:
            raise ValueError(f"x must have shape [batch, {self.input_size}].")
        u, z = self.in_proj(x).chunk(2, dim=-1)
        u = causal_conv_step(u, self.conv_weight, state[0], self.conv_bias, "silu")
        return self.out_proj(selective_step(**self._inputs(u, z), state=state[1]))


class RecurrentStack(nn.Module):
    """Recurrent layers on a residual stream: ``(input [B, T, width], states) -> (output [B, T, width], states)``.

    Before each layer (:class:`GRU`, :class:`GatedDelta`, :class:`SelectiveScan`:
    width in, width out) the stream takes in what the one before gave and is
    normalised, in one pass; a last norm gives the output.
    """

    def __init__(self, layers, width: int, eps: float = 1e-5) -> None:
        super().__init__()
        self.layers = nn.ModuleList(layers)
        self.norms = nn.ModuleList(LayerNorm(width, eps) for _ in range(len(self.layers) + 1))

    def _run(self, x, call):
        y, stream = self.norms[0](x), x
        for i, norm in enumerate(self.norms[1:]):
            y, stream = norm(call(i, y), stream)
        return y

    def forward(self, x: torch.Tensor, states=None):
        last = []

        def call(i, y):
            out, state = self.layers[i](y, None if states is None else states[i])
            last.append(state)
            return out

        return self._run(x, call), last

    @torch.no_grad()
    def step(self, x: torch.Tensor, states) -> torch.Tensor:
        """One token of every sequence, [batch, width], through layers that have a step (:class:`GRU` has none: RuntimeError);
        states are updated in place.  Layers ahead of one that refuses its own state have moved theirs on."""
        if len(states) < len(self.layers):
            raise ValueError(f"RecurrentStack.step: {len(self.layers)} states are needed, one for each layer; there are {len(states)}.")
        for layer in self.layers:
            if not callable(getattr(layer, "step", None)):
                raise RuntimeError(f"RecurrentStack.step: {type(layer).__name__} has no step.")
        return self._run(x, lambda i, y: self.layers[i].step(y, states[i]))
