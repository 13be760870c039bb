"""The gated delta rule on the CUDA library: a recurrent layer whose state is a matrix.

Each batch row and value head keeps a state ``S [dk, dv]``; token t, with log
decay ``g_t`` and writing strength ``beta_t``, does::

    S' = exp(g_t) S;   u = beta_t (v_t - S'^T k_t);   S = S' + k_t u^T;   o_t = scale S^T q_t

* :func:`gated_delta_rule` runs all tokens of a batch (in chunks of 64 on the
  tensor cores) and has gradients for every input;
* :func:`gated_delta_step` runs one token and updates the state in place;
* :class:`GatedDelta` is the layer around them, with :class:`GRU`'s calling
  convention: ``(input, state) -> (output, state)``.

q, k and v are FP32 or bf16, gates and states FP32.  Sums are FP32; what the
tensor cores multiply keeps 22 bits of a number down to 2^-17 of the largest that
shares its scale, and 2^-39 of that below.  A token's head of q or k has a scale,
and so have 16 neighbouring value columns of a token; of a state, a quarter of its
key columns x 16 value columns, and 16 tokens in what they add to it.  So tokens of
any size leave one another their digits, except where a state holds them in
different key columns; and a key or value column that is 2^17 times smaller than its
neighbours loses digits to them.  Results are rounded to bf16 once.  Value heads may outnumber key heads (``Hv = n Hk``: value head h
reads key head ``h // n``).  Shape problems raise ``ValueError``, device and
dtype problems and CUDA failures ``RuntimeError``; there is no CPU fallback.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad

from . import _lib
from .gru import is_b200_available

MAX_HEAD_SIZE = 128

_DTYPES = {torch.float32: _lib.GRU_F32, torch.bfloat16: _lib.GRU_BF16}
_supported: dict = {}  # device index -> whether it is a B200


def _check(name, q, k, v, g, beta, state, lead):
    """Sizes, types and devices of one call; ``lead`` is the number of leading dimensions."""
    qs, vs = q.shape, v.shape
    if len(qs) != lead + 2 or len(vs) != lead + 2:
        dims = "batch" if lead == 1 else "batch, tokens"
        raise ValueError(f"{name}: q, k, v must have shape [{dims}, heads, size] and g, beta [{dims}, value heads].")
    if k.shape != qs:
        raise ValueError(f"{name}: k must have q's shape.")
    gates = vs[:-1]
    if vs[:lead] != qs[:lead] or g.shape != gates or beta.shape != gates:
        raise ValueError(f"{name}: v, g and beta must have q's leading dimensions and the same value heads.")
    Hk, dk = qs[-2:]
    Hv, dv = vs[-2:]
    if Hk < 1 or Hv < 1 or Hv % Hk:
        raise ValueError(f"{name}: the value heads must be a multiple of the key heads.")
    if not 1 <= dk <= MAX_HEAD_SIZE or not 1 <= dv <= MAX_HEAD_SIZE:
        raise ValueError(f"{name}: head sizes must be in [1, {MAX_HEAD_SIZE}].")
    if state is not None and state.shape != (qs[0], Hv, dk, dv):
        raise ValueError(f"{name}: the state must have shape {(qs[0], Hv, dk, dv)}.")
    dev, dtype = q.get_device(), q.dtype
    if k.get_device() != dev or v.get_device() != dev or g.get_device() != dev or beta.get_device() != dev \
            or (state is not None and state.get_device() != dev):
        raise ValueError(f"{name}: all tensors must be on the same CUDA device.")
    if not q.is_cuda:
        raise RuntimeError(f"{name} requires CUDA tensors.")
    code = _DTYPES.get(dtype)
    if code is None or k.dtype != dtype or v.dtype != dtype:
        raise RuntimeError(f"{name}: q, k and v must all be float32 or all bfloat16.")
    f32 = torch.float32
    if g.dtype != f32 or beta.dtype != f32 or (state is not None and state.dtype != f32):
        raise RuntimeError(f"{name}: g, beta and the state must be float32.")
    ok = _supported.get(dev)
    if ok is None:
        ok = _supported[dev] = is_b200_available(dev)
    if not ok:
        raise RuntimeError("rnn_kernel_b200 requires a B200-class (sm_100) GPU.")
    return code


def _dense_heads(t):
    """t itself if its last dimension is dense (other strides are free), else a contiguous copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _args(code, q, k, v, g, beta, state, scale):
    """The C struct for [B, T, ...] tensors."""
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2:]
    return _lib.DELTA_ARGS.pack(code, B, T, Hk, Hv, dk, dv, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                g.data_ptr(), beta.data_ptr(), 0 if state is None else state.data_ptr(),
                                *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *g.stride(), *beta.stride())


@functools.lru_cache(maxsize=4096)
def _sizes(code, B, T, Hk, Hv, dk, dv):
    """Bytes of the stash, the forward's workspace and the backward's."""
    lib = _lib.load()
    a = _lib.DELTA_ARGS.pack(code, B, T, Hk, Hv, dk, dv, 1.0, *[0] * 21)
    return lib.gru_delta_stash_bytes(a), lib.gru_delta_workspace_bytes(a, 0), lib.gru_delta_workspace_bytes(a, 1)


def _forward(code, q, k, v, g, beta, state, scale, train):
    """out, the last state and, to train, what the gradient needs besides the inputs."""
    q, k, v = _dense_heads(q), _dense_heads(k), _dense_heads(v)
    state = None if state is None else state.contiguous()
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2:]
    dev = q.get_device()
    stash_bytes, ws_bytes, _ = _sizes(code, B, T, Hk, Hv, dk, dv)
    with _lib.on_device(dev):
        out = v.new_empty((B, T, Hv, dv))
        last = g.new_empty((B, Hv, dk, dv))
        memory = g.new_empty((stash_bytes if train else ws_bytes) // 4)
        where = (memory.data_ptr(), stash_bytes, 0, 0) if train else (0, 0, memory.data_ptr(), ws_bytes)
        _lib.check(_lib.load().gru_delta_forward(_args(code, q, k, v, g, beta, state, scale), out.data_ptr(), last.data_ptr(),
                                                 *where, _lib.raw_stream(dev)), "gru_delta_forward")
    return out, last, memory


class _NoSecondDerivative(torch.autograd.Function):
    """Passes gradients on; their own derivative raises, where without it they would count as constants."""

    @staticmethod
    def forward(ctx, anchor, *grads):
        return tuple(None if g is None else g.clone() for g in grads)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("gated_delta_rule has no second derivative.")


class GatedDeltaRuleFunction(torch.autograd.Function):
    """``(q, k, v, g, beta, state or None, scale) -> (out, last state)``; first derivatives, by backward only."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, scale):
        code = _check("gated_delta_rule", q, k, v, g, beta, state, 2)
        out, last, stash = _forward(code, q, k, v, g, beta, state, scale, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(g, stash)  # which holds what the gradient needs of the other inputs
        B, T, Hk, dk = q.shape
        ctx.sizes, ctx.scale, ctx.dtype = (code, B, T, Hk, v.shape[2], dk, v.shape[3]), scale, q.dtype
        return out, last

    @staticmethod
    def backward(ctx, dout, dlast):
        g, stash = ctx.saved_tensors
        _, B, T, Hk, Hv, dk, dv = ctx.sizes
        dev = g.get_device()
        stash_bytes, _, ws_bytes = _sizes(*ctx.sizes)
        with _lib.on_device(dev):
            dout = None if dout is None else dout.contiguous()
            dlast = None if dlast is None else dlast.contiguous()
            gq, gk = (g.new_empty((B, T, Hk, dk), dtype=ctx.dtype) for _ in range(2))
            gv = g.new_empty((B, T, Hv, dv), dtype=ctx.dtype)
            gg, gb = g.new_empty((B, T, Hv)), g.new_empty((B, T, Hv))
            gs = g.new_empty((B, Hv, dk, dv)) if ctx.needs_input_grad[5] else None
            ws = g.new_empty(ws_bytes // 4)
            a = _lib.DELTA_ARGS.pack(*ctx.sizes, ctx.scale, 0, 0, 0, g.data_ptr(), 0, 0, *[0] * 9, *g.stride(), 0, 0, 0)
            _lib.check(_lib.load().gru_delta_backward(
                a, 0 if dout is None else dout.data_ptr(), 0 if dlast is None else dlast.data_ptr(), stash.data_ptr(),
                stash_bytes, gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), gg.data_ptr(), gb.data_ptr(),
                0 if gs is None else gs.data_ptr(), ws.data_ptr(), ws_bytes, _lib.raw_stream(dev)), "gru_delta_backward")
        if torch.is_grad_enabled():  # create_graph=True
            gq, gk, gv, gg, gb, gs = _NoSecondDerivative.apply(torch.empty(0, requires_grad=True), gq, gk, gv, gg, gb, gs)
        return gq, gk, gv, gg, gb, gs, None


def _forward_mode() -> bool:
    """Inside a dual level: tensors may carry tangents, under no_grad too."""
    return forward_ad._current_level >= 0


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     initial_state: Optional[torch.Tensor] = None, scale: Optional[float] = None):
    """All tokens of a batch: ``(out [B, T, Hv, dv], last state [B, Hv, dk, dv])``.

    ``q``, ``k``: [B, T, Hk, dk]; ``v``: [B, T, Hv, dv]; ``g`` (log of the decay, <= 0
    in use; -inf forgets the state), ``beta``: [B, T, Hv].  ``scale`` defaults to
    ``dk ** -0.5``.  Keys are used as given: normalise them for a stable rule.
    The other strides than the last dimension's are free.
    """
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    needed = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state))
    if needed or _forward_mode() or _lib.traced():  # the Function refuses tangents; a trace's replay calls it again
        return GatedDeltaRuleFunction.apply(q, k, v, g, beta, initial_state, scale)
    code = _check("gated_delta_rule", q, k, v, g, beta, initial_state, 2)
    out, last, _ = _forward(code, q, k, v, g, beta, initial_state, scale, False)
    return out, last


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """One token: ``out [B, Hv, dv]``; ``state`` [B, Hv, dk, dv] (contiguous) is updated in place.

    ``q``, ``k``: [B, Hk, dk]; ``v``: [B, Hv, dv]; ``g``, ``beta``: [B, Hv].  No gradient.
    """
    code = _check("gated_delta_step", q, k, v, g, beta, state, 1)
    if _forward_mode() and any(forward_ad.unpack_dual(t).tangent is not None for t in (q, k, v, g, beta, state)):
        raise RuntimeError("gated_delta_step has no derivative.")
    if _lib.traced():
        raise RuntimeError("gated_delta_step cannot be traced: it updates its state in place.")
    if not state.is_contiguous():
        raise ValueError("gated_delta_step: the state is updated in place and must be contiguous.")
    q, k, v = _dense_heads(q), _dense_heads(k), _dense_heads(v)
    B, Hk, dk = q.shape
    Hv, dv = v.shape[1:]
    dev = q.get_device()
    (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    (gb, gh), (bb, bh) = g.stride(), beta.stride()
    a = _lib.DELTA_ARGS.pack(code, B, 1, Hk, Hv, dk, dv, dk ** -0.5 if scale is None else scale, q.data_ptr(), k.data_ptr(),
                             v.data_ptr(), g.data_ptr(), beta.data_ptr(), 0, qb, 0, qh, kb, 0, kh, vb, 0, vh, gb, 0, gh,
                             bb, 0, bh)
    with _lib.on_device(dev):
        out = v.new_empty((B, Hv, dv))
        _lib.check(_lib.load().gru_delta_step(a, state.data_ptr(), out.data_ptr(), _lib.raw_stream(dev)), "gru_delta_step")
    torch.autograd.graph.increment_version(state)
    return out


class GatedDelta(nn.Module):
    """A gated delta rule layer: ``(input [B, T, input_size], state) -> (output [B, T, output], state)``.

    One projection makes q, k (L2-normalised), v, the decay and the writing
    strength of every head; the heads' outputs, RMS-normalised per head, go
    through an output projection back to ``output_size`` (default: the input's).
    """

    def __init__(self, input_size: int, num_heads: int = 4, head_size: int = 64, num_key_heads: Optional[int] = None,
                 output_size: Optional[int] = None) -> None:
        super().__init__()
        num_key_heads = num_heads if num_key_heads is None else num_key_heads
        if input_size < 1 or num_heads < 1 or num_key_heads < 1 or num_heads % num_key_heads:
            raise ValueError("GatedDelta: num_heads must be a positive multiple of num_key_heads, input_size >= 1.")
        if not 1 <= head_size <= MAX_HEAD_SIZE:
            raise ValueError(f"GatedDelta: head_size must be in [1, {MAX_HEAD_SIZE}].")
        self.input_size, self.num_heads, self.num_key_heads, self.head_size = input_size, num_heads, num_key_heads, head_size
        self.output_size = input_size if output_size is None else output_size
        self._split = (num_key_heads * head_size, num_key_heads * head_size, num_heads * head_size, num_heads, num_heads)
        self.in_proj = nn.Linear(input_size, sum(self._split), bias=False)
        self.out_proj = nn.Linear(num_heads * head_size, self.output_size, bias=False)
        self.norm_weight = nn.Parameter(torch.ones(head_size))
        # decays from a few tokens to a few hundred
        self.log_rate = nn.Parameter(torch.linspace(-5.0, 0.0, num_heads))

    def init_state(self, batch: int) -> torch.Tensor:
        return torch.zeros(batch, self.num_heads, self.head_size, self.head_size, dtype=torch.float32,
                           device=self.log_rate.device)

    def _project(self, x):
        q, k, v, a, b = self.in_proj(x).split(self._split, dim=-1)
        keys, values = (self.num_key_heads, self.head_size), (self.num_heads, self.head_size)
        # back to v's type, which under autocast is the projection's and not x's
        q = F.normalize(q.unflatten(-1, keys).float(), dim=-1).to(v.dtype)
        k = F.normalize(k.unflatten(-1, keys).float(), dim=-1).to(v.dtype)
        g = -self.log_rate.float().exp() * F.softplus(a.float())
        return q, k, v.unflatten(-1, values), g, b.float().sigmoid()

    def _finish(self, o):
        rms = o.float().square().mean(-1, keepdim=True).add(1e-6).rsqrt()
        return self.out_proj((o * rms * self.norm_weight).to(o.dtype).flatten(-2))

    def forward(self, x: torch.Tensor, state: Optional[torch.Tensor] = None):
        if x.dim() != 3 or x.shape[-1] != self.input_size:
            raise ValueError(f"x must have shape [batch, seq, {self.input_size}].")
        o, last = gated_delta_rule(*self._project(x), initial_state=state)
        return self._finish(o), last

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        """One token of every sequence, [batch, input_size]; ``state`` is updated in place."""
        if x.dim() != 2 or x.shape[-1] != self.input_size:
            raise ValueError(f"x must have shape [batch, {self.input_size}].")
        return self._finish(gated_delta_step(*self._project(x), state))
