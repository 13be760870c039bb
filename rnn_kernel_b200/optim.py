"""AdamW on the CUDA library: every tensor's step in one launch, moments in 32 or in 8 bits.

The reference harness trains with ``torch.optim.AdamW`` (rnn_benchmark.py);
:class:`AdamW` computes the same update (decoupled weight decay, bias
correction) in FP32 for FP32 or bf16 weights::

    m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
    p = (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

``state_bits=8`` holds each moment in one byte: blocks of 256 elements share an
FP32 scale, codes are logarithmic with 3 mantissa bits, and rounding is
stochastic from ``(seed, step, position)``, so a run repeats bit for bit; ``eps``
must be 2^-50 or more, since second moments below 2^-100 are held as zero.  A
block that meets a gradient that is not finite has NaN moments from then on,
as 32-bit moments of those elements would.  CUDA tensors only; there is no
fallback.
"""
from __future__ import annotations

import functools
import math
import warnings
from typing import Iterable, Optional

import numpy as np
import torch

from . import _lib

STATE_BLOCK = 256  # elements per 8-bit scale; every tensor's moments start a block
# a block's second moments below 2^-100 are held as zero, so eps has to be at least their root
MIN_EPS_8 = 2.0 ** -50

_DTYPES = {torch.float32: _lib.GRU_F32, torch.bfloat16: _lib.GRU_BF16}
# gru_adamw_tensor of include/rnn_kernel_b200.h
_ENTRY = np.dtype([("param", "u8"), ("grad", "u8"), ("n", "i8"), ("state_offset", "i8"), ("decay", "f4"),
                   ("step_size", "f4"), ("inv_sqrt_bc2", "f4"), ("pad", "f4")])


@functools.lru_cache(maxsize=1)
def _reader():
    """The C++ reader of tensors, or None (said once) where it cannot be built: the Python below does the same."""
    try:
        return _lib.host().adamw_addresses
    except Exception as e:  # no compiler, no headers, a module that does not load
        warnings.warn(f"AdamW reads its tensors in Python, some 0.5 us each: the module _host is not available ({e})")
        return None


class _TypeTable:
    """The C call's table of the parameters of one element type."""

    def __init__(self, opt: "AdamW", dt: torch.dtype, group_of: np.ndarray) -> None:
        self.dtype, self.code = dt, _DTYPES[dt]
        self.index = np.array([i for i, p in enumerate(opt.params) if p.dtype == dt], dtype=np.int64)
        self.params = [opt.params[i] for i in self.index]
        self.group = group_of[self.index]
        cuts = [0] + (np.flatnonzero(np.diff(self.group)) + 1).tolist() + [len(self.index)]
        self.groups = [(lo, hi, int(self.group[lo])) for lo, hi in zip(cuts[:-1], cuts[1:])]
        self.entries = np.zeros(len(self.index), dtype=_ENTRY)
        self.entries["n"], self.entries["state_offset"] = opt._sizes[self.index], opt._offsets[self.index]
        self._bind()

    def _bind(self) -> None:
        """What belongs to this object alone: the address of its own entries, which a copy of it does not share."""
        self.address = self.entries.ctypes.data
        self.addresses = _reader()
        self.copies = None  # dense copies of gradients that are not, until the launch

    def __getstate__(self) -> dict:
        # for copy.deepcopy and pickle: they make new entries, elsewhere
        return {k: v for k, v in self.__dict__.items() if k not in ("address", "addresses", "copies")}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._bind()

    def gather(self, device: torch.device) -> Optional[np.ndarray]:
        """Fills in this step's addresses; the mask of parameters without a gradient, None where all have one."""
        if self.addresses is not None and self.addresses(self.params, self.address, self.code, device.index):
            return None
        grads = []
        # a new .data may lie where the old one did
        for p, n in zip(self.params, self.entries["n"].tolist()):
            if p.dtype != self.dtype or p.numel() != n or p.device != device or not p.is_contiguous():
                raise RuntimeError("AdamW: a parameter's type, size, device or layout has changed.")
            g = p.grad
            if g is not None and (g.layout is not torch.strided or g.dtype != self.dtype or g.device != device):
                raise RuntimeError("AdamW: gradients must be dense and of their parameter's type.")
            if g is not None and g.numel() != n:
                raise RuntimeError("AdamW: a gradient's size is not what its parameter's was.")
            grads.append(g)
        without = np.array([g is None for g in grads])
        self.copies = grads = [g if g is None else g.contiguous() for g in grads]
        self.entries["param"] = [p.data_ptr() for p in self.params]
        self.entries["grad"] = [0 if g is None else g.data_ptr() for g in grads]
        return without if without.any() else None


class AdamW:
    """``torch.optim.AdamW``'s update over all tensors at once.

    ``params`` is an iterable of tensors, or of dicts with ``"params"`` and
    optionally ``"lr"`` and ``"weight_decay"``; ``param_groups`` holds them, and
    a schedule may set a group's ``"lr"`` between steps (the object is no
    ``torch.optim.Optimizer``, which torch's schedulers ask for; its parameters
    are fixed).  Parameters without a gradient are skipped and keep their own step
    count.  Copies and pickles are optimizers of their own.

    ``capturable=True`` keeps the step count on the device, so that a step
    captured in a CUDA graph advances with every replay; the learning rates
    are those at capture, and every parameter needs its gradient.
    """

    def __init__(self, params: Iterable, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, seed: int = 0, capturable: bool = False) -> None:
        if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
            raise ValueError("betas must be in [0, 1).")
        if not eps >= 0.0:
            raise ValueError("eps must be >= 0.")
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32.")
        if state_bits == 8 and not eps >= MIN_EPS_8:
            raise ValueError("eps must be >= 2^-50 with 8-bit moments: smaller second moments' roots count as zero.")
        self.betas, self.eps = (float(betas[0]), float(betas[1])), float(eps)
        self.state_bits, self.seed, self.capturable = state_bits, int(seed) & 0xFFFFFFFF, bool(capturable)
        groups = list(params)
        if not groups:
            raise ValueError("AdamW got no parameters.")
        if not isinstance(groups[0], dict):
            groups = [{"params": groups}]
        self.param_groups = []
        for g in groups:
            ps = g["params"]
            ps = [ps] if isinstance(ps, torch.Tensor) else list(ps)
            group = {"params": ps, "lr": float(g.get("lr", lr)), "weight_decay": float(g.get("weight_decay", weight_decay))}
            if not group["lr"] >= 0.0 or not group["weight_decay"] >= 0.0:
                raise ValueError("lr and weight_decay must be >= 0.")
            self.param_groups.append(group)
        self.params = [p for g in self.param_groups for p in g["params"]]
        if not self.params or len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("AdamW needs parameters, each of them once.")
        for p in self.params:
            if not isinstance(p, torch.Tensor) or not p.is_cuda or p.dtype not in _DTYPES:
                raise RuntimeError("AdamW: FP32 or bf16 CUDA parameters are required.")
            if not p.is_contiguous():
                raise ValueError("AdamW: parameters must be contiguous.")
        self.device = self.params[0].device
        if any(p.device != self.device for p in self.params):
            raise ValueError("AdamW: all parameters must be on the same CUDA device.")

        sizes = np.array([p.numel() for p in self.params], dtype=np.int64)
        ends = np.cumsum(-(-sizes // STATE_BLOCK) * STATE_BLOCK)
        self.state_elems = int(ends[-1])
        self._offsets = np.concatenate([np.zeros(1, np.int64), ends[:-1]])
        self._sizes = sizes
        n = max(self.state_elems, STATE_BLOCK)
        kind = torch.float32 if state_bits == 32 else torch.uint8
        self.exp_avg = torch.zeros(n, dtype=kind, device=self.device)[:self.state_elems]
        self.exp_avg_sq = torch.zeros(n, dtype=kind, device=self.device)[:self.state_elems]
        self.scale_avg = self.scale_sq = None
        if state_bits == 8:
            self.scale_avg = torch.zeros(n // STATE_BLOCK, device=self.device)
            self.scale_sq = torch.zeros(n // STATE_BLOCK, device=self.device)
        self._calls = 0
        self._steps = np.zeros(len(self.params), dtype=np.int64)
        self._device_step = torch.zeros(1, dtype=torch.int64, device=self.device) if capturable else None
        self._scalars = torch.zeros(3, device=self.device) if capturable else None
        group_of = np.array([i for i, g in enumerate(self.param_groups) for _ in g["params"]], dtype=np.int64)
        # one table per element type, its entries in the parameters' order
        self._tables = [_TypeTable(self, dt, group_of) for dt in _DTYPES if any(p.dtype == dt for p in self.params)]
        self._steady = True  # every parameter has had its gradient in every step: _steps is not kept up

    def step(self, grad_scale: float = 1.0) -> None:
        """Updates the parameters in place from their ``.grad`` times ``grad_scale``."""
        lib = _lib.load()
        missing = [t.gather(self.device) for t in self._tables]
        if any(m is not None for m in missing):
            if self.capturable:
                raise RuntimeError("AdamW(capturable=True): every parameter needs a gradient.")
            if self._steady:
                self._steps[:] = self._calls
            self._steady = False
        before = self._calls, None if self._steady else self._steps.copy()
        self._calls += 1
        b1, b2 = self.betas
        dev = self.device.index
        scales = (None, None) if self.scale_avg is None else (self.scale_avg.data_ptr(), self.scale_sq.data_ptr())
        counter = None if self._device_step is None else self._device_step.data_ptr()
        scalars = None if self._scalars is None else self._scalars.data_ptr()
        try:
            with _lib.on_device(dev):
                stream = _lib.raw_stream(dev)
                for table, without in zip(self._tables, missing):
                    entries, address = table.entries, table.address
                    if without is not None:
                        entries = entries[~without]
                        address = entries.ctypes.data
                    if not len(entries):
                        continue
                    self._rates(table, entries, without)
                    _lib.check(lib.gru_adamw_step(
                        address, len(entries), table.code, self.state_bits, self.exp_avg.data_ptr(),
                        self.exp_avg_sq.data_ptr(), *scales, self.state_elems, b1, b2, self.eps, grad_scale, self.seed,
                        self._calls, counter, scalars, stream), "gru_adamw_step")
                    counter = None  # counted once for all element types
                    table.copies = None
        except Exception:
            # a refused step is none: its number stays the next one's
            self._calls = before[0]
            if before[1] is not None:
                self._steps[:] = before[1]
            raise
        torch.autograd.graph.increment_version(self.params)

    def _rates(self, table, entries, without) -> None:
        """Writes the learning rates, decays and bias corrections of this step; counts it."""
        b1, b2 = self.betas
        if self._steady:
            # all parameters are at the same step
            t = self._calls
            r1, r2 = (1.0, 0.0) if self.capturable else (1.0 - b1 ** t, 1.0 / math.sqrt(1.0 - b2 ** t))
            for lo, hi, i in table.groups:
                lr = self.param_groups[i]["lr"]
                part = entries[lo:hi]
                part["decay"] = 1.0 - lr * self.param_groups[i]["weight_decay"]
                part["step_size"] = lr / r1
                part["inv_sqrt_bc2"] = r2
            return
        index = table.index if without is None else table.index[~without]
        group = table.group if without is None else table.group[~without]
        self._steps[index] += 1
        t = self._steps[index]
        lr = np.array([g["lr"] for g in self.param_groups])
        entries["decay"] = (1.0 - lr * np.array([g["weight_decay"] for g in self.param_groups]))[group]
        entries["step_size"] = lr[group] / (1.0 - b1 ** t)
        entries["inv_sqrt_bc2"] = 1.0 / np.sqrt(1.0 - b2 ** t)

    def zero_grad(self, set_to_none: bool = True) -> None:
        for p in self.params:
            if p.grad is not None:
                if set_to_none:
                    p.grad = None
                else:
                    p.grad.zero_()

    def moments(self):
        """Both moments as FP32 buffers: tensor i's at ``[offset_i, offset_i + numel_i)`` (:meth:`offsets`), zeros
        between.  32-bit moments are the optimizer's own buffers, 8-bit ones are decoded into new ones."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        m = torch.empty(self.state_elems, device=self.device)
        v = torch.empty(self.state_elems, device=self.device)
        dev = self.device.index
        with _lib.on_device(dev):
            _lib.check(_lib.load().gru_adamw_decode(
                self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), self.scale_avg.data_ptr(), self.scale_sq.data_ptr(),
                self.state_elems, m.data_ptr(), v.data_ptr(), _lib.raw_stream(dev)),
                "gru_adamw_decode")
        return m, v

    def offsets(self):
        """(offset, elements) of each parameter's moments in :meth:`moments`' buffers, in order."""
        return list(zip(self._offsets.tolist(), self._sizes.tolist()))

    def state_dict(self) -> dict:
        """What continues this run bit for bit: moments as they are held, counts, betas, eps and the groups' rates."""
        calls = self._calls if self._device_step is None else int(self._device_step)
        steps = [calls] * len(self.params) if self._steady else self._steps.tolist()
        return {"state_bits": self.state_bits, "betas": self.betas, "eps": self.eps, "seed": self.seed, "sizes": self._sizes.tolist(), "calls": calls,
                "steps": steps, "exp_avg": self.exp_avg.clone(), "exp_avg_sq": self.exp_avg_sq.clone(),
                "scale_avg": None if self.scale_avg is None else self.scale_avg.clone(),
                "scale_sq": None if self.scale_sq is None else self.scale_sq.clone(),
                "groups": [{"lr": g["lr"], "weight_decay": g["weight_decay"]} for g in self.param_groups]}

    @torch.no_grad()
    def load_state_dict(self, state: dict) -> None:
        if state["state_bits"] != self.state_bits or list(state["sizes"]) != self._sizes.tolist() \
                or len(state["groups"]) != len(self.param_groups):
            raise ValueError("AdamW: the state belongs to other parameters or another state_bits.")
        if self._device_step is not None:
            if any(t != state["calls"] for t in state["steps"]):
                raise ValueError("AdamW(capturable=True): the state's parameters have different step counts.")
            self._device_step.fill_(state["calls"])
        self._calls, self.seed = int(state["calls"]), int(state["seed"])
        if "betas" in state:  # states of before they were saved keep what this object was made with
            self.betas, self.eps = (float(state["betas"][0]), float(state["betas"][1])), float(state["eps"])
        self._steps[:] = state["steps"]
        self._steady = all(t == self._calls for t in state["steps"])
        for name in ("exp_avg", "exp_avg_sq", "scale_avg", "scale_sq"):
            mine: Optional[torch.Tensor] = getattr(self, name)
            if mine is not None:
                mine.copy_(state[name])
        for g, s in zip(self.param_groups, state["groups"]):
            g.update(lr=float(s["lr"]), weight_decay=float(s["weight_decay"]))
