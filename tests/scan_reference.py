"""Plain 64-bit selective scan, causal convolution and layer norm for the tests (torch, any device; differentiable by autograd)."""
import math

import pytest
import torch
import torch.nn.functional as F

from rnn_kernel_b200 import _lib


@pytest.fixture(autouse=True, params=["C++", "Python"])
def caller(request, monkeypatch):
    """Every test that imports this runs with the calls made by the module in C++ and with those made in Python."""
    if request.param == "Python":
        monkeypatch.setattr(_lib, "operators", lambda: None)
    else:
        assert _lib.operators() is not None


def scan(x, dt, A, B, C, skip=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None):
    """``(out [B, T, D], last state)`` in float64, token by token, from inputs of any type."""
    b, T, D = x.shape
    G, N = B.shape[2:]
    x, dt, A, B, C = (t.double() for t in (x, dt, A, B, C))
    B, C = (t.repeat_interleave(D // G, dim=2) for t in (B, C))
    step = dt if dt_bias is None else dt + dt_bias.double()
    step = F.softplus(step, threshold=60.0) if dt_softplus else step
    h = x.new_zeros(b, D, N) if initial_state is None else initial_state.double()
    outs = []
    for t in range(T):
        h = torch.exp(step[:, t, :, None] * A) * h + (step[:, t] * x[:, t])[..., None] * B[:, t]
        outs.append((h * C[:, t]).sum(-1))
    y = torch.stack(outs, 1) if outs else x.new_zeros(b, T, D)
    y = y if skip is None else y + skip.double() * x
    return y if z is None else y * F.silu(z.double()), h


def scan_inputs(b, T, D, N, G=1, dtype=torch.float32, seed=0, device="cuda", gate=True, skip=True, bias=True, state=True):
    """Keyword arguments of a call.  Steps of softplus from about 1e-3 to 1e-1, rates of about 1 to N: states remember up to
    about a thousand tokens."""
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=device, generator=gen)

    start = torch.exp(torch.rand(D, device=device, generator=gen) * math.log(100.0) + math.log(1e-3))
    raw = torch.log(torch.expm1(start))
    kw = dict(x=normal(b, T, D).to(dtype), dt=(0.5 * normal(b, T, D) + (0.0 if bias else raw)).to(dtype),
              A=-torch.arange(1, N + 1, device=device) * torch.exp(0.3 * normal(D, N)),
              B=normal(b, T, G, N).to(dtype), C=normal(b, T, G, N).to(dtype), dt_softplus=True)
    if skip:
        kw["skip"] = normal(D)
    if gate:
        kw["z"] = normal(b, T, D).to(dtype)
    if bias:
        kw["dt_bias"] = raw
    if state:
        kw["initial_state"] = normal(b, D, N)
    return kw


def conv(x, weight, bias=None, activation=None, initial_state=None):
    """``(out, last W - 1 inputs)`` in float64."""
    W, (b, T, D) = weight.shape[1], x.shape
    state = x.new_zeros(b, W - 1, D) if initial_state is None else initial_state
    padded = torch.cat([state.double(), x.double()], 1)
    y = sum(weight.double()[:, j] * padded[:, j:j + T] for j in range(W))
    y = y if bias is None else y + bias.double()
    return F.silu(y) if activation == "silu" else y, padded[:, T:]


def norm(x, weight, bias=None, eps=1e-5, residual=None):
    """The norm in float64, and the sum as the residual's type holds it (its rounding passes a gradient as it is)."""
    s = x.double()
    if residual is not None:
        s = s + residual.double()
        kept = residual.kept if hasattr(residual, "kept") else residual.dtype
        s = s + (s.detach().to(kept).double() - s.detach())
    c = s - s.mean(-1, keepdim=True)
    y = c / (c.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    y = y if bias is None else y + bias.double()
    return y if residual is None else (y, s)


def rel(x, y):
    """The error's 2-norm over the result's."""
    y = y.detach().double()
    return float((x.detach().double() - y.detach()).norm() / y.norm().clamp_min(1e-300))


def leaves(kw, wide=False):
    """The tensors of a call's arguments, each with a gradient of its own; ``wide``: in float64."""
    return {n: (t.detach().double() if wide else t.detach().clone()).requires_grad_(True) if isinstance(t, torch.Tensor) else t
            for n, t in kw.items()}


def tensors(kw):
    return [t for t in kw.values() if isinstance(t, torch.Tensor)]
