"""The forms that the kernels take for many sequences or rows: several channels a thread in the scan's single token, warps that
hold a row of two or four loads a lane in the norm, four sequences a thread in the convolution's single token; and inputs whose
batch rows and tokens lie further apart than 32 bits count.

Tolerances (relative 2-norm of an output's error), as each operator's own tests derive them: 1e-5 for the scan, 2e-6 for the
convolution and the norm, and half a step of 2^-7 more where an output is bf16."""
import pytest
import torch

from rnn_kernel_b200 import causal_conv, causal_conv_step, layer_norm, selective_scan, selective_step
from rnn_kernel_b200.scan import _near

from . import scan_reference as R
from .scan_reference import caller  # noqa: F401

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 0.0, BF16: 2.0 ** -8}


def close(x, y, tol, what=""):
    assert x.shape == y.shape and torch.isfinite(x).all(), what
    assert R.rel(x, y) <= tol + HALF[x.dtype], (what, R.rel(x, y))


# B, D, N, G: 1, 2, 4, 8 and 16 lanes a channel; groups of one channel to more than a thread's; channels that end inside a thread's
STEPS = [(610, 1000, 3, 1), (300, 1015, 7, 5), (152, 2000, 8, 1), (300, 1016, 8, 127), (76, 2001, 13, 3), (80, 1900, 16, 4),
         (76, 2000, 16, 2000), (40, 1900, 32, 2), (39, 1953, 20, 7), (20, 1900, 64, 1), (38, 1001, 50, 7)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", STEPS)
def test_scan_step(size, dtype):
    B, D, N, G = size
    lanes = next(n for n in (1, 2, 4, 8, 16) if 4 * n >= N)
    assert B * D * lanes // 1024 >= 4 * 148  # where a thread takes several channels
    kw = R.scan_inputs(B, 1, D, N, G, dtype=dtype, seed=B, gate=B % 3 != 0, skip=B % 2 == 0, bias=B % 5 != 0)
    state = kw.pop("initial_state")
    want, last = R.scan(**kw, initial_state=state)
    one = {n: v[:, 0] if n in ("x", "dt", "B", "C", "z") else v for n, v in kw.items()}
    close(selective_step(state=state, **one), want[:, 0], 1e-5, "out")
    close(state, last, 1e-5, "state")


# x's type, the width, the residual's and the weights' type
NORMS = [(F32, D, F32) for D in (132, 192, 256, 260, 384, 512)]
NORMS += [(BF16, D, other) for D in (136, 256, 264, 384, 512, 520, 768, 1000, 1024) for other in (BF16, F32)]


@pytest.mark.parametrize("rows", [601, 4099])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,D,other", NORMS)
def test_norm(dtype, D, other, residual, rows):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(D + rows)

    def normal(*s):
        return torch.randn(*s, device="cuda", generator=gen)

    kw = dict(x=(normal(rows, D) + normal(rows, 1)).to(dtype), weight=(1 + 0.3 * normal(D)).to(other), bias=(0.3 * normal(D)).to(other))
    if residual:
        kw["residual"] = normal(rows, D).to(other)
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    if residual:
        plain["residual"].kept = other
    outs, want = layer_norm(**mine), R.norm(**plain)
    outs, want = (o if residual else (o,) for o in (outs, want))
    close(outs[0], want[0], 2e-6, "out")
    if residual:
        assert torch.equal(outs[1], want[1].to(other))
    d = [normal(rows, D).to(o.dtype) for o in outs]
    got = torch.autograd.grad(outs, R.tensors(mine), d)
    true = torch.autograd.grad(want, R.tensors(plain), [t.double() for t in d])
    for n, a, b in zip(kw, got, true):
        close(a, b, 2e-6, n)


@pytest.mark.parametrize("size", [(228, 4000, 4), (460, 2000, 3), (230, 2000, 7), (228, 2000, 5), (229, 1001, 4), (457, 500, 8)])
def test_conv_step_fp32(size):
    B, D, W = size
    gen = torch.Generator(device="cuda")
    gen.manual_seed(W)
    x, s, w, b = (torch.randn(*n, device="cuda", generator=gen) for n in ((B, 1, D), (B, W - 1, D), (D, W), (D,)))
    w *= W ** -0.5
    want, last = R.conv(x, w, b, "silu", s)
    close(causal_conv_step(x[:, 0], w, s, b, "silu"), want[:, 0], 2e-6)
    assert torch.equal(s, last.float())


def far_scan(dtype):
    """Inputs [2, 4, ...] in one piece of memory, tokens 2^31 - 16 bytes apart, batch rows four times that: 17 GB.  And the same dense."""
    size = torch.empty((), dtype=dtype).element_size()
    token = (2 ** 31 - 16) // size
    kw = R.scan_inputs(2, 4, 40, 8, 2, dtype=dtype, seed=3)
    memory = torch.empty(7 * token + 256, dtype=dtype, device="cuda")
    far, at = dict(kw), 0
    for n in ("x", "dt", "z", "B", "C"):
        last = kw[n].shape[2:]
        far[n] = memory.as_strided(kw[n].shape, (4 * token, token, *torch.empty(last).stride()), at).copy_(kw[n])
        at += last.numel()
    return kw, far


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_of_far_tokens_and_batch_rows(dtype):
    kw, far = far_scan(dtype)
    assert all(_near(far[n]) is far[n] for n in ("x", "dt", "z", "B", "C"))  # read where they are

    def run(kw):
        mine = {n: t.detach().requires_grad_(True) if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
        outs = selective_scan(**mine)
        return (*outs, *torch.autograd.grad(outs, R.tensors(mine), [torch.ones_like(o, memory_format=torch.contiguous_format) for o in outs]))

    assert all(torch.equal(a, b) for a, b in zip(run(far), run(kw)))
    # one token of every sequence
    def one(kw):
        return {n: t[:, 3] if n in ("x", "dt", "B", "C", "z") else t for n, t in kw.items() if n != "initial_state"}

    s1, s2 = kw["initial_state"].clone(), kw["initial_state"].clone()
    assert torch.equal(selective_step(state=s1, **one(far)), selective_step(state=s2, **one(kw))) and torch.equal(s1, s2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_conv_of_far_tokens_and_batch_rows(dtype):
    _, far = far_scan(dtype)
    x, w = far["x"], torch.randn(40, 4, device="cuda")

    def run(x):
        mine, weight = x.detach().requires_grad_(True), w.clone().requires_grad_(True)
        outs = causal_conv(mine, weight, None, "silu")
        return (*outs, *torch.autograd.grad(outs, (mine, weight), [torch.ones_like(o, memory_format=torch.contiguous_format) for o in outs]))

    assert all(torch.equal(a, b) for a, b in zip(run(x), run(x.contiguous())))


def test_gate_of_negative_numbers():
    """Each value of x / (1 + e^-x) by itself: x times log2(e) rounded, 2^-24 of it, and that constant's own rounding, 1.4e-8, are
    |x| 7.4e-8 of the exponential; the hardware's exponential adds 2^-22, the sum with one 2^-24, the reciprocal 2^-23 and the
    product with x 2^-24."""
    x = -torch.linspace(0.001, 87.0, 1 << 20, device="cuda").view(1, -1, 1)
    w = torch.tensor([[0.0, 1.0]], device="cuda")
    out, _ = causal_conv(x, w, activation="silu")
    wide = x.double()
    want = wide / (1.0 + torch.exp(-wide))
    off = ((out.double() - want) / want).abs()
    assert bool((off <= wide.abs() * 7.4e-8 + 2.0 ** -22 + 2.0 ** -23 + 2.0 ** -23).all())
