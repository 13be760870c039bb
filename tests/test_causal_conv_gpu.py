"""The causal convolution's kernels against a plain 64-bit form: every width, lengths around the runs that threads take, odd
channels, strides, states, gradients and the single token.

Tolerances (relative 2-norm).  FP32 outputs: a sum of at most 8 products (4e-7 at the worst), the sigmoid (2^-21), and for the
weights' gradients FP32 sums over at most 512 tokens, then over 8 of those sums, before FP64 ones (an error of 2^-25 of the
sum so far at each, which average out to 256^0.5 2^-25 = 5e-7): 2e-6.  bf16 outputs: the last rounding is at
most half a step of 2^-7, that is 2^-8 of each element and so of the 2-norm, on top of 2e-6."""
import pytest
import torch

from rnn_kernel_b200 import causal_conv, causal_conv_step

from . import scan_reference as R
from .scan_reference import caller  # noqa: F401

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.0 ** -8 + 2e-6}


def close(x, y, dtype, what=""):
    assert x.dtype == dtype and x.shape == y.shape and torch.isfinite(x).all(), what
    if float(y.detach().double().norm()) > 0:
        assert R.rel(x, y) <= TOL[dtype], (what, R.rel(x, y))
    else:
        assert x.numel() == 0 or float(x.abs().max()) == 0, what


def inputs(b, T, D, W, dtype=torch.float32, wtype=torch.float32, seed=0, bias=True, state=True, activation="silu"):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    kw = dict(x=normal(b, T, D).to(dtype), weight=(W ** -0.5 * normal(D, W)).to(wtype), activation=activation)
    if bias:
        kw["bias"] = (0.5 * normal(D)).to(wtype)
    if state:
        kw["initial_state"] = normal(b, W - 1, D).to(dtype)
    return kw


SIZES = [
    # B, T, D, W
    (1, 1, 1, 2),
    (2, 1, 4, 4),
    (1, 2, 33, 4),
    (2, 3, 128, 8),
    (3, 7, 12, 5),
    (1, 31, 130, 3),
    (2, 32, 256, 4),
    (1, 33, 64, 7),
    (2, 255, 36, 4),
    (1, 256, 20, 6),
    (2, 300, 129, 2),
    (1, 1000, 8, 4),
]


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("size", SIZES)
def test_values_and_gradients(size, types):
    k = sum(size)
    kw = inputs(*size, *types, seed=k, bias=k % 3 != 0, state=k % 4 != 0, activation="silu" if k % 2 else None)
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    outs, want = causal_conv(**mine), R.conv(**plain)
    close(outs[0], want[0], types[0], "out")
    assert torch.equal(outs[1], want[1].to(types[0]))
    torch.manual_seed(1)
    grads = [torch.randn_like(o) for o in outs]
    got = torch.autograd.grad(outs, R.tensors(mine), grads)
    true = torch.autograd.grad(want, R.tensors(plain), [g.double() for g in grads])
    for n, a, t in zip([n for n, t in kw.items() if isinstance(t, torch.Tensor)], got, true):
        close(a, t, kw[n].dtype, n)


@pytest.mark.parametrize("size", [(1, 1100, 18944, 4), (2, 700, 9001, 3), (1, 900, 9472, 8)])
def test_values_and_gradients_with_long_runs(size):
    """Channels enough to fill the GPU, so that a thread takes many turns."""
    kw = inputs(*size, seed=sum(size))
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    outs, want = causal_conv(**mine), R.conv(**plain)
    close(outs[0], want[0], torch.float32, "out")
    assert torch.equal(outs[1], want[1].float())
    grads = [torch.randn_like(o) for o in outs]
    got = torch.autograd.grad(outs, R.tensors(mine), grads)
    true = torch.autograd.grad(want, R.tensors(plain), [g.double() for g in grads])
    for n, a, t in zip([n for n, t in kw.items() if isinstance(t, torch.Tensor)], got, true):
        close(a, t, torch.float32, n)


@pytest.mark.parametrize("size", [(225, 4096, 4), (229, 1001, 5), (230, 2048, 8)])
def test_a_step_of_many_sequences(size):
    B, D, W = size
    kw = inputs(B, 1, D, W, torch.bfloat16, seed=B)
    state = kw.pop("initial_state")
    want, last = R.conv(initial_state=state, **kw)
    x = kw.pop("x")
    close(causal_conv_step(x[:, 0], state=state, **kw), want[:, 0], torch.bfloat16)
    assert torch.equal(state, last.to(torch.bfloat16))


@pytest.mark.parametrize("W", range(2, 9))
def test_every_width_in_pieces_and_token_by_token(W):
    kw = inputs(2, 60, 24, W, seed=W)
    x, s = kw.pop("x"), kw.pop("initial_state")
    want, last = R.conv(x, initial_state=s, **kw)
    outs = []
    for a, b in ((0, 1), (1, 3), (3, 40)):
        o, s = causal_conv(x[:, a:b], initial_state=s, **kw)
        outs.append(o)
    for t in range(40, 60):
        version = s._version
        outs.append(causal_conv_step(x[:, t], state=s, **kw)[:, None])
        assert s._version > version
    close(torch.cat(outs, 1), want, torch.float32)
    assert torch.equal(s, last.float())


@pytest.mark.parametrize("which", [0, 1])
def test_gradient_only_from_one_output(which):
    kw = inputs(2, 50, 40, 4, seed=3)
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    o, r = causal_conv(**mine)[which], R.conv(**plain)[which]
    d = torch.randn_like(o)
    got = torch.autograd.grad(o, R.tensors(mine), d)
    want = torch.autograd.grad(r, R.tensors(plain), d.double(), allow_unused=True)
    for a, b in zip(got, want):
        close(a, torch.zeros_like(a) if b is None else b, torch.float32)


def test_gradient_against_differences():
    kw = inputs(1, 37, 12, 4, seed=11)
    mine = R.leaves(kw)
    outs = causal_conv(**mine)
    ds = [torch.randn_like(o).double() for o in outs]
    grads = torch.autograd.grad(outs, R.tensors(mine), [d.float() for d in ds])

    def loss(args):
        return float(sum((o * d).sum() for o, d in zip(R.conv(**args), ds)))

    for n, g in zip([n for n, t in kw.items() if isinstance(t, torch.Tensor)], grads):
        d, h = torch.randn_like(kw[n]).double(), 1e-6
        wide = {k: t.double() if isinstance(t, torch.Tensor) else t for k, t in kw.items()}
        diff = (loss({**wide, n: wide[n] + h * d}) - loss({**wide, n: wide[n] - h * d})) / (2 * h)
        assert abs(float((g.double() * d).sum()) - diff) <= 2e-6 * float(g.double().norm() * d.norm()), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    kw = inputs(2, 45, 32, 4, dtype, seed=7)
    want = causal_conv(**kw)
    x = kw["x"]
    wide = torch.cat([x.new_zeros(2, 45, 1), x, x], -1)
    forms = [wide[..., 1:33], wide[..., 33:], x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(1, 2).contiguous().transpose(1, 2),
             torch.cat([x, x], -1)[..., :32]]
    for form in forms:
        mine = R.leaves(kw)
        mine["x"] = form.detach().requires_grad_(True)
        got = causal_conv(**mine)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        g, = torch.autograd.grad(got[0].sum(), mine["x"])
        plain = R.leaves(kw, wide=True)
        close(g, torch.autograd.grad(R.conv(**plain)[0].sum(), plain["x"])[0], dtype)
    s = kw["initial_state"]
    one = dict(weight=kw["weight"], bias=kw["bias"], activation="silu")
    a, b = s.clone(), torch.zeros(s.numel() + 1, dtype=dtype, device="cuda")[1:].view(s.shape).copy_(s)
    assert torch.equal(causal_conv_step(x[:, 0], state=a, **one), causal_conv_step(wide[:, 0, 1:33], state=b, **one))
    assert torch.equal(a, b)
    far = torch.zeros((1 << 31) + 64, dtype=dtype, device="cuda").as_strided((2, 1, 32), (1 << 31, 32, 1))
    far.copy_(x[:, :1])
    assert torch.equal(causal_conv(**dict(kw, x=far))[0], causal_conv(**dict(kw, x=x[:, :1]))[0])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_numbers_reach_their_window_alone(bad):
    kw = inputs(2, 80, 20, 4, seed=5)
    mine = R.leaves(kw)
    clean, _ = causal_conv(**mine)
    grads = torch.autograd.grad(clean.sum(), mine["x"])[0]
    x = kw["x"].clone()
    x[1, 33, 6] = bad
    mine = R.leaves(dict(kw, x=x))
    out, _ = causal_conv(**mine)
    ok = torch.ones_like(x, dtype=torch.bool)
    ok[1, 33:37, 6] = False
    assert torch.equal(out[ok], clean[ok])
    g = torch.autograd.grad(out.sum(), mine["x"])[0]
    ok[1, 30:37, 6] = False
    assert torch.equal(g[ok], grads[ok])


def test_large_activations():
    """silu far out: x above, zero below."""
    x = torch.tensor([[[1e30, -1e30, 200.0, -200.0, 90.0, -90.0]]], device="cuda")
    w = torch.tensor([[0.0, 1.0]], device="cuda").expand(6, 2)
    mine = x.clone().requires_grad_(True)
    out, _ = causal_conv(mine, w, activation="silu")
    assert torch.equal(out.detach().relu(), x.relu()) and float(out.detach().clamp(max=0).abs().max()) < 1e-30
    g, = torch.autograd.grad(out.sum(), mine)
    assert torch.allclose(g, (x > 0).float(), atol=1e-30)


def test_nothing_to_do_and_refusals():
    for b, T in ((0, 5), (3, 0), (0, 0)):
        kw = inputs(b, T, 16, 4)
        mine = R.leaves(kw)
        out, last = causal_conv(**mine)
        assert out.shape == (b, T, 16) and torch.equal(last, kw["initial_state"])
        g = torch.autograd.grad((out, last), R.tensors(mine), (torch.ones_like(out), torch.ones_like(last)))
        assert float(g[1].abs().sum()) == 0 and torch.equal(g[3], torch.ones_like(last))
        kw.pop("initial_state")
        assert float(causal_conv(**kw)[1].abs().sum()) == 0
    kw = inputs(2, 5, 16, 4)
    for bad, error in ((dict(x=kw["x"].half()), RuntimeError), (dict(weight=kw["weight"].bfloat16()), RuntimeError),
                       (dict(bias=kw["bias"].bfloat16()), RuntimeError), (dict(initial_state=kw["initial_state"].bfloat16()), RuntimeError),
                       (dict(weight=kw["weight"].cpu()), ValueError), (dict(activation="relu"), ValueError)):
        with pytest.raises(error):
            causal_conv(**{**kw, **bad})
    with pytest.raises(ValueError, match="contiguous"):
        causal_conv_step(kw["x"][:, 0], kw["weight"], kw["initial_state"].transpose(1, 2).contiguous().transpose(1, 2))
    mine = R.leaves(kw)
    g, = torch.autograd.grad(causal_conv(**mine)[0].sum(), mine["x"], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


def test_graph_replay_and_determinism():
    kw, new = inputs(2, 300, 64, 4, seed=1), inputs(2, 300, 64, 4, seed=2)

    def run(mine):
        outs = causal_conv(**mine)
        return (*outs, *torch.autograd.grad(outs, R.tensors(mine), [torch.ones_like(o) for o in outs]))

    want = run(R.leaves(new))
    assert all(torch.equal(a, b) for a, b in zip(run(R.leaves(new)), want))
    mine = R.leaves(kw)
    run(mine)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(mine)
    with torch.no_grad():
        for n, t in new.items():
            if isinstance(t, torch.Tensor):
                mine[n].copy_(t)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
