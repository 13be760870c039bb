"""Layer norm's kernels against a plain 64-bit form: widths around every way to deal out a row, types, residuals, strides,
rows with large offsets, gradients.

Tolerances (relative 2-norm).  FP32 outputs: a mean and a variance of up to 16384 terms as a tree of sums of at most 32 terms
a thread, a few 2^-24 together; each output some five roundings more: 2e-6 (34 * 2^-24).  The input's gradient takes means
away from terms of their size, which costs up to ten times that where a row has few elements: 2e-5 below a width of 16.
bf16 outputs: the last rounding is at most half a step of 2^-7, that is 2^-8 of each element and so of the 2-norm, on top of 2e-6."""
import pytest
import torch

from rnn_kernel_b200 import LayerNorm, layer_norm

from . import scan_reference as R
from .scan_reference import caller  # noqa: F401

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-6, torch.bfloat16: 2.0 ** -8 + 2e-6}
F32, BF16 = torch.float32, torch.bfloat16


def close(x, y, dtype, what="", times=1.0):
    assert x.dtype == dtype and x.shape == y.shape and torch.isfinite(x).all(), what
    assert R.rel(x, y) <= times * TOL[dtype], (what, R.rel(x, y))


def inputs(shape, dtype, wtype, kept, seed=0, bias=True):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, device="cuda", generator=gen)

    D = shape[-1]
    kw = dict(x=(normal(*shape) + normal(*shape[:-1], 1)).to(dtype), weight=(1 + 0.3 * normal(D)).to(wtype))
    if bias:
        kw["bias"] = (0.3 * normal(D)).to(wtype)
    if kept is not None:
        kw["residual"] = normal(*shape).to(kept)
    return kw


def reference(kw, **more):
    plain = R.leaves(kw, wide=True)
    args = dict(plain)
    if "residual" in args:
        args["residual"].kept = kw["residual"].dtype
    return plain, R.norm(**args, **more)


def both(o):
    return o if isinstance(o, tuple) else (o,)


WIDTHS = [8, 16, 24, 31, 32, 64, 100, 255, 256, 257, 512, 516, 768, 1000, 1024, 1032, 2048, 2056, 4096, 4100, 8192, 8193, 12288, 16384, 16383]
TYPES = [(F32, F32, None), (F32, F32, F32), (BF16, BF16, None), (BF16, F32, BF16), (BF16, F32, F32), (BF16, BF16, BF16)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_values_and_gradients(D, types):
    rows = 1 + D % 7 if D > 4000 else 37
    kw = inputs((rows, D), *types, seed=D, bias=D % 3 != 0)
    mine = R.leaves(kw)
    plain, want = reference(kw)
    outs, want = both(layer_norm(**mine)), both(want)
    close(outs[0], want[0], types[0], "out")
    if types[2] is not None:
        assert torch.equal(outs[1], want[1].to(types[2]))
    with torch.no_grad():
        again = both(layer_norm(**kw))
    assert all(torch.equal(a, b) for a, b in zip(again, outs))
    torch.manual_seed(1)
    grads = [torch.randn_like(o) for o in outs]
    got = torch.autograd.grad(outs, R.tensors(mine), grads)
    true = torch.autograd.grad(want, R.tensors(plain), [g.double() for g in grads])
    for n, a, t in zip(kw, got, true):
        close(a, t, kw[n].dtype, n, times=10.0 if D < 16 and kw[n].dtype == F32 else 1.0)


@pytest.mark.parametrize("D", [1, 2, 3, 5])
def test_few_elements(D):
    """The input's gradient all but vanishes here: errors against the terms that cancel, of the size of rstd |dy w|."""
    kw = inputs((50, D), F32, F32, None, seed=D)
    mine = R.leaves(kw)
    plain, want = reference(kw)
    out = layer_norm(**mine)
    # rstd is up to eps^-1/2 = 316 and multiplies the mean's rounding
    assert float((out - want).detach().abs().max()) <= 316 * 8 * 2.0 ** -24 * float(kw["x"].abs().max() + 1)
    d = torch.randn_like(out)
    got = torch.autograd.grad(out, R.tensors(mine), d)
    true = torch.autograd.grad(want, R.tensors(plain), d.double())
    s = kw["x"].double()
    rstd = (s.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    size = rstd * (d * kw["weight"]).abs().amax(-1, keepdim=True) * (1 + rstd * s.abs().amax(-1, keepdim=True))
    assert bool(((got[0] - true[0]).abs() <= 40 * 2.0 ** -24 * size).all())


def test_a_row_of_one_value_and_large_offsets():
    x = torch.full((3, 256), 7.25, device="cuda")
    x[1] = 0
    w, b = torch.randn(256, device="cuda"), torch.randn(256, device="cuda")
    assert torch.equal(layer_norm(x, w, b), b.expand(3, 256))
    # an offset of 2^12 times the spread costs the 12 bits that x has lost already, no more
    x = torch.randn(5, 640, device="cuda") + 4096.0
    assert R.rel(layer_norm(x, w.repeat(3)[:640]), R.norm(x, w.repeat(3)[:640])) < 2 ** 12 * 2.0 ** -24


def test_shapes_strides_and_offsets():
    kw = inputs((2, 3, 5, 64), F32, F32, F32, seed=3)
    out, s = layer_norm(**kw)
    flat = layer_norm(kw["x"].reshape(-1, 64), kw["weight"], kw["bias"], residual=kw["residual"].reshape(-1, 64))
    assert out.shape == kw["x"].shape and torch.equal(out.view(-1, 64), flat[0]) and torch.equal(s.view(-1, 64), flat[1])
    x, r = kw["x"].reshape(-1, 64), kw["residual"].reshape(-1, 64)
    wide = torch.cat([x.new_zeros(30, 1), x, r], -1)
    for a, b in ((wide[:, 1:65], wide[:, 65:]), (torch.cat([x, r], -1)[:, :64], r), (x.t().contiguous().t(), r), (x, r.t().contiguous().t())):
        mine = dict(x=a.detach().requires_grad_(True), residual=b.detach().requires_grad_(True), weight=kw["weight"], bias=kw["bias"])
        got = layer_norm(**mine)
        assert R.rel(got[0], flat[0]) <= TOL[F32] and torch.equal(got[1], flat[1])
        g = torch.autograd.grad(got[0].sum(), (mine["x"], mine["residual"]))
        assert torch.equal(g[0], g[1])
    one = layer_norm(x[0], kw["weight"])
    assert one.shape == (64,) and R.rel(one, R.norm(x[0], kw["weight"])) <= TOL[F32]
    far = torch.zeros((1 << 31) + 64, dtype=BF16, device="cuda").as_strided((2, 64), (1 << 31, 1))
    far.copy_(x[:2])
    assert torch.equal(layer_norm(far, kw["weight"]), layer_norm(x[:2].bfloat16(), kw["weight"]))


@pytest.mark.parametrize("rows", [1, 2, 591, 593, 5000])
@pytest.mark.parametrize("D", [40, 640, 1280])
def test_many_rows(rows, D):
    kw = inputs((rows, D), F32, F32, F32, seed=rows)
    mine = R.leaves(kw)
    plain, want = reference(kw)
    outs = layer_norm(**mine)
    grads = [torch.randn_like(o) for o in outs]
    got = torch.autograd.grad(outs, R.tensors(mine), grads)
    for n, a, t in zip(kw, got, torch.autograd.grad(want, R.tensors(plain), [g.double() for g in grads])):
        close(a, t, F32, n)


def test_gradient_only_from_one_output_and_none():
    kw = inputs((20, 96), BF16, F32, F32, seed=5)
    for which in (0, 1):
        mine = R.leaves(kw)
        plain, want = reference(kw)
        o = layer_norm(**mine)[which]
        d = torch.randn_like(o)
        got = torch.autograd.grad(o, R.tensors(mine), d)
        true = torch.autograd.grad(want[which], R.tensors(plain), d.double(), allow_unused=True)
        for n, a, t in zip(kw, got, true):
            if t is None or float(t.norm()) == 0:
                assert float(a.abs().max()) == 0
            else:
                close(a, t, kw[n].dtype, n)


def test_gradient_against_differences():
    kw = inputs((7, 48), F32, F32, F32, seed=6)
    mine = R.leaves(kw)
    outs = layer_norm(**mine)
    ds = [torch.randn_like(o).double() for o in outs]
    grads = torch.autograd.grad(outs, R.tensors(mine), [d.float() for d in ds])

    def loss(args):
        s = args["x"] + args["residual"]  # without the sum's rounding, 2^-24 of it
        c = s - s.mean(-1, keepdim=True)
        y = c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * args["weight"] + args["bias"]
        return float((y * ds[0]).sum() + (s * ds[1]).sum())

    for n, g in zip(kw, grads):
        d, h = torch.randn_like(kw[n]).double(), 1e-6
        wide = {k: t.double() for k, t in kw.items()}
        diff = (loss({**wide, n: wide[n] + h * d}) - loss({**wide, n: wide[n] - h * d})) / (2 * h)
        assert abs(float((g.double() * d).sum()) - diff) <= 2e-6 * float(g.double().norm() * d.norm()), n


def test_bad_numbers_stay_in_their_row():
    kw = inputs((9, 300), F32, F32, None, seed=7)
    clean = layer_norm(**kw)
    for bad in (float("nan"), float("inf")):
        x = kw["x"].clone()
        x[4, 17] = bad
        out = layer_norm(**dict(kw, x=x))
        rest = torch.arange(9, device="cuda") != 4
        assert torch.equal(out[rest], clean[rest]) and not torch.isfinite(out[4]).any()


def test_nothing_to_do_refusals_and_second_derivatives():
    kw = inputs((0, 32), F32, F32, F32)
    mine = R.leaves(kw)
    outs = layer_norm(**mine)
    g = torch.autograd.grad(outs, R.tensors(mine), [torch.ones_like(o) for o in outs])
    assert outs[0].shape == (0, 32) and float(g[1].abs().sum()) == 0 == float(g[2].abs().sum())
    kw = inputs((4, 32), BF16, F32, F32)
    for bad, error in ((dict(x=kw["x"].half()), RuntimeError), (dict(weight=kw["weight"].half()), RuntimeError),
                       (dict(bias=kw["bias"].bfloat16()), RuntimeError), (dict(residual=kw["residual"].half()), RuntimeError),
                       (dict(residual=kw["residual"][:3]), ValueError), (dict(weight=kw["weight"][:31]), ValueError),
                       (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError), (dict(weight=kw["weight"].cpu()), ValueError)):
        with pytest.raises(error):
            layer_norm(**{**kw, **bad})
    with pytest.raises(RuntimeError):
        layer_norm(kw["x"].float(), kw["weight"], kw["bias"], residual=kw["residual"].bfloat16())
    mine = R.leaves(kw)
    g, = torch.autograd.grad(layer_norm(**mine)[0].sum(), mine["x"], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.float().sum().backward()


def test_graph_replay_and_determinism():
    kw, new = inputs((700, 512), F32, F32, F32, seed=1), inputs((700, 512), F32, F32, F32, seed=2)

    def run(mine):
        outs = layer_norm(**mine)
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
            mine[n].copy_(t)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_module():
    m = LayerNorm(40).cuda()
    x = torch.randn(3, 40, device="cuda")
    assert R.rel(m(x), R.norm(x, m.weight, m.bias)) <= TOL[F32]
    y, s = m(x, x)
    assert torch.equal(s, x + x) and R.rel(y, R.norm(2 * x, m.weight, m.bias)) <= TOL[F32]
    assert LayerNorm(8, bias=False).bias is None
