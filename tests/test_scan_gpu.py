"""The selective scan's kernels against a plain 64-bit recurrence: values, gradients (the formula's and differences), lengths
from none to many blocks, odd sizes, groups, strides, padded tokens, numbers that are not finite, streams and graphs.

Tolerances (relative 2-norm of an output's error).  FP32 outputs: a token's decay is off by a few 2^-23 (its exponent's
rounding, the hardware's exponential); a state that remembers m tokens has about sqrt(m) of such errors, and m is at most
about 1000 for the inputs here: 32 * 2^-22 = 8e-6, and 1e-5 leaves room for the few 2^-24 of everything else.  bf16 outputs:
the last rounding is at most half a step of 2^-7, that is 2^-8 of each element and so of the 2-norm, on top of 1e-5."""
import pytest
import torch
import torch.utils.checkpoint

from rnn_kernel_b200 import causal_conv, layer_norm, selective_scan, selective_step

from . import scan_reference as R
from .scan_reference import caller  # noqa: F401

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8 + 1e-5}


def close(x, y, dtype, what=""):
    assert x.dtype == dtype and x.shape == y.shape and torch.isfinite(x).all(), what
    if float(y.detach().double().norm()) > 0:
        assert R.rel(x, y) <= TOL[dtype], (what, R.rel(x, y))
    else:
        assert float(x.detach().abs().max()) == 0, what


SIZES = [
    # B, T, D, N, G
    (1, 1, 1, 1, 1),
    (2, 1, 32, 16, 1),
    (1, 2, 33, 4, 1),
    (2, 15, 40, 16, 2),
    (1, 16, 64, 16, 1),
    (1, 17, 64, 3, 1),
    (3, 63, 96, 64, 3),
    (1, 64, 31, 5, 1),
    (2, 65, 32, 16, 1),
    (1, 129, 100, 16, 4),
    (2, 257, 47, 17, 1),
    (1, 1030, 64, 16, 1),
    (5, 128, 9, 1, 3),
    (1, 2100, 5, 33, 1),
    (2, 90, 130, 32, 1),
    (1, 300, 64, 24, 1),
    (2, 130, 70, 10, 2),
    (1, 700, 64, 12, 1),
    (3, 40, 66, 8, 1),
]
OPTIONS = [dict(), dict(gate=False), dict(skip=False, bias=False), dict(gate=False, skip=False, state=False)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", SIZES)
def test_values_and_gradients(size, dtype):
    kw = R.scan_inputs(*size, dtype=dtype, seed=sum(size), **OPTIONS[sum(size) % len(OPTIONS)])
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    outs, want = selective_scan(**mine), R.scan(**plain)
    close(outs[0], want[0], dtype, "out")
    close(outs[1], want[1], torch.float32, "last")
    with torch.no_grad():
        again = selective_scan(**kw)
    assert torch.equal(again[0], outs[0]) and torch.equal(again[1], outs[1])
    torch.manual_seed(1)
    grads = [torch.randn_like(o) for o in outs]
    got = torch.autograd.grad(outs, R.tensors(mine), grads)
    true = torch.autograd.grad(want, R.tensors(plain), [g.double() for g in grads])
    names = [n for n, t in kw.items() if isinstance(t, torch.Tensor)]
    for n, a, t in zip(names, got, true):
        close(a, t, kw[n].dtype, n)


@pytest.mark.parametrize("option", OPTIONS)
def test_options_together(option):
    kw = R.scan_inputs(2, 70, 36, 7, 2, seed=9, **option)
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    (o, s), (po, ps) = selective_scan(**mine), R.scan(**plain)
    close(o, po, torch.float32)
    close(s, ps, torch.float32)
    # sum() hands an expanded (stride 0) gradient back
    for a, b in zip(torch.autograd.grad(o.sum(), R.tensors(mine)), torch.autograd.grad(po.sum(), R.tensors(plain))):
        close(a, b, torch.float32)


def test_without_softplus():
    kw = R.scan_inputs(1, 90, 40, 8, seed=3, bias=False)
    kw.update(dt=torch.nn.functional.softplus(kw["dt"]), dt_softplus=False)
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    outs, want = selective_scan(**mine), R.scan(**plain)
    g = [torch.randn_like(o) for o in outs]
    for a, b in zip(torch.autograd.grad(outs, R.tensors(mine), g),
                    torch.autograd.grad(want, R.tensors(plain), [t.double() for t in g])):
        close(a, b, torch.float32)


@pytest.mark.parametrize("which", [0, 1])
def test_gradient_only_from_one_output(which):
    kw = R.scan_inputs(2, 70, 40, 6, seed=3)
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    o, r = selective_scan(**mine)[which], R.scan(**plain)[which]
    d = torch.randn_like(o)
    got = torch.autograd.grad(o, R.tensors(mine), d)
    want = torch.autograd.grad(r, R.tensors(plain), d.double(), allow_unused=True)
    for a, b in zip(got, want):
        close(a, torch.zeros_like(a) if b is None else b, torch.float32)


def test_gradient_against_differences():
    kw = R.scan_inputs(1, 67, 24, 6, 2, seed=11)
    mine = R.leaves(kw)
    outs = selective_scan(**mine)
    torch.manual_seed(2)
    ds = [torch.randn_like(o).double() for o in outs]
    grads = torch.autograd.grad(outs, R.tensors(mine), [d.float() for d in ds])
    names = [n for n, t in kw.items() if isinstance(t, torch.Tensor)]

    def loss(args):
        return float(sum((o * d).sum() for o, d in zip(R.scan(**args), ds)))

    for n, g in zip(names, grads):
        d = torch.randn_like(kw[n]).double()
        h = 1e-6  # central differences in 64 bits: errors about h^2 and 1e-16 / h relative, far below the tolerance
        wide = {k: t.double() if isinstance(t, torch.Tensor) else t for k, t in kw.items()}
        diff = (loss({**wide, n: wide[n] + h * d}) - loss({**wide, n: wide[n] - h * d})) / (2 * h)
        scale = float(g.double().norm() * d.norm())  # a projection's error is a fraction of this
        assert abs(float((g.double() * d).sum()) - diff) <= 1e-5 * scale, n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_of_fused_projections(dtype):
    b, T, D, N, G = 2, 75, 48, 6, 2
    kw = R.scan_inputs(b, T, D, N, G, dtype=dtype, seed=7)
    mine = R.leaves(kw)
    out, last = selective_scan(**mine)
    g = torch.autograd.grad((out, last), R.tensors(mine), (torch.ones_like(out), torch.ones_like(last)))
    # one element in front: nothing of it is aligned to more than an element
    wide = torch.cat([kw["x"].new_zeros(b, T, 1), kw["x"], kw["z"], kw["dt"]], -1)[..., 1:]
    x, z, dt = wide.split(D, -1)
    bc = torch.cat([kw["B"].flatten(2), kw["C"].flatten(2), kw["x"][..., :3]], -1)
    B, C = bc[..., :G * N].unflatten(-1, (G, N)), bc[..., G * N:2 * G * N].unflatten(-1, (G, N))
    strided = dict(kw, x=x, z=z, dt=dt, B=B, C=C)
    out_s, last_s = selective_scan(**strided)
    assert torch.equal(out_s, out) and torch.equal(last_s, last)
    # tokens first; a last dimension that is not dense; a transposed A
    strided = dict(kw, x=kw["x"].transpose(0, 1).contiguous().transpose(0, 1), dt=kw["dt"].transpose(1, 2).contiguous().transpose(1, 2),
                   B=kw["B"].transpose(2, 3).contiguous().transpose(2, 3), A=kw["A"].t().contiguous().t(),
                   initial_state=kw["initial_state"].transpose(1, 2).contiguous().transpose(1, 2))
    mine = {n: t.detach().requires_grad_(True) if isinstance(t, torch.Tensor) else t for n, t in strided.items()}
    out_s, last_s = selective_scan(**mine)
    assert torch.equal(out_s, out) and torch.equal(last_s, last)
    for a, c in zip(torch.autograd.grad((out_s, last_s), R.tensors(mine), (torch.ones_like(out), torch.ones_like(last))), g):
        assert torch.equal(a, c)


def test_broadcast_inputs_get_summed_gradients():
    kw = R.scan_inputs(3, 40, 32, 8, seed=4)
    one = {n: kw[n][:1].clone().requires_grad_(True) for n in ("B", "C", "dt")}
    wide = {n: kw[n][:1].double().requires_grad_(True) for n in one}
    out, _ = selective_scan(**{**kw, **{n: t.expand(3, *t.shape[1:]) for n, t in one.items()}})
    ref, _ = R.scan(**{**kw, **{n: t.expand(3, *t.shape[1:]) for n, t in wide.items()}})
    d = torch.randn_like(out)
    for a, b in zip(torch.autograd.grad(out, list(one.values()), d), torch.autograd.grad(ref, list(wide.values()), d.double())):
        close(a, b, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_behind_64_bit_offsets(dtype):
    """Rows 2^31 elements apart: offsets pass 32 bits."""
    kw = R.scan_inputs(1, 2, 40, 5, dtype=dtype, seed=5)
    want = selective_scan(**kw)
    far = torch.zeros((1 << 31) + 64, dtype=dtype, device="cuda").as_strided((1, 2, 40), (1, 1 << 31, 1))
    far.copy_(kw["x"])
    got = selective_scan(**dict(kw, x=far))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("cut", [1, 16, 63, 100])
def test_a_sequence_in_pieces_and_token_by_token(cut):
    kw = R.scan_inputs(2, 140, 50, 16, 2, seed=6)
    want, last = R.scan(**kw)

    def piece(a, b, state):
        return {**{n: t[:, a:b] if n in ("x", "dt", "B", "C", "z") else t for n, t in kw.items()}, "initial_state": state}

    o1, s = selective_scan(**piece(0, cut, kw["initial_state"]))
    o2, s2 = selective_scan(**piece(cut, 130, s))
    close(torch.cat([o1, o2], 1), want[:, :130], torch.float32)
    for t in range(130, 140):
        one = {n: v[:, 0] if n in ("x", "dt", "B", "C", "z") else v for n, v in piece(t, t + 1, None).items()}
        one.pop("initial_state")
        close(selective_step(state=s2, **one), want[:, t], torch.float32)
    close(s2, last, torch.float32)


STEPS = [(1, 1, 1, 1), (3, 40, 16, 1), (2, 33, 3, 3), (130, 100, 64, 2), (5, 64, 17, 1), (70, 2048, 16, 1), (4, 1000, 8, 4), (1, 31, 2, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", STEPS)
def test_step(size, dtype):
    b, D, N, G = size
    kw = R.scan_inputs(b, 1, D, N, G, dtype=dtype, seed=sum(size), **OPTIONS[sum(size) % 3])
    state = kw.pop("initial_state")
    want, last = R.scan(**kw, initial_state=state)
    one = {n: v[:, 0] if n in ("x", "dt", "B", "C", "z") else v for n, v in kw.items()}
    version = state._version
    out = selective_step(state=state, **one)
    assert state._version > version
    close(out, want[:, 0], dtype)
    close(state, last, torch.float32)


def test_step_strides():
    kw = R.scan_inputs(6, 1, 40, 6, 2, seed=8)
    state = kw.pop("initial_state")
    one = {n: v[:, 0] if n in ("x", "dt", "B", "C", "z") else v for n, v in kw.items()}
    s1, s2 = state.clone(), torch.zeros(6 * 40 * 6 + 1, device="cuda")[1:].view(6, 40, 6).copy_(state)  # 4-byte aligned
    both = torch.cat([one["x"], one["z"]], -1)
    out = selective_step(state=s1, **one)
    out2 = selective_step(state=s2, **dict(one, x=both[:, :40], z=both[:, 40:], B=one["B"].transpose(1, 2).contiguous().transpose(1, 2)))
    assert torch.equal(out, out2) and torch.equal(s1, s2)


def test_padding_by_a_step_of_nothing():
    """A raw step of -inf passes the state on and gets no gradient.  (Where a sequence ends, its state is the token's own;
    behind more tokens it comes from the pieces' sums, whose rounding differs: both are held to the recurrence.)"""
    kw = R.scan_inputs(2, 100, 40, 16, seed=10)
    short = {n: t[:, :53] if n in ("x", "dt", "B", "C", "z") else t for n, t in kw.items()}
    dt = kw["dt"].clone()
    dt[:, 53:] = float("-inf")
    mine = R.leaves(dict(kw, dt=dt))
    out, last = selective_scan(**mine)
    o2, l2 = selective_scan(**short)
    assert torch.equal(out[:, :53], o2)
    want = R.scan(**short)[1]
    close(last, want, torch.float32)
    close(l2, want, torch.float32)
    g = torch.autograd.grad((out[:, :53].sum(), last.sum()), [mine["x"], mine["dt"]])
    assert all(torch.isfinite(t).all() for t in g) and float(g[1][:, 53:].abs().max()) == 0


def test_decays_that_forget_everything():
    kw = R.scan_inputs(1, 70, 33, 6, seed=12)
    kw["A"][:, 0] = float("-inf")
    kw["A"][:, 1] = -1e30
    kw["A"][:, 2] = 0.0
    got = selective_scan(**kw)
    want = R.scan(**kw)
    close(got[0], want[0], torch.float32)
    close(got[1], want[1], torch.float32)


@pytest.mark.parametrize("T", [16, 17, 300, 2100])
def test_a_zero_state_stays_zero_where_it_would_grow(T):
    """A is positive here, and the product of the decays overflows; nothing enters the state before the last token, whose
    share of it is dt x B = B, without a rounding."""
    kw = R.scan_inputs(1, T, 40, 5, 1, gate=False, skip=False, bias=False, state=False)
    kw["x"].zero_()
    kw["x"][:, -1] = 1.0
    kw["dt"].fill_(1.0)
    kw["A"].fill_(20.0)
    out, last = selective_scan(**{**kw, "dt_softplus": False})
    assert torch.equal(last, kw["B"][:, -1].float().expand(1, 40, 5))
    assert float(out[:, :-1].abs().max()) == 0
    close(out[:, -1], (kw["B"].double() * kw["C"].double())[:, -1].sum(-1).expand(1, 40), torch.float32)


@pytest.mark.parametrize("name", ["x", "dt", "B", "C", "z"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_numbers_reach_no_earlier_token_and_no_other_sequence(name, bad):
    kw = R.scan_inputs(2, 150, 40, 8, seed=13)
    clean = selective_scan(**kw)
    t = kw[name].clone()
    t[1, 81] = bad
    out, last = selective_scan(**dict(kw, **{name: t}))
    assert torch.equal(out[0], clean[0][0]) and torch.equal(out[1, :81], clean[0][1, :81])
    assert torch.equal(last[0], clean[1][0])
    assert not torch.equal(out[1, 81], clean[0][1, 81])
    if name in ("x", "z"):  # nor another channel
        t = kw[name].clone()
        t[1, 81, 7] = bad
        out, last = selective_scan(**dict(kw, **{name: t}))
        rest = torch.arange(40, device="cuda") != 7
        assert torch.equal(out[:, :, rest], clean[0][:, :, rest]) and torch.equal(last[:, rest], clean[1][:, rest])


def test_nothing_to_do():
    for b, T in ((0, 5), (3, 0), (0, 0)):
        kw = R.scan_inputs(b, T, 16, 4, seed=1)
        mine = R.leaves(kw)
        out, last = selective_scan(**mine)
        assert out.shape == (b, T, 16) and torch.equal(last, kw["initial_state"])
        g = torch.autograd.grad((out, last), R.tensors(mine), (torch.ones_like(out), torch.ones_like(last)))
        for t, d in zip(R.tensors(kw), g):
            assert d.shape == t.shape
        assert torch.equal(g[-1], torch.ones_like(last)) and float(g[2].abs().sum()) == 0
        kw.pop("initial_state")
        assert float(selective_scan(**kw)[1].abs().sum()) == 0
    kw = R.scan_inputs(0, 1, 16, 4, seed=1)
    one = {n: v[:, 0] if n in ("x", "dt", "B", "C", "z") else v for n, v in kw.items() if n != "initial_state"}
    assert selective_step(state=kw["initial_state"], **one).shape == (0, 16)


def test_same_results_every_time_and_alone():
    kw = R.scan_inputs(3, 200, 70, 16, seed=14)
    runs = []
    for _ in range(2):
        mine = R.leaves(kw)
        outs = selective_scan(**mine)
        runs.append((*outs, *torch.autograd.grad(outs, R.tensors(mine), [torch.ones_like(o) for o in outs])))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    alone, _ = selective_scan(**{n: t[1:2] if n in ("x", "dt", "B", "C", "z", "initial_state") else t for n, t in kw.items()})
    assert torch.equal(alone[0], runs[0][0][1])


def test_second_derivatives_and_tangents_raise():
    kw = R.scan_inputs(1, 5, 8, 4)
    mine = R.leaves(kw)
    out, _ = selective_scan(**mine)
    g, = torch.autograd.grad(out.sum(), mine["x"], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(kw["x"], torch.ones_like(kw["x"]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            selective_scan(**dict(kw, x=dual))
        one = {n: v[:, 0] if n in ("x", "dt", "B", "C", "z") else v for n, v in kw.items() if n != "initial_state"}
        with pytest.raises(RuntimeError, match="derivative"):
            selective_step(state=kw["initial_state"], **dict(one, x=dual[:, 0]))


def test_streams_and_graphs():
    """Two graphs captured one after another, replayed on new inputs, on a stream of their own, beside eager calls."""
    sets = [R.scan_inputs(2, 150, 64, 16, seed=s) for s in (20, 21, 22)]
    want = []
    for kw in sets:
        mine = R.leaves(kw)
        outs = selective_scan(**mine)
        want.append((*outs, *torch.autograd.grad(outs, R.tensors(mine), [torch.ones_like(o) for o in outs])))
    stream = torch.cuda.Stream()
    graphs = []
    for kw in sets[:2]:
        mine = R.leaves(kw)
        graph = torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            outs = selective_scan(**mine)
            got = (*outs, *torch.autograd.grad(outs, R.tensors(mine), [torch.ones_like(o) for o in outs]))
        graphs.append((graph, mine, got))
    for graph, mine, got in graphs:
        with torch.no_grad():
            for n, t in sets[2].items():
                if isinstance(t, torch.Tensor):
                    mine[n].copy_(t)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for graph, _, _ in graphs:
            graph.replay()
        eager = selective_scan(**sets[0])
    torch.cuda.synchronize()
    for _, _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(got, want[2]))
    assert torch.equal(eager[0], want[0][0])


def test_saved_tensors_through_hooks_and_checkpoints():
    kw = R.scan_inputs(2, 70, 64, 16, 2, seed=30)
    w, b = torch.randn(2, 64, device="cuda")
    cw = torch.randn(64, 4, device="cuda")

    def run(x, A, cw, w):
        y, s = layer_norm(x, w, b, residual=x)
        u, _ = causal_conv(y, cw, None, "silu")
        return selective_scan(**{**kw, "x": u, "A": A})[0] + s

    def grads(how):
        leaves = [t.clone().requires_grad_() for t in (kw["x"], kw["A"], cw, w)]
        out = how(*leaves)
        return (out, *torch.autograd.grad(out, leaves, torch.ones_like(out)))

    want = grads(run)
    with torch.autograd.graph.save_on_cpu():
        kept = grads(run)
    again = grads(lambda *t: torch.utils.checkpoint.checkpoint(run, *t, use_reentrant=False))
    for got in (kept, again):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    kw = R.scan_inputs(2, 6, 8, 4, 2)
    one = {n: v[:, 0] if n in ("x", "dt", "B", "C", "z") else v for n, v in kw.items() if n != "initial_state"}
    s = kw["initial_state"]
    for bad, error in ((dict(x=kw["x"].half()), RuntimeError), (dict(dt=kw["dt"].bfloat16()), RuntimeError),
                       (dict(A=kw["A"].double()), RuntimeError), (dict(initial_state=s.bfloat16()), RuntimeError),
                       (dict(skip=kw["skip"].bfloat16()), RuntimeError), (dict(B=kw["B"].cpu()), ValueError),
                       (dict(A=kw["A"][:, :3]), ValueError), (dict(z=kw["z"][:, :5]), ValueError)):
        with pytest.raises(error):
            selective_scan(**{**kw, **bad})
    with pytest.raises(ValueError, match="contiguous"):
        selective_step(state=s.transpose(1, 2).contiguous().transpose(1, 2), **one)
    with pytest.raises(RuntimeError):
        selective_step(state=s.bfloat16(), **one)
    # numbers that torch would negate when it reads them
    for call in (lambda: selective_scan(**{**kw, "x": torch._neg_view(kw["x"])}), lambda: selective_step(state=torch._neg_view(s), **one),
                 lambda: causal_conv(torch._neg_view(kw["x"]), torch.ones(8, 4, device="cuda")),
                 lambda: layer_norm(torch._neg_view(kw["x"]), torch.ones(8, device="cuda"))):
        with pytest.raises(RuntimeError, match="negation"):
            call()
