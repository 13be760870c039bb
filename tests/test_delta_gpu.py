"""The gated delta rule's kernels against a plain 64-bit recurrence: values, gradients (the formula's and differences),
sizes from one token to many chunks, odd head sizes, shared heads, strides, decays that forget everything, and refusals.

Tolerances (relative 2-norm of an output's error).  FP32 outputs: operands reach the tensor cores as planes with a
residue below 2^-22 of an element, mostly far below, and sums are FP32; a chunk's result passes about six products of
up to 128 terms one after another, each with a rounding or truncation error of a few 2^-24, and decays keep chunks from
piling up: 2e-6 is some thirty 2^-24.  bf16 outputs: rounding to 8 bits alone is at most 2^-9 relative and 2^-9 / sqrt(3) in the 2-norm where values
spread evenly over a binade (0.0017); 3e-3 allows for it and the 2^-18 of two planes."""
import pytest
import torch

from rnn_kernel_b200 import GatedDelta, gated_delta_rule, gated_delta_step

from . import delta_reference as R

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "g", "beta", "state")
TOL = {torch.float32: 2e-6, torch.bfloat16: 3e-3}


def rel(x, y):
    y = y.double()
    return float((x.double() - y).norm() / y.norm().clamp_min(1e-300))


def close(x, y, dtype):
    assert x.dtype == dtype and torch.isfinite(x).all()
    assert rel(x, y) <= TOL[dtype], rel(x, y)


def with_grad(tensors):
    return [t.detach().clone().requires_grad_(True) for t in tensors]


SIZES = [
    # B, T, Hk, Hv, dk, dv
    (1, 1, 1, 1, 1, 1),
    (2, 1, 1, 2, 64, 64),
    (1, 2, 1, 1, 128, 128),
    (2, 63, 2, 2, 64, 32),
    (1, 64, 1, 3, 65, 33),
    (1, 65, 2, 4, 128, 128),
    (3, 130, 1, 1, 17, 127),
    (2, 200, 2, 6, 40, 72),
    (1, 513, 1, 2, 128, 96),
    (5, 128, 3, 3, 127, 1),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", SIZES)
def test_values_and_gradients(size, dtype):
    x = R.inputs(*size, dtype=dtype, seed=sum(size))
    mine, plain = with_grad(x), with_grad([t.double() for t in x])
    out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
    out_r, last_r = R.rule(*plain)
    close(out, out_r, dtype)
    close(last, last_r, torch.float32)
    torch.manual_seed(1)
    do, ds = torch.randn_like(out), torch.randn_like(last)
    got = torch.autograd.grad((out, last), mine, (do, ds))
    want = torch.autograd.grad((out_r, last_r), plain, (do.double(), ds.double()))
    for name, a, b, t in zip(NAMES, got, want, x):
        assert a.shape == t.shape, name
        if float(b.norm()) > 0:
            close(a, b, t.dtype)


@pytest.mark.parametrize("size", [(2, 70, 1, 2, 64, 48), (1, 129, 2, 2, 128, 64)])
def test_gradient_only_from_one_output(size):
    x = R.inputs(*size, seed=3)
    for which in (0, 1):
        mine, plain = with_grad(x), with_grad([t.double() for t in x])
        o, r = gated_delta_rule(*mine[:5], initial_state=mine[5])[which], R.rule(*plain)[which]
        d = torch.randn_like(o)
        # which = 1: q takes no part
        got = torch.autograd.grad(o, mine, d)
        want = torch.autograd.grad(r, plain, d.double(), allow_unused=True)
        for a, b in zip(got, want):
            if b is None or float(b.norm()) == 0:
                assert float(a.abs().max()) == 0
            else:
                close(a, b, a.dtype)


def test_no_initial_state_and_broadcast_gradient():
    q, k, v, g, beta, _ = R.inputs(2, 100, 1, 2, 64, 64, seed=5)
    mine, plain = with_grad((q, k, v, g, beta)), with_grad([t.double() for t in (q, k, v, g, beta)])
    out, last = gated_delta_rule(*mine, scale=0.3)
    out_r, last_r = R.rule(*plain, scale=0.3)
    close(out, out_r, torch.float32)
    close(last, last_r, torch.float32)
    # sum() hands an expanded (stride 0) gradient back
    for a, b in zip(torch.autograd.grad(out.sum(), mine), torch.autograd.grad(out_r.sum(), plain)):
        close(a, b, torch.float32)


def test_gradient_against_differences():
    x = [t for t in R.inputs(1, 67, 1, 2, 24, 16, seed=11)]
    mine = with_grad(x)
    out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
    torch.manual_seed(2)
    do, ds = torch.randn_like(out).double(), torch.randn_like(last).double()
    grads = torch.autograd.grad((out, last), mine, (do.float(), ds.float()))

    def loss(xs):
        o, s = R.rule(*xs)
        return float((o * do).sum() + (s * ds).sum())

    for i, name in enumerate(NAMES):
        d = torch.randn_like(x[i]).double()
        h = 1e-5  # central differences in 64 bits: error about h^2 relative, far below the tolerance
        wide = [t.double() for t in x]
        up, down = list(wide), list(wide)
        up[i], down[i] = wide[i] + h * d, wide[i] - h * d
        diff = (loss(up) - loss(down)) / (2 * h)
        along = float((grads[i].double() * d).sum())
        scale = float(grads[i].double().norm() * d.norm())  # a projection's error is a fraction of this
        assert abs(along - diff) <= 2e-6 * scale, name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_of_a_fused_projection(dtype):
    B, T, Hk, Hv, dk, dv = 2, 75, 2, 4, 32, 48
    q, k, v, g, beta, s = R.inputs(B, T, Hk, Hv, dk, dv, dtype=dtype, seed=7)
    both = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], dim=-1)
    # one element in front: nothing of it is aligned to more than an element
    both = torch.cat([both.new_zeros(B, T, 1), both], dim=-1)[..., 1:]
    qs, ks, vs = both.split((Hk * dk, Hk * dk, Hv * dv), dim=-1)
    qs, ks, vs = qs.unflatten(-1, (Hk, dk)), ks.unflatten(-1, (Hk, dk)), vs.unflatten(-1, (Hv, dv))
    gs = torch.stack([beta, g], dim=-1)
    out, last = gated_delta_rule(qs, ks, vs, gs[..., 1], gs[..., 0], initial_state=s)
    out_c, last_c = gated_delta_rule(q, k, v, g, beta, initial_state=s)
    assert torch.equal(out, out_c) and torch.equal(last, last_c)
    # heads first, and a last dimension that is not dense
    out_t, last_t = gated_delta_rule(q.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(2, 3).contiguous().transpose(2, 3),
                                     v, g.transpose(1, 2).contiguous().transpose(1, 2), beta, initial_state=s)
    assert torch.equal(out_t, out_c) and torch.equal(last_t, last_c)


def test_strides_gradients():
    q, k, v, g, beta, s = R.inputs(2, 75, 2, 4, 32, 48, seed=8)
    want = with_grad((q, k, v, g, beta, s))
    a = gated_delta_rule(*want[:5], initial_state=want[5])
    do = torch.randn_like(a[0])
    wg = torch.autograd.grad(a[0], want, do)
    mine = [t.detach().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True) for t in want]
    b = gated_delta_rule(*mine[:5], initial_state=mine[5])
    for x, y in zip(torch.autograd.grad(b[0], mine, do), wg):
        assert torch.equal(x, y)


def test_decay_that_forgets():
    q, k, v, g, beta, s = R.inputs(1, 150, 1, 2, 64, 64, seed=9)
    g[:, 20] = float("-inf")
    g[:, 64] = float("-inf")  # a chunk's first token
    g[:, 127, 0] = -5000.0    # a chunk's last
    g[:, 70:90, 1] = -80.0
    mine = with_grad((q, k, v, g, beta, s))
    plain = with_grad([t.double() for t in (q, k, v, g, beta, s)])
    out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
    out_r, last_r = R.rule(*plain)
    close(out, out_r, torch.float32)
    close(last, last_r, torch.float32)
    do, ds = torch.randn_like(out), torch.randn_like(last)
    got = torch.autograd.grad((out, last), mine, (do, ds))
    # where g is -inf the 64-bit gradient is exp(-inf) * finite = 0
    want = torch.autograd.grad((out_r, last_r), plain, (do.double(), ds.double()))
    for name, a, b in zip(NAMES, got, want):
        close(a, b, torch.float32)
    assert float(got[3][:, 20].abs().max()) == 0 and float(got[3][0, 127, 0]) == 0


def test_zero_strength_and_equal_keys():
    """beta = 0 writes nothing (and nothing divides by it); equal unit keys with beta = 1 are the hardest inverse."""
    q, k, v, g, beta, s = R.inputs(1, 128, 1, 2, 32, 32, seed=10)
    k = k[:, :1].expand_as(k).contiguous()
    beta = torch.ones_like(beta)
    beta[:, ::3] = 0.0
    g = torch.zeros_like(g)
    mine, plain = with_grad((q, k, v, g, beta, s)), with_grad([t.double() for t in (q, k, v, g, beta, s)])
    out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
    out_r, last_r = R.rule(*plain)
    close(out, out_r, torch.float32)
    close(last, last_r, torch.float32)
    do = torch.randn_like(out)
    for a, b in zip(torch.autograd.grad(out, mine, do), torch.autograd.grad(out_r, plain, do.double())):
        close(a, b, torch.float32)


def test_empty():
    q, k, v, g, beta, s = R.inputs(2, 0, 1, 2, 16, 8, seed=0)
    mine = with_grad((q, k, v, g, beta, s))
    out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
    assert out.shape == (2, 0, 2, 8) and torch.equal(last, s)
    d = torch.randn_like(last)
    grads = torch.autograd.grad(last, mine, d)
    assert torch.equal(grads[5], d)
    out, last = gated_delta_rule(q, k, v, g, beta)
    assert float(last.abs().max()) == 0
    x = R.inputs(0, 5, 1, 2, 16, 8, seed=0)
    out, last = gated_delta_rule(*x[:5], initial_state=x[5])
    assert out.shape == (0, 5, 2, 8) and last.shape == (0, 2, 16, 8)
    assert gated_delta_step(*(t[:, 0] for t in x[:5]), x[5]).shape == (0, 2, 8)


def test_nan_stays_with_its_head():
    q, k, v, g, beta, s = R.inputs(2, 100, 2, 4, 64, 64, seed=12)
    clean, _ = gated_delta_rule(q, k, v, g, beta, initial_state=s)
    v = v.clone()
    v[1, 50, 3, 7] = float("nan")
    out, last = gated_delta_rule(q, k, v, g, beta, initial_state=s)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :, :3], clean[1, :, :3])
    assert torch.isnan(out[1, 50:, 3, 7]).all() and torch.isnan(last[1, 3, :, 7]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("what", ["q", "k", "v", "g", "beta", "state"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_reaches_no_earlier_token(dtype, what, bad):
    """A token's output does not depend on later tokens, not even on a NaN in them (an infinite g aside, which is none)."""
    x = list(R.inputs(1, 140, 1, 2, 48, 32, dtype=dtype, seed=15))
    i, t = NAMES.index(what), 75
    clean, _ = gated_delta_rule(*x[:5], initial_state=x[5])
    x[i] = x[i].clone()
    if what == "state":
        x[i][0, 1, 3, 5] = bad
    elif what in ("g", "beta"):
        x[i][0, t, 1] = bad
    else:
        x[i][0, t, -1, 5] = bad
    out, last = gated_delta_rule(*x[:5], initial_state=x[5])
    if what == "state":
        assert torch.isnan(out[0, :, 1, 5]).all()
        # the column of the state that is not finite, and no other
        rest = [c for c in range(32) if c != 5]
        assert rel(out[..., 1, rest], clean[..., 1, rest]) <= TOL[dtype]
        assert torch.equal(out[:, :, 0], clean[:, :, 0])
        return
    heads = slice(0, 2) if what in ("q", "k") else slice(1, 2)  # of one key head, both value heads
    assert rel(out[:, :t, heads], clean[:, :t, heads]) <= TOL[dtype] and torch.isfinite(out[:, :t]).all()
    assert not torch.isfinite(out[0, t, 1]).all()
    if what == "q":
        assert rel(out[:, t + 1:], clean[:, t + 1:]) <= TOL[dtype]
    else:
        assert not torch.isfinite(last[0, 1]).all()
    if what not in ("q", "k"):
        assert torch.equal(out[:, :, 0], clean[:, :, 0])


def test_repeats_bit_for_bit_and_on_another_stream():
    x = R.inputs(3, 190, 2, 6, 128, 64, dtype=torch.bfloat16, seed=13)

    def once():
        mine = with_grad(x)
        out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
        return (out, last) + torch.autograd.grad((out.float().square().sum() + last.square().sum()), mine)

    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = once()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1), (3, 2, 6, 96, 81), (2, 1, 2, 128, 128), (4, 2, 2, 33, 64), (1, 1, 1, 127, 30)])
def test_step(size, dtype):
    B, Hk, Hv, dk, dv = size
    q, k, v, g, beta, s = R.inputs(B, 4, Hk, Hv, dk, dv, dtype=dtype, seed=sum(size))
    g[:, 2, 0] = float("-inf")
    state, want = s.clone(), s.double()
    for t in range(4):
        before = state._version
        out = gated_delta_step(q[:, t], k[:, t], v[:, t], g[:, t], beta[:, t], state)
        o, want = R.rule(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], g[:, t:t + 1], beta[:, t:t + 1], want)
        close(out, o[:, 0], dtype)
        close(state, want, torch.float32)
        assert state._version > before
    # a state that starts off a 16-byte boundary
    odd = torch.zeros(s.numel() + 1, device="cuda")[1:].view(s.shape).copy_(s)
    aligned = s.clone()
    a = gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], odd)
    b = gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], aligned)
    assert torch.equal(a, b) and torch.equal(odd, aligned)


def test_steps_continue_a_prompt():
    x = R.inputs(2, 140, 2, 4, 64, 64, seed=21)
    out, last = gated_delta_rule(*x[:5], initial_state=x[5])
    part, state = gated_delta_rule(*(t[:, :130] for t in x[:5]), initial_state=x[5])
    assert rel(part, out[:, :130]) <= 1e-6
    for t in range(130, 140):
        o = gated_delta_step(*(y[:, t] for y in x[:5]), state)
        assert rel(o, out[:, t]) <= 2e-6
    assert rel(state, last) <= 2e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sequence_in_ranges(dtype):
    """Many chunks of many heads are worked on in overlapped ranges; pieces of the same sequence, one after the other,
    give the same bits."""
    x = R.inputs(1, 4101, 4, 32, 32, 32, dtype=dtype, seed=14)
    with torch.no_grad():
        out, last = gated_delta_rule(*x[:5], initial_state=x[5])
        state, parts = x[5], []
        for a in range(0, 4101, 1024):
            o, state = gated_delta_rule(*(t[:, a:a + 1024] for t in x[:5]), initial_state=state)
            parts.append(o)
        assert torch.equal(torch.cat(parts, 1), out) and torch.equal(state, last)
        out_r, last_r = R.rule(*x)
    close(out, out_r, dtype)
    close(last, last_r, torch.float32)
    mine = with_grad(x)
    out_t, last_t = gated_delta_rule(*mine[:5], initial_state=mine[5])
    assert torch.equal(last_t, last)
    close(out_t.detach(), out_r, dtype)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        out_g, last_g = gated_delta_rule(*x[:5], initial_state=x[5])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out_g, out) and torch.equal(last_g, last)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [-60, -7, 40])
def test_scaled_values_give_scaled_results(dtype, power):
    """Tiles carry their own power of two, so values, states and queries of any size lose nothing: bit for bit."""
    x = R.inputs(1, 150, 1, 2, 72, 40, dtype=dtype, seed=16)
    f = 2.0 ** power
    runs = []
    for scale in (1.0, f):
        q, k, v, g, beta, s = x
        mine = with_grad((q * 2.0 ** 20 if scale != 1.0 else q, k, v * scale, g, beta, s * scale))
        out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
        do = torch.ones_like(out) * (k.new_tensor(1.5))
        grads = torch.autograd.grad((out, last), mine, (do, torch.ones_like(last) * 2.0 ** 20 if scale != 1.0 else torch.ones_like(last)))
        runs.append((out, last) + grads)
    (o, l, dq, dk, dv, dg, db, ds), (o2, l2, dq2, dk2, dv2, dg2, db2, ds2) = runs
    big = 2.0 ** 20
    assert torch.equal(o2.float(), o.float() * (f * big)) and torch.equal(l2, l * f)
    # out's gradient times q's factor, dS's likewise: all sums grow alike
    assert torch.equal(dq2.float(), dq.float() * f) and torch.equal(dk2.float(), dk.float() * (f * big))
    assert torch.equal(dv2.float(), dv.float() * big) and torch.equal(ds2, ds * big)
    assert torch.equal(dg2, dg * (f * big)) and torch.equal(db2, db * (f * big))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_offsets_past_32_bits(dtype):
    x = R.inputs(2, 70, 1, 2, 16, 24, dtype=dtype, seed=17)
    want = gated_delta_rule(*x[:5], initial_state=x[5])
    far = 2 ** 31 + 64  # elements between the two sequences
    base = torch.empty(far + 70 * 2 * 24, dtype=dtype, device="cuda")
    wide = []
    for t in x[:3]:
        w = base.as_strided(t.shape, (far,) + t.stride()[1:])
        wide.append(w.copy_(t))
        got = gated_delta_rule(*(w if t is y else y for y in x[:3]), *x[3:5], initial_state=x[5])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        state, other = x[5].clone(), x[5].clone()
        a = gated_delta_step(*((w if t is y else y)[:, 3] for y in x[:3]), x[3][:, 3], x[4][:, 3], state)
        b = gated_delta_step(*(y[:, 3] for y in x[:5]), other)
        assert torch.equal(a, b) and torch.equal(state, other)


def test_refusals():
    q, k, v, g, beta, s = R.inputs(2, 5, 2, 4, 16, 8)
    with pytest.raises(ValueError, match="shape"):
        gated_delta_rule(q[0], k, v, g, beta)
    with pytest.raises(ValueError, match="q's shape"):
        gated_delta_rule(q, k[..., :8], v, g, beta)
    with pytest.raises(ValueError, match="leading"):
        gated_delta_rule(q, k, v, g[:, :4], beta)
    with pytest.raises(ValueError, match="multiple"):
        gated_delta_rule(q, k, v[:, :, :3], g[..., :3], beta[..., :3])
    with pytest.raises(ValueError, match="state"):
        gated_delta_rule(q, k, v, g, beta, initial_state=s[..., :4])
    with pytest.raises(ValueError, match="same CUDA device"):
        gated_delta_rule(q, k, v, g.cpu(), beta)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_delta_rule(*(t.cpu() for t in (q, k, v, g, beta)))
    with pytest.raises(RuntimeError, match="float32 or all bfloat16"):
        gated_delta_rule(q.double(), k.double(), v.double(), g, beta)
    with pytest.raises(RuntimeError, match="float32 or all bfloat16"):
        gated_delta_rule(q.bfloat16(), k, v, g, beta)
    with pytest.raises(RuntimeError, match="must be float32"):
        gated_delta_rule(q, k, v, g.bfloat16(), beta)
    big = R.inputs(1, 2, 1, 1, 129, 8)
    with pytest.raises(ValueError, match="128"):
        gated_delta_rule(*big[:5])
    with pytest.raises(ValueError, match="contiguous"):
        gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], s.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError, match="state"):
        gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], s[:1])


def test_layer_prompt_then_tokens():
    torch.manual_seed(0)
    layer = GatedDelta(48, num_heads=4, head_size=32, num_key_heads=2, output_size=20).cuda()
    x = torch.randn(3, 70, 48, device="cuda")
    with torch.no_grad():
        whole, last = layer(x)
        part, state = layer(x[:, :60], layer.init_state(3))
        for t in range(60, 70):
            y = layer.step(x[:, t], state)
            torch.testing.assert_close(y, whole[:, t], rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(part, whole[:, :60], rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(state, last, rtol=1e-4, atol=1e-5)
    y, _ = layer(x)
    y.square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in layer.parameters())
    with pytest.raises(ValueError):
        layer(x[..., :40])
    with pytest.raises(ValueError):
        GatedDelta(8, num_heads=3, num_key_heads=2)


def test_rule_in_a_cuda_graph():
    x = R.inputs(2, 90, 1, 2, 64, 64, seed=30)
    mine = with_grad(x)

    def body():
        out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
        return (out, last) + torch.autograd.grad(out.square().sum() + last.square().sum(), mine)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = body()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = body()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(30, 130, 3, 6, 64, 40), (20, 100, 4, 12, 128, 33)])
def test_a_sequence_alone_gives_what_it_gives_in_a_batch(dtype, size):
    """Grids of different sizes share the work out differently; no sum depends on how."""
    B, T, Hk, Hv, dk, dv = size
    ts = R.inputs(B, T, Hk, Hv, dk, dv, dtype=dtype, seed=5)
    do = torch.randn(B, T, Hv, dv, device="cuda").to(dtype)
    ds = torch.randn(B, Hv, dk, dv, device="cuda")

    def run(n):
        x = with_grad([t[n] for t in ts])
        o, s = gated_delta_rule(*x)
        torch.autograd.backward([o, s], [do[n], ds[n]])
        return [o, s, *(t.grad for t in x)]

    whole = run(slice(None))
    for b in (0, B // 2, B - 1):
        one = run(slice(b, b + 1))
        for name, x, y in zip(("o", "state", "dq", "dk", "dv", "dg", "dbeta", "ds"), whole, one):
            assert torch.equal(x[b : b + 1], y), (name, b)
    with torch.no_grad():
        o, s = gated_delta_rule(*(t[:1] for t in ts))
        many, last = gated_delta_rule(*ts)
    assert torch.equal(many[:1], o) and torch.equal(last[:1], s)
