"""How exact the gated delta rule's outputs are element by element and token by token, where tests/test_delta_gpu.py
compares whole tensors by their 2-norm."""
import pytest
import torch

from rnn_kernel_b200 import gated_delta_rule

from . import delta_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("size", [(1, 77, 2, 4, 64, 64), (2, 300, 1, 2, 128, 128)])
def test_bf16_outputs_are_fp32_results_rounded_once(size, train):
    """An FP32 result (a relative error of 2e-6 of the outputs' root mean square, rms) rounds to another bf16 number
    than the exact one where it lies within that error of the middle of two, which are 2^-8 |x| apart or more: for a share
    of 2 * 2e-6 * 2^8 * mean(rms / |x|) of the elements, and that mean is below 10 over elements that a bf16 number
    tells from zero.  One percent is twice that."""
    x = R.inputs(*size, dtype=torch.bfloat16, seed=sum(size))
    with torch.set_grad_enabled(train):
        if train:
            x = [t.requires_grad_(True) for t in x]
        out, _ = gated_delta_rule(*x[:5], initial_state=x[5])
    want, _ = R.rule(*(t.detach() for t in x))
    assert float((out.detach() != want.bfloat16()).float().mean()) <= 0.01


def plain(x, do=None, ds=None, dtype=torch.float64):
    """The recurrence token by token in `dtype`: out, last state and, with do and ds, every input's gradient."""
    x = [t.detach().to(dtype).requires_grad_(do is not None) for t in x]
    q, k, v, g, beta, s = x
    Hv, dk = v.shape[2], q.shape[3]
    qr, kr = (t.repeat_interleave(Hv // t.shape[2], dim=2) for t in (q, k))
    outs = []
    for t in range(q.shape[1]):
        s = s * g[:, t].exp()[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (s * kr[:, t, :, :, None]).sum(-2))
        s = s + kr[:, t, :, :, None] * u[..., None, :]
        outs.append((s * qr[:, t, :, :, None]).sum(-2) * dk ** -0.5)
    out = torch.stack(outs, 1)
    if do is None:
        return out, s
    return (out, s) + torch.autograd.grad((out, s), x, (do.to(dtype), ds.to(dtype)))


NAMES = ("out", "state", "dq", "dk", "dv", "dg", "dbeta", "dstate")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [20, 30, 40])
@pytest.mark.parametrize("what", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("dk", [64, 128])
def test_a_large_token_leaves_the_others_their_digits(what, power, dtype, dk):
    """One token's q, k, v or output gradient is 2^20 to 2^40 times the others', amid its 16 tokens and its chunk.  Each
    token's vectors (each stretch's numbers: before it, it, after it) are as exact as FP32 arithmetic leaves them.

    The allowance, of a token's own size: 1e-5 in FP32 (2e-6 bounds whole tensors, see test_delta_gpu.py; a single token
    may cancel a few times as much), 3e-3 where the result is bf16; and 16 times the error of the plain FP32 recurrence in
    the same stretch (root mean square), since planes keep 22 bits of 24 and chunks take some four products in turn."""
    T, t = 150, 75
    x = list(R.inputs(1, T, 1, 2, dk, 48, dtype=dtype, seed=power))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(power + 1)
    do = torch.randn(1, T, 2, 48, device="cuda", generator=gen).to(dtype)
    ds = torch.randn(1, 2, dk, 48, device="cuda", generator=gen)
    for name, i in (("q", 0), ("k", 1), ("v", 2)):
        if what == name:
            x[i][:, t] *= 2.0 ** power
    if what == "dout":
        do[:, t] *= 2.0 ** power
    mine = [y.clone().requires_grad_(True) for y in x]
    out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
    got = (out.detach(), last.detach()) + torch.autograd.grad((out, last), mine, (do, ds))
    want, rough = plain(x, do, ds), plain(x, do, ds, torch.float32)
    for name, a, b, c in zip(NAMES, got, want, rough):
        assert torch.isfinite(a).all(), name
        allowed = 3e-3 if a.dtype == torch.bfloat16 else 1e-5
        a, c = a.double(), c.double()
        if name in ("state", "dstate"):
            assert float((a - b).norm()) <= allowed * float(b.norm()) + 16 * float((c - b).norm()), name
            continue
        for part in (slice(0, t), slice(t, t + 1), slice(t + 1, T)):
            err, rerr, size = ((y[:, part]) for y in (a - b, c - b, b))
            if name in ("dg", "dbeta"):  # numbers: a stretch of one head's
                err, rerr, size = (y.norm(dim=1) for y in (err, rerr, size))
            else:
                err, rerr, size = (y.norm(dim=-1) for y in (err, rerr, size))
            rough_rel = float((rerr / size).square().mean().sqrt())
            worst = float((err / size).max())
            assert worst <= allowed + 16 * rough_rel, (name, part, worst, rough_rel)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("strength", [float("-inf"), -400.0])
@pytest.mark.parametrize("t", [75, 80, 96])
def test_nothing_comes_through_a_reset(t, dtype, strength):
    """Tokens after a decay of zero (or one far below FP32) get the same bits whatever was before it, and however small
    their own values are."""
    T = 150
    q, k, v, g, beta, s = R.inputs(1, T, 1, 2, 64, 48, dtype=dtype, seed=3)
    g[:, t] = strength
    v[:, t:] *= 2.0 ** -80
    do, ds = torch.randn_like(v), torch.randn_like(s)
    runs = []  # with other values before it, and other gradients from it on
    for factor in (1.0, 2.0 ** 40):
        w = v.clone()
        w[:, :t] = torch.randn_like(w[:, :t]) * factor
        d = do.clone()
        d[:, :t] *= 2.0 ** -80
        d[:, t:] = torch.randn_like(d[:, t:]) * factor  # which the gradients of earlier tokens must not see
        w0, d1 = torch.randn_like(s) * factor, torch.randn_like(ds) * factor
        x = [y.clone().requires_grad_(True) for y in (q, k, w, g, beta, w0)]
        out, last = gated_delta_rule(*x[:5], initial_state=x[5])
        runs.append((out.detach()[:, t:], last.detach(), torch.autograd.grad((out, last), x, (d, d1))))
    (o, l, a), (o2, l2, b) = runs
    assert torch.equal(o, o2) and torch.equal(l, l2) and float(o.abs().max()) > 0
    assert torch.equal(a[2][:, :t], b[2][:, :t]) and torch.equal(a[5], b[5])  # dv before it, and the initial state's


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(2, 150, 1, 2, 64, 48), (1, 100, 2, 4, 128, 33), (1, 70, 1, 3, 40, 72)])
def test_every_token_of_its_own_size(size, dtype):
    """Values, queries, output gradients (2^-12 to 2^12), keys (2^-24 to 1) and strengths (2^-20 to 1) of every token's own
    size.  The allowance is that of one large token, above; the plain recurrence's error is taken over all tokens."""
    B, T, Hk, Hv, dk, dv = size
    x = list(R.inputs(*size, dtype=dtype, seed=T))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(T)

    def powers(lo, hi, heads):
        return torch.exp2(torch.randint(lo, hi + 1, (B, T, heads), device="cuda", generator=gen).float())

    x[0] = (x[0].float() * powers(-12, 12, Hk)[..., None]).to(dtype)
    x[1] = (x[1].float() * powers(-24, 0, Hk)[..., None]).to(dtype)
    x[2] = (x[2].float() * powers(-12, 12, Hv)[..., None]).to(dtype)
    x[4] = x[4] * powers(-20, 0, Hv)
    do = (torch.randn(B, T, Hv, dv, device="cuda", generator=gen) * powers(-12, 12, Hv)[..., None]).to(dtype)
    ds = torch.randn(B, Hv, dk, dv, device="cuda", generator=gen)
    mine = [y.clone().requires_grad_(True) for y in x]
    out, last = gated_delta_rule(*mine[:5], initial_state=mine[5])
    got = (out.detach(), last.detach()) + torch.autograd.grad((out, last), mine, (do, ds))
    want, rough = plain(x, do, ds), plain(x, do, ds, torch.float32)
    for name, a, b, c in zip(NAMES, got, want, rough):
        allowed = 3e-3 if a.dtype == torch.bfloat16 else 1e-5
        err, rerr, length = a.double() - b, c.double() - b, b
        if name in ("state", "dstate"):
            err, rerr, length = (y.flatten(2).norm(dim=-1) for y in (err, rerr, length))
        elif name in ("dg", "dbeta"):
            # single numbers may cancel: a token's, among the eight around it
            err, rerr, length = (y.square().unfold(1, 8, 1).sum(-1).sqrt() for y in (err, rerr, length))
        else:
            err, rerr, length = (y.norm(dim=-1) for y in (err, rerr, length))
        rough_rel = float((rerr / length).square().mean().sqrt())
        worst = float((err / length).max())
        assert worst <= allowed + 16 * rough_rel, (name, worst, rough_rel)
