"""States are worked on in fours; those that a call does not have stay out of its results where dt x or an output's
gradient is infinite.  B, C and the outputs' gradients are positive and there is no skip, so an infinity meets none of the
other sign.  Finite numbers are held to 1e-5, as the scan's own tests derive it."""
import pytest
import torch

from rnn_kernel_b200 import selective_scan, selective_step

from . import scan_reference as R
from .scan_reference import caller  # noqa: F401

pytestmark = pytest.mark.gpu

INF = float("inf")


def same(x, y):
    """The same infinities, no NaN, and finite numbers as near as the scan's are."""
    x, y = x.double(), y.detach().double()
    assert not x.isnan().any() and not y.isnan().any()
    assert torch.equal(x.isinf(), y.isinf()) and torch.equal(x[x.isinf()], y[y.isinf()])
    fine = y.isfinite()
    assert R.rel(x[fine], y[fine]) <= 1e-5


def inputs(T, N):
    kw = R.scan_inputs(2, T, 40, N, seed=N, gate=False, skip=False)
    kw["B"], kw["C"] = kw["B"].abs() + 0.1, kw["C"].abs() + 0.1
    kw["x"][1, 0, 3] = INF
    return kw


@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 7, 11, 13, 18, 27, 30, 33, 62])
def test_values_and_gradients(N):
    kw = inputs(3, N)
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    outs, want = selective_scan(**mine), R.scan(**plain)
    assert bool(want[0][1, :, 3].isinf().all())
    for a, b in zip(outs, want):
        same(a, b)
    names = ("x", "dt", "B", "C", "initial_state")
    d = [torch.rand_like(o) + 0.1 for o in outs]
    got = torch.autograd.grad(outs, [mine[n] for n in names], d)
    true = torch.autograd.grad(want, [plain[n] for n in names], [t.double() for t in d])
    assert bool(true[1][1, 1:, 3].isinf().all())
    for a, b in zip(got, true):
        same(a, b)


@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 7, 11, 13, 18, 27, 30, 33, 62])
def test_an_infinite_gradient(N):
    kw = inputs(3, N)
    kw["x"][1, 0, 3] = 1.0
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    outs, want = selective_scan(**mine), R.scan(**plain)
    names = ("x", "initial_state")
    d = [torch.rand_like(o) + 0.1 for o in outs]
    d[0][1, 2, 3] = INF
    got = torch.autograd.grad(outs, [mine[n] for n in names], d)
    true = torch.autograd.grad(want, [plain[n] for n in names], [t.double() for t in d])
    assert bool(true[0][1, :, 3].isinf().all()) and bool(true[1][1, 3].isinf().all())
    for a, b in zip(got, true):
        same(a, b)


@pytest.mark.parametrize("B", [1, 80])
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 7, 11, 13, 18, 27, 30, 33, 62])
def test_step(B, N):
    kw = {n: t.repeat(B, *[1] * (t.dim() - 1)) if n in ("x", "dt", "B", "C", "initial_state") else t for n, t in inputs(1, N).items()}
    state = kw.pop("initial_state")
    want, last = R.scan(**kw, initial_state=state)
    one = {n: t[:, 0] if n in ("x", "dt", "B", "C") else t for n, t in kw.items()}
    same(selective_step(state=state, **one), want[:, 0])
    same(state, last)
