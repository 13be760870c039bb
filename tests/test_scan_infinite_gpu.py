"""Infinite states of the selective scan: a decay above zero leaves an infinity as it is, over a block, over pieces of a
sequence and back in the gradient.  (Decays here are all above 2^-126, where the kernels' numbers end: rates of at most about
30 e^1, steps of at most about 0.5.)  Finite numbers beside it are held to 1e-5, as the scan's own tests derive it."""
import pytest
import torch

from rnn_kernel_b200 import selective_scan

from . import scan_reference as R
from .scan_reference import caller  # noqa: F401

pytestmark = pytest.mark.gpu

INF = float("inf")


def same(x, y):
    """The same infinities and NaN, and finite numbers as near as the scan's are."""
    x, y = x.double(), y.detach().double()
    assert torch.equal(x.isnan(), y.isnan())
    assert torch.equal(x.isinf(), y.isinf()) and torch.equal(x[x.isinf()], y[y.isinf()])
    fine = y.isfinite()
    assert R.rel(x[fine], y[fine]) <= 1e-5


# B, T, D, N, G; the long ones are cut into pieces
SIZES = [(1, 1, 40, 2, 1), (2, 15, 40, 4, 1), (2, 16, 40, 8, 2), (1, 17, 64, 16, 1), (2, 100, 70, 12, 2), (1, 300, 64, 24, 1),
         (1, 2100, 9, 30, 1), (2, 1500, 66, 16, 1), (1, 700, 40, 7, 1)]


def inputs(size, **kw):
    kw = R.scan_inputs(*size, seed=sum(size), **kw)
    kw["A"][:, 0] = 0.0
    return kw


@pytest.mark.parametrize("size", SIZES)
def test_a_state_that_starts_infinite(size):
    kw = inputs(size)
    s = kw["initial_state"]
    s[0, 3, 0] = INF  # A = 0: the difference of decays is 0
    s[-1, 5, -1] = -INF  # the fastest decay: over a piece of the sequence it is 0 in FP32
    s[0, 7, size[3] // 2] = INF
    out, last = selective_scan(**kw)
    want = R.scan(**kw)
    assert int(want[1].isinf().sum()) == 3
    same(last, want[1])
    same(out, want[0])


@pytest.mark.parametrize("size", SIZES)
def test_a_token_that_makes_states_infinite(size):
    kw = inputs(size, gate=False)
    kw["x"][0, min(size[1] - 1, 5), 3] = INF
    out, last = selective_scan(**kw)
    want = R.scan(**kw)
    assert bool(want[1][0, 3].isinf().all())
    same(last, want[1])
    same(out, want[0])


@pytest.mark.parametrize("size", SIZES)
def test_an_infinite_gradient_of_the_last_state(size):
    kw = inputs(size)
    mine, plain = R.leaves(kw), R.leaves(kw, wide=True)
    outs, want = selective_scan(**mine), R.scan(**plain)
    d = [torch.randn_like(o) for o in outs]
    d[1][0, 3, 0] = INF
    d[1][-1, 5, -1] = -INF
    got, = torch.autograd.grad(outs, mine["initial_state"], d)
    true, = torch.autograd.grad(want, plain["initial_state"], [t.double() for t in d])
    assert int(true.isinf().sum()) == 2
    same(got, true)
