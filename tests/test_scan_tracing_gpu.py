"""torch.jit.trace: a traced call of the scan, the convolution and the norm computes what the call does, with gradients and
without; the single tokens, which change a state in place, refuse to be traced.  All comparisons are of equal bits."""
import pytest
import torch

from rnn_kernel_b200 import LayerNorm, SelectiveScan, causal_conv, causal_conv_step, layer_norm, selective_scan, selective_step

from . import scan_reference as R
from .scan_reference import caller  # noqa: F401

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::DeprecationWarning"),
              pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")]

KW = dict(b=2, T=70, D=24, N=6, G=2)


def calls():
    kw = R.scan_inputs(**KW, device="cuda")
    w, b, cw = torch.randn(24, device="cuda"), torch.randn(24, device="cuda"), torch.randn(24, 4, device="cuda")
    rest = {n: t for n, t in kw.items() if n != "x"}
    few = {n: t for n, t in rest.items() if n not in ("skip", "z", "dt_bias", "initial_state")}
    torch.manual_seed(0)
    layer, norm = SelectiveScan(24).cuda(), LayerNorm(24).cuda()
    return {"scan": lambda x: selective_scan(x, **rest), "scan without options": lambda x: selective_scan(x, **few),
            "conv": lambda x: causal_conv(x, cw, b, "silu"), "conv without options": lambda x: causal_conv(x, cw),
            "norm": lambda x: layer_norm(x, w, b), "norm and sum": lambda x: layer_norm(x, w, residual=2 * x),
            "layer": layer, "norm layer": norm}


def flat(y):
    return tuple(t for part in y for t in flat(part)) if isinstance(y, tuple) else (y,)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", ["scan", "scan without options", "conv", "conv without options", "norm", "norm and sum", "layer", "norm layer"])
def test_a_traced_call_computes(name, grad):
    call = calls()[name]
    x, new = (torch.randn(2, 70, 24, device="cuda", requires_grad=grad) for _ in range(2))
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(call, (x,), check_trace=False)
        want, got = flat(call(new)), flat(traced(new))
        torch.empty(1 << 22, device="cuda").fill_(7.0)  # what an output that nobody wrote would be likely to hold
        again = flat(traced(new))
    assert len(want) == len(got)
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    if grad:
        d = [torch.randn_like(t) for t in want]
        assert torch.equal(torch.autograd.grad(want, new, d)[0], torch.autograd.grad(got, new, d)[0])


def test_single_tokens_refuse():
    kw = {n: t[:, 0] if n in ("x", "dt", "B", "C", "z") else t for n, t in R.scan_inputs(**KW, device="cuda").items()}
    state, conv_state, cw = kw.pop("initial_state"), torch.zeros(2, 3, 24, device="cuda"), torch.randn(24, 4, device="cuda")
    x = kw.pop("x")
    before = state.clone()
    for call in (lambda x: selective_step(x, state=state, **kw), lambda x: causal_conv_step(x, cw, conv_state)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (x,), check_trace=False)
    assert torch.equal(state, before) and float(conv_state.abs().sum()) == 0
