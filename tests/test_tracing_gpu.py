"""torch.jit.trace of the GRU without gradients and of the gated delta rule: a traced call computes what the call does; the
delta rule's single token, which changes a state in place, refuses to be traced.  All comparisons are of equal bits."""
import pytest
import torch

from rnn_kernel_b200 import GRU, GatedDelta, gated_delta_rule, gated_delta_step
from rnn_kernel_b200.gru import gru_forward_inference

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::DeprecationWarning"),
              pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")]


def flat(y):
    return tuple(t for part in y for t in flat(part)) if isinstance(y, tuple) else (y,)


def calls():
    torch.manual_seed(0)
    gru, delta = GRU(32, 32, num_layers=2).cuda(), GatedDelta(32, num_heads=1, head_size=32).cuda()
    params = [p.detach() for p in gru.layer_parameters(0)]
    h0 = torch.randn(2, 32, device="cuda")
    g, beta = -torch.rand(2, 40, 2, device="cuda"), torch.rand(2, 40, 2, device="cuda")

    def rule(x):
        k = torch.nn.functional.normalize(x.unflatten(-1, (2, 16)), dim=-1)
        return gated_delta_rule(x.unflatten(-1, (2, 16)), k, 2 * x.unflatten(-1, (2, 16)), g, beta)

    return {"gru": gru, "gru inference": lambda x: gru_forward_inference(x, h0, *params), "delta layer": delta, "rule": rule}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", ["gru", "gru inference", "delta layer", "rule"])
def test_a_traced_call_computes(name, grad):
    call = calls()[name]
    x, new = (torch.randn(2, 40, 32, device="cuda", requires_grad=grad) for _ in range(2))
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(call, (x,), check_trace=False)
        want, got = flat(call(new)), flat(traced(new))
        torch.empty(1 << 22, device="cuda").fill_(7.0)  # what an output that nobody wrote would be likely to hold
        again = flat(traced(new))
    assert len(want) == len(got)
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    if grad and name != "gru inference":
        d = [torch.randn_like(t) for t in want]
        assert torch.equal(torch.autograd.grad(want, new, d)[0], torch.autograd.grad(got, new, d)[0])


def test_the_delta_rules_single_token_refuses():
    q, k, v = torch.randn(3, 2, 2, 16, device="cuda")
    g, beta = -torch.rand(2, 2, device="cuda"), torch.rand(2, 2, device="cuda")
    state = torch.randn(2, 2, 16, 16, device="cuda")
    before = state.clone()
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda q: gated_delta_step(q, k, v, g, beta, state), (q,), check_trace=False)
    assert torch.equal(state, before)
