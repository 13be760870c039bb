"""What the gated delta rule does with derivatives that it does not have, and when it keeps what a gradient needs."""
import pytest
import torch
from torch.autograd import forward_ad

from rnn_kernel_b200 import gated_delta_rule, gated_delta_step

from . import delta_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("use_state", [True, False])
def test_second_derivative_raises(use_state):
    x = [t.requires_grad_(True) for t in R.inputs(1, 70, 1, 2, 16, 24, seed=1)]
    out, _ = gated_delta_rule(*x[:5], initial_state=x[5] if use_state else None)
    wrt = x if use_state else x[:5]
    plain = torch.autograd.grad(out.square().sum(), wrt, retain_graph=True)
    grads = torch.autograd.grad(out.square().sum(), wrt, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, grads))
    # beside a term that has one, the penalty's part would be missing without a word
    loss = sum(t.square().sum() for t in wrt) + grads[0].square().sum()
    with pytest.raises(RuntimeError, match="second derivative"):
        loss.backward()


@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_raises(no_grad):
    x = R.inputs(1, 5, 1, 2, 16, 24, seed=2)
    want = gated_delta_rule(*x[:5], initial_state=x[5])
    with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        # tensors without a tangent are served
        for a, b in zip(gated_delta_rule(*x[:5], initial_state=x[5]), want):
            assert torch.equal(a, b)
        for i in range(6):
            y = list(x)
            y[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises((NotImplementedError, RuntimeError), match="jvp|derivative"):
                gated_delta_rule(*y[:5], initial_state=y[5])
            y = [t[:, 0] for t in y[:5]] + [y[5].clone() if i < 5 else y[5]]
            with pytest.raises(RuntimeError, match="derivative"):
                gated_delta_step(*y)


def test_without_a_gradient_to_keep_for_the_forward_keeps_nothing():
    """Gradients enabled, but no input asks for one: no more memory than under no_grad, and outputs without a graph."""
    x = R.inputs(2, 512, 2, 4, 64, 64, dtype=torch.bfloat16, seed=3)

    def peak(grad):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        with torch.set_grad_enabled(grad):
            out, last = gated_delta_rule(*x[:5], initial_state=x[5])
        held = torch.cuda.memory_allocated() - before
        return torch.cuda.max_memory_allocated() - before, held, out, last

    _, _, out, last = peak(False)
    top, held, *_ = peak(False)
    top_g, held_g, out_g, last_g = peak(True)
    assert (top_g, held_g) == (top, held)
    assert not out_g.requires_grad and torch.equal(out_g, out) and torch.equal(last_g, last)
    for i in range(6):  # one input that does is enough
        y = [t.clone().requires_grad_(j == i) for j, t in enumerate(x)]
        out_y, last_y = gated_delta_rule(*y[:5], initial_state=y[5])
        assert out_y.requires_grad and last_y.requires_grad
        assert torch.autograd.grad(out_y.sum() + last_y.sum(), y[i])[0].shape == y[i].shape
