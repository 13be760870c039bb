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
