"""8-bit moments hold a block of second moments below 2^-100 as zero: eps has to be no less than their root, 2^-50."""
import numpy as np
import pytest
import torch

from rnn_kernel_b200 import AdamW, _lib, optim


@pytest.mark.parametrize("eps", [0.0, 1e-30, 2.0 ** -51])
def test_too_small_eps_is_refused(eps):
    p = [torch.zeros(3)]
    with pytest.raises(ValueError, match="2.-50"):
        AdamW(p, eps=eps, state_bits=8)
    for bits in (8, 32):
        with pytest.raises(RuntimeError, match="CUDA"):  # the next check
            AdamW(p, eps=eps if bits == 32 else 1e-15, state_bits=bits)
    e = np.zeros(1, dtype=optim._ENTRY)  # a tensor of no elements: nothing to do once it is accepted
    lib = _lib.load()

    def step(bits, eps):
        return lib.gru_adamw_step(e.ctypes.data, 1, _lib.GRU_F32, bits, 0, 0, 0, 0, 256, 0.9, 0.999, eps, 1.0, 0, 1, 0, 0, 0)

    assert step(8, eps) == _lib.GRU_ERR_INVALID and "eps" in _lib.last_error()
    assert step(8, 2.0 ** -50) == step(32, eps) == _lib.GRU_OK


@pytest.mark.gpu
def test_least_eps_keeps_steps_finite_where_second_moments_vanish():
    """Gradients whose squares (1e-32) fall below 2^-100, then none: the step is at most lr m / eps."""
    p = torch.nn.Parameter(torch.zeros(512, device="cuda"))
    opt = AdamW([p], lr=1e-3, eps=2.0 ** -50, weight_decay=0.0, state_bits=8)
    p.grad = torch.full_like(p, 1e-16)
    p.grad[256:] = 1.0
    for _ in range(3):
        opt.step()
        p.grad = torch.zeros_like(p)
    # the first step's moments: m / (1 - b1) = 1e-16, held to within 1/8 of it
    assert torch.isfinite(p).all() and float(p.detach()[:256].abs().max()) <= 3 * 1e-3 * 1.25e-16 / 2.0 ** -50
