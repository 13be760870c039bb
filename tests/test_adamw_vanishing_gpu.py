"""8-bit moments beside gradients so small that their squares vanish in FP32."""
import pytest
import torch

from rnn_kernel_b200 import AdamW

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_whose_squares_vanish_leave_their_weights(dtype):
    """In a block of gradients of one, an element's is 1e-25.  Its first moment, 1e-26, is far below the least code
    (1e-6 here), to which a random rounding still lifts one in 65536; beside its second moment, 1e-53 and so zero, that
    would be a step of lr 1e-6 / eps = 100 lr.  Exactly, a step is lr 1e-25 / eps = 1e-17 lr."""
    p = torch.nn.Parameter(torch.zeros(1 << 22, dtype=dtype, device="cuda"))
    opt = AdamW([p], lr=1.0, weight_decay=0.0, state_bits=8)
    p.grad = torch.full_like(p, 1e-25)
    p.grad[::256] = 1.0
    for _ in range(3):
        opt.step()
    small = p.detach().view(-1, 256)[:, 1:]
    assert float(small.abs().max()) <= 3 * 2e-17
    m, v = (t.view(-1, 256)[:, 1:] for t in opt.moments())
    assert float(m.abs().max()) == 0 and float(v.max()) == 0
