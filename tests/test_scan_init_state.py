"""SelectiveScan.init_state gives the convolution's state the type that the projection has, under autocast too."""
import pytest
import torch

from rnn_kernel_b200 import SelectiveScan

from . import scan_reference as R


def test_types():
    m = SelectiveScan(16)
    assert m.init_state(2)[0].dtype == torch.float32
    with torch.autocast("cpu", torch.bfloat16):
        conv, h = m.init_state(2)
        assert conv.dtype == torch.bfloat16 and h.dtype == torch.float32
        assert m.init_state(2, torch.float32)[0].dtype == torch.float32
    with torch.autocast("cpu", torch.bfloat16, enabled=False):
        assert m.init_state(2)[0].dtype == torch.float32
    assert m.bfloat16().init_state(2)[0].dtype == torch.bfloat16
    assert SelectiveScan(16).to("meta").init_state(2)[0].device.type == "meta"  # which has no autocast


@pytest.mark.gpu
def test_a_layer_serves_under_autocast_from_its_first_token():
    """Against the same tokens at once: each side's bf16 roundings, some ten of 2^-9 on average in each: 4e-2, as for the
    stack; the projection of the convolution's state is one sum that two products may round to neighbours: 2^-7."""
    torch.manual_seed(0)
    m = SelectiveScan(48).cuda()
    x = torch.randn(3, 5, 48, device="cuda")
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        want, last = m(x, m.init_state(3))
        state = m.init_state(3)
        got = torch.stack([m.step(x[:, t], state) for t in range(5)], 1)
    assert R.rel(got, want) <= 4e-2 and R.rel(state[1], last[1]) <= 4e-2 and R.rel(state[0], last[0]) <= 2.0 ** -7
