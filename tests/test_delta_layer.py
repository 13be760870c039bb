"""The GatedDelta layer in the types that a model runs it in."""
import pytest
import torch
import torch.nn.functional as F

from rnn_kernel_b200 import GatedDelta

from . import delta_reference as R


def layer(device="cpu"):
    torch.manual_seed(0)
    return GatedDelta(48, num_heads=4, head_size=32, num_key_heads=2, output_size=20).to(device)


def test_projection_gives_one_type_under_autocast():
    with torch.autocast("cpu", torch.bfloat16):
        q, k, v, g, beta = layer()._project(torch.randn(2, 5, 48))
    assert q.dtype == k.dtype == v.dtype == torch.bfloat16
    assert g.dtype == beta.dtype == torch.float32


def test_state_is_fp32_under_another_default_type():
    m = layer()
    torch.set_default_dtype(torch.bfloat16)
    try:
        assert m.init_state(2).dtype == torch.float32
    finally:
        torch.set_default_dtype(torch.float32)


def plain(m, x, state):
    """The layer in 64 bits from the parameters and inputs as they are."""
    p = {n: t.detach().double() for n, t in m.named_parameters()}
    q, k, v, a, b = (x.double() @ p["in_proj.weight"].t()).split(m._split, dim=-1)
    q, k = (F.normalize(t.unflatten(-1, (2, 32)), dim=-1) for t in (q, k))
    g = -p["log_rate"].exp() * F.softplus(a)
    o, last = R.rule(q, k, v.unflatten(-1, (4, 32)), g, b.sigmoid(), state.double())
    o = o * o.square().mean(-1, keepdim=True).add(1e-6).rsqrt() * p["norm_weight"]
    return o.flatten(-2) @ p["out_proj.weight"].t(), last


def rel(x, y):
    return float((x.double() - y).norm() / y.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["autocast", "bfloat16"])
def test_bf16_layer_trains_and_serves(how):
    """Some ten bf16 roundings (2^-9 each) one after another, of numbers that a normalisation keeps near one: 3e-2 is
    fifteen of them."""
    m = layer("cuda")
    x = torch.randn(3, 70, 48, device="cuda")
    cast = torch.autocast("cuda", torch.bfloat16, enabled=how == "autocast")
    if how == "bfloat16":
        m, x = m.bfloat16(), x.bfloat16()
    with torch.no_grad():
        want, want_last = plain(m, x, torch.zeros(3, 4, 32, 32, device="cuda"))
    with cast:
        y, last = m(x)
    assert y.dtype == torch.bfloat16 and last.dtype == torch.float32
    assert rel(y, want) <= 3e-2 and rel(last, want_last) <= 3e-2
    y.float().square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0 for p in m.parameters())
    with torch.no_grad(), cast:
        _, state = m(x[:, :60], m.init_state(3))
        for t in range(60, 70):
            out = m.step(x[:, t], state)
            assert out.dtype == torch.bfloat16 and rel(out, want[:, t]) <= 3e-2
    assert rel(state, want_last) <= 3e-2
