"""The operators together, as a stacked model uses them: norm, projection, convolution, scan, on a residual stream."""
import pytest
import torch
import torch.nn.functional as F

from rnn_kernel_b200 import GRU, DataParallelTrainer, GatedDelta, GraphedTrainStep, RecurrentStack, SelectiveScan

from . import scan_reference as R
from .scan_reference import caller  # noqa: F401

pytestmark = pytest.mark.gpu


def plain_layer(m, x, state):
    """SelectiveScan in 64 bits from a dict of its parameters."""
    conv, h = state
    u, z = (x @ m["in_proj.weight"].t()).chunk(2, -1)
    u, conv = R.conv(u, m["conv_weight"], m["conv_bias"], "silu", conv)
    rank = m["dt_proj.weight"].shape[1]
    groups = m["groups"]
    rest = u @ m["x_proj.weight"].t()
    low, (b, c) = rest[..., :rank], rest[..., rank:].chunk(2, -1)
    y, h = R.scan(u, low @ m["dt_proj.weight"].t(), -m["log_rate"].exp(), b.unflatten(-1, (groups, -1)), c.unflatten(-1, (groups, -1)),
                  m["skip"], z, m["dt_bias"], True, h)
    return y @ m["out_proj.weight"].t(), (conv, h)


def plain_stack(params, groups, x, states):
    stream, out = None, x
    for i, state in enumerate(states):
        stream = out if stream is None else stream + out
        y = R.norm(stream, params[f"norms.{i}.weight"], params[f"norms.{i}.bias"])
        layer = {n.split(".", 2)[2]: p for n, p in params.items() if n.startswith(f"layers.{i}.")}
        out, _ = plain_layer(dict(layer, groups=groups), y, state)
    n = len(states)
    return R.norm(stream + out, params[f"norms.{n}.weight"], params[f"norms.{n}.bias"])


def stack(width=48, layers=2, groups=2, **kw):
    torch.manual_seed(0)
    m = RecurrentStack([SelectiveScan(width, 80, state_size=8, num_groups=groups, **kw) for _ in range(layers)], width).cuda()
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.endswith("bias") and p.dim() == 1:
                p.add_(0.1 * torch.randn_like(p))
    return m


def zeros(b, dtype=torch.float64):
    return [(torch.zeros(b, 3, 80, dtype=dtype, device="cuda"), torch.zeros(b, 80, 8, dtype=dtype, device="cuda")) for _ in range(2)]


@pytest.fixture
def exact_products():
    was = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = was


def test_stack_trains_and_serves_in_fp32(exact_products):
    """Two layers of some eight operations each, every one 1e-5 of its size off at most: 2e-4."""
    m = stack()
    x = torch.randn(3, 70, 48, device="cuda", requires_grad=True)
    params = {n: p.detach().double().requires_grad_(True) for n, p in m.named_parameters()}
    wide = x.detach().double().requires_grad_(True)
    want = plain_stack(params, 2, wide, zeros(3))
    y, states = m(x)
    assert R.rel(y, want) <= 2e-4
    d = torch.randn_like(y)
    names, leaves = zip(*m.named_parameters())
    got = torch.autograd.grad(y, (x, *leaves), d)
    true = torch.autograd.grad(want, (wide, *params.values()), d.double())
    for n, a, b in zip(("x", *names), got, true):
        assert R.rel(a, b) <= 2e-4, (n, R.rel(a, b))
    with torch.no_grad():
        _, states = m(x[:, :60])
        for t in range(60, 70):
            assert R.rel(m.step(x[:, t], states), want[:, t]) <= 2e-4


@pytest.mark.parametrize("how", ["autocast", "bfloat16"])
def test_stack_in_bf16(how):
    """Some twenty bf16 roundings (2^-9 each on average) one after another of numbers that norms keep near one: 4e-2."""
    m = stack()
    x = torch.randn(3, 70, 48, device="cuda")
    cast = torch.autocast("cuda", torch.bfloat16, enabled=how == "autocast")
    if how == "bfloat16":
        m, x = m.bfloat16(), x.bfloat16()
    with torch.no_grad():
        want = plain_stack({n: p.detach().double() for n, p in m.named_parameters()}, 2, x.double(), zeros(3))
    with cast:
        y, states = m(x)
        y.float().square().mean().backward()
    assert R.rel(y, want) <= 4e-2
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0 for p in m.parameters())
    with torch.no_grad(), cast:
        _, states = m(x[:, :60])
        for t in range(60, 70):
            assert R.rel(m.step(x[:, t], states), want[:, t]) <= 4e-2


def test_stack_of_all_recurrent_layers_trains():
    torch.manual_seed(0)
    m = RecurrentStack([GRU(64, 64), GatedDelta(64, num_heads=2, head_size=32), SelectiveScan(64)], 64).cuda()
    trainer = DataParallelTrainer(m, lr=1e-3, optimizer="adamw")
    x, y = torch.randn(2, 4, 40, 64, device="cuda")
    before = trainer.flat.clone()
    loss = trainer.step(x, y)
    assert torch.isfinite(loss) and torch.isfinite(trainer.flat).all()
    assert all(p.grad is not None and float(p.grad.abs().max()) > 0 for p in m.parameters())
    assert not torch.equal(before, trainer.flat)


def test_graph_replay_equals_eager():
    def train(graphed):
        torch.manual_seed(1)
        m = RecurrentStack([SelectiveScan(32), SelectiveScan(32)], 32).cuda()
        trainer = DataParallelTrainer(m, lr=1e-2)
        x, y = torch.randn(2, 4, 40, 32, device="cuda")
        if graphed:
            steps = GraphedTrainStep(trainer, [(x, y)], warmup=2)
            for _ in range(3):
                steps.step()
            torch.cuda.synchronize()
        else:
            for _ in range(5):
                trainer.step(x, y)
        return trainer.flat.clone()

    assert torch.equal(train(True), train(False))


def test_layer_continues_from_a_state():
    m = stack(groups=1)
    layer = m.layers[0]
    x = torch.randn(2, 50, 48, device="cuda")
    with torch.no_grad():
        y, last = layer(x)
        a, state = layer(x[:, :2])
        b, state = layer(x[:, 2:], state)
    assert R.rel(torch.cat([a, b], 1), y) <= 1e-4 and R.rel(state[1], last[1]) <= 1e-4
    # states of the default type's own zeros
    conv, h = layer.init_state(2)
    assert conv.dtype == F.silu(x).dtype and float(h.abs().sum()) == 0
