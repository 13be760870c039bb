"""AdamW's saved state is all that a run's continuation depends on, and what the trainer's attributes do with it."""
import pytest
import torch

from rnn_kernel_b200 import GRU, AdamW, DataParallelTrainer, mse_loss

pytestmark = pytest.mark.gpu


def params_of(sizes, seed=0):
    torch.manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in sizes]


def gradients(ps, step):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(step)
    for p in ps:
        p.grad = torch.randn(p.shape, device="cuda", generator=gen)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_state_brings_betas_and_eps(bits, capturable):
    ps = params_of([513, 40])
    opt = AdamW(ps, lr=1e-2, betas=(0.8, 0.95), eps=1e-4, weight_decay=0.1, state_bits=bits, seed=9, capturable=capturable)
    for t in range(3):
        gradients(ps, t)
        opt.step()
    saved = opt.state_dict()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = AdamW(qs, lr=5.0, betas=(0.5, 0.5), eps=1e-8, state_bits=bits, capturable=capturable)
    other.load_state_dict(saved)
    for t in range(3, 6):
        for x, o in ((ps, opt), (qs, other)):
            gradients(x, t)
            o.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p.detach(), q.detach())
    # a state of before betas and eps were part of it
    old = {k: v for k, v in saved.items() if k not in ("betas", "eps")}
    third = AdamW(params_of([513, 40]), betas=(0.7, 0.8), eps=1e-3, state_bits=bits, capturable=capturable)
    third.load_state_dict(old)
    assert third.betas == (0.7, 0.8) and third.eps == 1e-3


@pytest.mark.parametrize("optimizer", ["sgd", "adamw"])
def test_trainer_learning_rate_counts(optimizer):
    torch.manual_seed(0)
    x, y = torch.randn(4, 10, 8, device="cuda"), torch.randn(4, 10, 16, device="cuda")

    def run(change):
        torch.manual_seed(1)
        trainer = DataParallelTrainer(GRU(8, 16).cuda(), lr=1e-2, optimizer=optimizer)
        trainer.step(x, y)
        change(trainer)
        before = trainer.flat.clone()
        trainer.step(x, y)
        return trainer.lr, trainer.flat - before

    def by_attribute(t):
        t.lr = 0.0

    def by_group(t):
        t.optimizer.param_groups[0]["lr"] = 0.0

    lr, moved = run(lambda t: None)
    assert lr == 1e-2 and float(moved.abs().max()) > 0
    for change in (by_attribute, by_group) if optimizer == "adamw" else (by_attribute,):
        lr, moved = run(change)
        assert lr == 0.0 and float(moved.abs().max()) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_steps_as_the_optimizer_over_its_parameters(bits):
    """8-bit moments: every parameter's blocks are its own, though all lie in one buffer."""
    torch.manual_seed(0)
    x, y = torch.randn(4, 10, 7, device="cuda"), torch.randn(4, 10, 13, device="cuda")

    def module():
        torch.manual_seed(1)
        return GRU(7, 13, num_layers=2).cuda()

    trainer = DataParallelTrainer(module(), lr=1e-2, optimizer="adamw", state_bits=bits)
    m = module()
    opt = AdamW(m.parameters(), lr=1e-2, state_bits=bits, capturable=True)
    for _ in range(4):
        trainer.step(x, y)
        opt.zero_grad()
        mse_loss(m(x)[0], y).backward()
        opt.step()
    for p, q in zip(trainer.module.parameters(), m.parameters()):
        assert torch.equal(p.detach(), q.detach())
    if bits == 8:
        assert [n for _, n in trainer.optimizer.offsets()] == [p.numel() for p in m.parameters()]


@pytest.mark.parametrize("missing", [False, True])
def test_a_refused_step_is_not_counted(missing):
    """The call refuses (a negative eps), the caller mends it: as if it had not been made."""
    a, b = params_of([300, 40], seed=2), params_of([300, 40], seed=2)
    oa, ob = AdamW(a, lr=1e-2, state_bits=8), AdamW(b, lr=1e-2, state_bits=8)
    for t in range(4):
        for ps in (a, b):
            gradients(ps, t)
            if missing and t == 1:
                ps[1].grad = None
        if t == 2:
            eps, ob.eps = ob.eps, -1.0
            with pytest.raises(RuntimeError, match="eps"):
                ob.step()
            ob.eps = eps
        oa.step()
        ob.step()
    assert oa.state_dict()["steps"] == ob.state_dict()["steps"]
    assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(a, b))
