"""AdamW against torch.optim.AdamW run in 64 bits, its 8-bit moments against their written definition (bit for bit), and
training with it.

Tolerances.  One step with 32-bit moments rounds m, v and p a few times each in FP32: with errors of a few 2^-24
relative per step, 20 steps stay below 1e-5 of the distance that the weights moved plus 1e-6 of the weights.  bf16
weights are rounded to 8 bits every step, which 64-bit weights are not: the reference is rounded the same way."""
import numpy as np
import pytest
import torch

from rnn_kernel_b200 import GRU, AdamW, DataParallelTrainer, GatedDelta, GraphedTrainStep

pytestmark = pytest.mark.gpu

SIZES = [1, 3, 255, 256, 257, 2047, 2048, 2049, 70001]


def params_of(sizes, dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(n, device="cuda").to(dtype)) for n in sizes]


def grads_of(params, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    for p in params:
        mag = torch.exp(2 * torch.randn(p.shape, device="cuda", generator=gen) - 5)
        p.grad = (torch.randn(p.shape, device="cuda", generator=gen) * mag).to(p.dtype)


@pytest.mark.parametrize("hyper", [dict(), dict(betas=(0.0, 0.5), eps=1e-3, weight_decay=0.3), dict(lr=0.0)])
def test_matches_torch(hyper):
    ps = params_of(SIZES)
    opt = AdamW(ps, **{"lr": 1e-2, **hyper})
    wide = [torch.nn.Parameter(p.detach().double()) for p in ps]
    ref = torch.optim.AdamW(wide, **{"lr": 1e-2, "weight_decay": 1e-2, **hyper})
    start = [p.detach().clone() for p in ps]
    for step in range(20):
        grads_of(ps, step)
        for p, w in zip(ps, wide):
            w.grad = p.grad.double()
        opt.step()
        ref.step()
    for p, w, s in zip(ps, wide, start):
        err = (p.detach().double() - w.detach()).abs()
        bound = 1e-5 * (w.detach() - s.double()).abs() + 1e-6 * w.detach().abs() + 1e-7
        assert bool((err <= bound).all())
    m, v = opt.moments()
    for (o, n), w in zip(opt.offsets(), wide):
        # by the norm: where gradients of both signs cancel, one element's own size says nothing of its rounding
        for got, want in ((m[o:o + n], ref.state[w]["exp_avg"]), (v[o:o + n], ref.state[w]["exp_avg_sq"])):
            assert float((got.double() - want).norm()) <= 1e-5 * float(want.norm())


def test_bf16_weights_round_once():
    ps = params_of(SIZES, torch.bfloat16)
    opt = AdamW(ps, lr=1e-2, weight_decay=0.1)
    wide = [p.detach().float() for p in ps]
    m = [torch.zeros_like(w) for w in wide]
    v = [torch.zeros_like(w) for w in wide]
    for step in range(1, 6):
        grads_of(ps, step)
        opt.step()
        for i, p in enumerate(ps):
            g = p.grad.float()
            m[i] = m[i] * 0.9 + g * (1 - 0.9)
            v[i] = v[i] * 0.999 + (g * g) * (1 - 0.999)
            den = v[i].sqrt() * (1 / np.sqrt(1 - 0.999 ** step)) + 1e-8
            wide[i] = (wide[i] * (1 - 1e-2 * 0.1) - (m[i] * (1e-2 / (1 - 0.9 ** step))) / den).bfloat16().float()
            # the same operations in the same order
            assert float((p.detach().float() - wide[i]).abs().max()) == 0


def encode_reference(x, noise, ebits):
    """8-bit codes and scales of one block (numpy float32), from their written definition."""
    x = x.astype(np.float32)
    scale = np.float32(np.abs(x).max() * np.float32(1 / 1.875))
    if scale < np.float32(2.0 ** -100):
        scale = np.float32(0)
    codes = []
    inv = np.float32(0) if scale == 0 else np.float32(1) / scale
    for xi, n in zip(x, noise):
        r = np.float32(abs(xi) * inv)
        bits = int(np.array(r).view(np.uint32)) + (int(n) << 4)
        code = min((bits >> 20) - ((128 - (1 << ebits)) << 3), (1 << (ebits + 3)) - 1)
        if ebits == 4:
            least = np.float32(2.0 ** -15 * 1.125)
            if r < least:
                code = int(r > np.float32(n) * np.float32(least / 65536))
            code |= 128 if xi < 0 else 0
        else:
            code = max(code, 1) if r > 0 else 0
        codes.append(code)
    return codes, scale


def value_reference(code, scale, ebits):
    low = code & 0x7F if ebits == 4 else code
    if low == 0:
        return np.float32(0)
    x = np.float32(2.0 ** ((low >> 3) + 1 - (1 << ebits)) * (1 + (low & 7) / 8))
    return np.float32((-x if ebits == 4 and code & 128 else x) * scale)


def noise_reference(i, seed, step):
    key = (seed * 0x8DA6B343 + step * 0xD8163841) & 0xFFFFFFFF
    h = (i * 0x9E3779B1 + key) & 0xFFFFFFFF
    h = ((h ^ (h >> 15)) * 0xB5297A4D) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0x68E31DA5) & 0xFFFFFFFF
    return h ^ (h >> 16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_8_bit_moments_follow_their_definition(dtype):
    ps = params_of([300, 5, 256], dtype)
    opt = AdamW(ps, lr=1e-2, state_bits=8, seed=77)
    f = np.float32
    n = opt.state_elems
    m, v = np.zeros(n, f), np.zeros(n, f)
    for step in range(1, 4):
        grads_of(ps, step)
        ps[2].grad[:200] *= 1e-9  # far below the block's largest
        g = np.zeros(n, f)
        for (o, k), p in zip(opt.offsets(), ps):
            g[o:o + k] = p.grad.float().cpu().numpy()
        opt.step()
        m = m * f(0.9) + g * f(1 - 0.9)
        v = v * f(0.999) + (g * g) * f(1 - 0.999)
        got_m, got_v = (t.cpu().numpy() for t in opt.moments())
        codes = opt.exp_avg.cpu().numpy(), opt.exp_avg_sq.cpu().numpy()
        for at in range(0, n, 256):
            noise = [noise_reference(at + i, 77, step) for i in range(256)]
            cm, sm = encode_reference(m[at:at + 256], [x >> 16 for x in noise], 4)
            cv, sv = encode_reference(v[at:at + 256], [x & 0xFFFF for x in noise], 5)
            assert codes[0][at:at + 256].tolist() == cm and codes[1][at:at + 256].tolist() == cv
            m[at:at + 256] = [value_reference(c, sm, 4) for c in cm]
            v[at:at + 256] = [value_reference(c, sv, 5) for c in cv]
        assert np.array_equal(m, got_m) and np.array_equal(v, got_v)


def test_8_bit_average_is_unbiased_and_does_not_stall():
    """With g constant, v tends to g^2 though one step moves it by less than half a code's distance."""
    p = torch.nn.Parameter(torch.zeros(1 << 16, device="cuda"))
    opt = AdamW([p], lr=0.0, state_bits=8, seed=3)
    p.grad = torch.ones_like(p)
    p.grad[::256] = 8.0  # every block's scale
    for _ in range(700):
        opt.step()
    _, v = opt.moments()
    rest = v.view(-1, 256)[:, 1:]
    want = 1 - 0.999 ** 700
    # a code's spread is at most 1/16 of it, random from step to step: over 65280 elements the mean is far nearer
    assert abs(float(rest.mean()) - want) <= 0.01 * want


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_tensors_give_the_same(bits):
    sizes = [257, 1000, 4097]
    a = params_of(sizes, seed=4)
    flat = torch.zeros(sum(sizes) + 1, device="cuda")
    b, at = [], 1
    for p in a:
        b.append(torch.nn.Parameter(flat[at:at + p.numel()].copy_(p.detach())))
        at += p.numel()
    oa, ob = AdamW(a, state_bits=bits), AdamW(b, state_bits=bits)
    for step in range(3):
        grads_of(a, step)
        for x, y in zip(a, b):
            y.grad = torch.cat([x.grad[:1], x.grad])[1:]
        oa.step()
        ob.step()
    for x, y in zip(a, b):
        assert torch.equal(x.detach(), y.detach())


def test_many_tensors_of_two_types_groups_and_missing_gradients():
    sizes = [1 + (37 * i) % 901 for i in range(700)]  # more than one table
    ps = [p for i, n in enumerate(sizes) for p in params_of([n], torch.bfloat16 if i % 3 == 0 else torch.float32, seed=i)]
    opt = AdamW([dict(params=ps[:300], lr=1e-2), dict(params=ps[300:], weight_decay=0.5)], lr=1e-3)
    wide = [torch.nn.Parameter(p.detach().double()) for p in ps]
    ref = torch.optim.AdamW([dict(params=wide[:300], lr=1e-2), dict(params=wide[300:], weight_decay=0.5)], lr=1e-3)
    for step in range(3):
        grads_of(ps, step)
        if step == 1:
            for p in ps[::5]:
                p.grad = None
        opt.param_groups[0]["lr"] = ref.param_groups[0]["lr"] = 1e-2 / (step + 1)
        versions = [p._version for p in ps]
        for p, w in zip(ps, wide):
            w.grad = None if p.grad is None else p.grad.double()
        opt.step()
        ref.step()
        with torch.no_grad():
            for p, w in zip(ps, wide):
                w.copy_(w.to(p.dtype) if p.dtype == torch.bfloat16 else w)
        assert all(p._version > a for p, a in zip(ps, versions))
        for p, w in zip(ps, wide):
            if p.dtype == torch.float32:
                torch.testing.assert_close(p.detach().double(), w.detach(), rtol=2e-6, atol=2e-7)
            else:
                # rounded alike every step, but for values at the middle of two
                torch.testing.assert_close(p.detach().double(), w.detach(), rtol=3 * 2.0 ** -9, atol=1e-6)


def test_gradients_that_are_not_dense():
    torch.manual_seed(5)
    ps = [torch.nn.Parameter(torch.randn(60, 80, device="cuda")) for _ in range(3)]
    wide = [torch.nn.Parameter(p.detach().double()) for p in ps]
    opt, ref = AdamW(ps), torch.optim.AdamW(wide, weight_decay=1e-2)
    for step in range(3):
        ps[0].grad = torch.randn(80, 60, device="cuda").t()
        ps[1].grad = torch.randn(1, 80, device="cuda").expand(60, 80)
        ps[2].grad = None if step == 1 else torch.randn(60, 80, device="cuda")
        for p, w in zip(ps, wide):
            w.grad = None if p.grad is None else p.grad.double()
        opt.step()
        ref.step()
    for p, w in zip(ps, wide):
        torch.testing.assert_close(p.detach().double(), w.detach(), rtol=2e-6, atol=2e-7)
    ps[0].grad = torch.sparse_coo_tensor(torch.zeros(2, 1, dtype=torch.long), torch.ones(1), (60, 80)).cuda()
    with pytest.raises(RuntimeError):
        opt.step()


def test_grad_scale_and_repeatability():
    runs = []
    for scale in (1.0, 0.25):
        ps = params_of([1000, 77], seed=6)
        opt = AdamW(ps, state_bits=8, seed=1)
        for step in range(4):
            grads_of(ps, step)
            for p in ps:
                p.grad /= scale
            opt.step(grad_scale=scale)
        runs.append([p.detach().clone() for p in ps])
    for a, b in zip(*runs):
        assert torch.equal(a, b)  # powers of two scale exactly


def test_non_finite_gradients_are_not_hidden():
    for bad in (float("nan"), float("inf")):
        for bits in (32, 8):
            ps = params_of([600], seed=7)
            opt = AdamW(ps, state_bits=bits)
            grads_of(ps, 0)
            ps[0].grad[300] = bad
            opt.step()
            assert not torch.isfinite(ps[0].detach()[300])
            assert torch.isfinite(ps[0].detach()[:256]).all()
            m, _ = opt.moments()
            assert not torch.isfinite(m[300])
            assert torch.isfinite(m[:256]).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_state_dict_resumes_bit_for_bit(bits, capturable):
    ps = params_of([513, 40], seed=8)
    opt = AdamW(ps, state_bits=bits, seed=9, capturable=capturable)
    for step in range(3):
        grads_of(ps, step)
        opt.step()
    saved, weights = opt.state_dict(), [p.detach().clone() for p in ps]
    qs = [torch.nn.Parameter(w.clone()) for w in weights]
    other = AdamW(qs, lr=5.0, state_bits=bits, capturable=capturable)
    other.load_state_dict(saved)
    for step in range(3, 6):
        grads_of(ps, step)
        grads_of(qs, step)
        opt.step()
        other.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p.detach(), q.detach())
    with pytest.raises(ValueError):
        AdamW(params_of([512, 40]), state_bits=bits).load_state_dict(saved)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_than_32_bits_of_elements(bits):
    n = 2 ** 31 + 300
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros_like(p)
    tail = torch.linspace(-1, 1, 700, device="cuda")
    p.grad[-700:] = tail.bfloat16()
    p.grad[0] = 1.0
    opt = AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits)
    opt.step()
    # the first step is lr * sign(g)
    got = p.detach()[-700:].float()
    torch.testing.assert_close(got, -1e-2 * tail.bfloat16().float().sign(), rtol=2.0 ** -8, atol=0)
    assert float(p.detach()[0]) == pytest.approx(-1e-2, rel=2.0 ** -8)
    assert int((p.detach()[:-700] != 0).sum()) == 1


def test_capturable_counts_on_the_device():
    a, b = params_of([3000], seed=10), params_of([3000], seed=10)
    oa, ob = AdamW(a), AdamW(b, capturable=True)
    grads_of(a, 0)
    b[0].grad = a[0].grad.clone()
    start = b[0].detach().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
    assert torch.equal(b[0].detach(), start)  # captured, not run
    for _ in range(5):
        oa.step()
        graph.replay()
    torch.testing.assert_close(a[0].detach(), b[0].detach(), rtol=1e-6, atol=1e-7)
    assert ob.state_dict()["calls"] == 5
    b[0].grad = None
    with pytest.raises(RuntimeError, match="gradient"):
        ob.step()


def test_refusals():
    p = params_of([10])
    with pytest.raises(ValueError, match="no parameters"):
        AdamW([])
    with pytest.raises(ValueError, match="betas"):
        AdamW(p, betas=(1.0, 0.9))
    with pytest.raises(ValueError, match="state_bits"):
        AdamW(p, state_bits=16)
    with pytest.raises(ValueError, match="once"):
        AdamW(p + p)
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([torch.randn(4, 4, device="cuda").t()])
    with pytest.raises(ValueError, match=">= 0"):
        AdamW(p, lr=-1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        AdamW([torch.zeros(3)])
    with pytest.raises(RuntimeError, match="CUDA"):
        AdamW([torch.zeros(3, device="cuda", dtype=torch.float64)])
    opt = AdamW(p)
    p[0].data = torch.zeros(11, device="cuda")
    p[0].grad = torch.zeros(11, device="cuda")
    with pytest.raises(RuntimeError, match="changed"):
        opt.step()


@pytest.mark.parametrize("make", [lambda: GRU(24, 32), lambda: GatedDelta(24, num_heads=2, head_size=16, output_size=32)])
@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_learns_with_adamw(make, bits):
    """A recurrent layer learns a fixed random target; the graphed step matches the eager one."""
    torch.manual_seed(0)
    x, y = torch.randn(8, 40, 24, device="cuda"), 0.3 * torch.randn(8, 40, 32, device="cuda")
    losses = {}
    for graphed in (False, True):
        torch.manual_seed(1)
        trainer = DataParallelTrainer(make().cuda(), lr=1e-2, optimizer="adamw", state_bits=bits)
        if graphed:
            step = GraphedTrainStep(trainer, [(x, y)], warmup=2, include_update=True)
            losses[graphed] = [float(step.step()) for _ in range(38)]
        else:
            losses[graphed] = [float(trainer.step(x, y)) for _ in range(40)][2:]
    assert losses[False][-1] < 0.8 * losses[False][0]
    np.testing.assert_allclose(losses[True], losses[False], rtol=1e-3)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_become_others_in_the_same_place_are_refused(bits):
    """A new .data may begin where the old one did, with other sizes or strides."""
    def fresh():
        p = [torch.nn.Parameter(torch.randn(12, 30, device="cuda")), torch.nn.Parameter(torch.randn(7, device="cuda"))]
        opt = AdamW(p, lr=0.1, state_bits=bits)
        for x in p:
            x.grad = torch.randn_like(x)
        opt.step()
        return p, opt

    for change in (lambda x: x.t(), lambda x: x[:5], lambda x: x[:, :10]):
        p, opt = fresh()
        p[0].grad = None
        p[0].data = change(p[0].data)
        p[0].grad = torch.randn(p[0].shape, device="cuda")
        before = [x.detach().clone() for x in p]
        with pytest.raises(RuntimeError, match="changed|size"):
            opt.step()
        assert all(torch.equal(a, b) for a, b in zip(before, p))

