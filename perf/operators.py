"""Measured cases of the gated delta rule (chunked forward, gradient, single-token step) and of the multi-tensor AdamW
step with 32- or 8-bit moments.

The gated delta rule keeps a matrix state S [dk, dv] per sequence and value head.  Token t, with decay a = exp(g_t):

    S' = a S;   u = beta_t (v_t - S'^T k_t);   S = S' + k_t u^T;   o_t = scale * S^T q_t

``own`` selects the framework's calls; otherwise the plain form in elementary 32-bit torch operations runs: the rule
over chunks of 64 tokens (the only loop is the one over chunks, which depend on one another), autograd for the
gradient, and AdamW as whole-buffer elementwise operations.
"""
import math

import torch
import torch.nn.functional as F

own = False

CHUNK = 64          # tokens per chunk of the plain form
BLOCK = 256         # elements that share one scale of an 8-bit moment; every tensor starts a new block
BETAS, EPS, LR, DECAY = (0.9, 0.999), 1e-8, 1e-3, 0.01
SEED = 12345        # of the 8-bit moments' stochastic rounding

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one user's token: latency of a serving step (16 value heads of 128 x 128 sharing 8 key heads)
        dict(name="step one sequence", kind="step", B=1, Hk=8, Hv=16, dk=128, dv=128, dtype="bfloat16"),
        # a serving batch's token: the states are read and written once
        dict(name="step batch of 64", kind="step", B=64, Hk=16, Hv=32, dk=128, dv=128, dtype="bfloat16"),
        # odd head sizes, three value heads to a key head, 32-bit inputs
        dict(name="step odd heads", kind="step", B=7, Hk=2, Hv=6, dk=96, dv=81, dtype="float32"),
        # a short prompt that ends inside its second chunk
        dict(name="prompt of 77", kind="forward", B=1, T=77, Hk=4, Hv=8, dk=64, dv=64, dtype="bfloat16"),
        # a long document's prompt: one sequence, all parallelism from heads and value columns
        dict(name="prompt of 16384", kind="forward", B=1, T=16384, Hk=16, Hv=32, dk=128, dv=128, dtype="bfloat16"),
        # the framework's benchmark sequence (batch 64, 512 steps, width 256 as 4 heads of 64) in its own 32 bits
        dict(name="train 64 x 512 x 256", kind="train", B=64, T=512, Hk=4, Hv=4, dk=64, dv=64, dtype="float32"),
        # a language model's layer: two value heads to a key head, 16-bit activations
        dict(name="train 4 x 2048", kind="train", B=4, T=2048, Hk=8, Hv=16, dk=128, dv=128, dtype="bfloat16"),
        # nothing a multiple of anything: 5 chunks and 13 tokens, head sizes that are no tile's
        dict(name="train odd 3 x 333", kind="train", B=3, T=333, Hk=2, Hv=2, dk=40, dv=72, dtype="float32"),
        # the weights of the benchmark's GRU (input and hidden 256, 2 layers) and a linear head: nine small tensors
        dict(name="adamw gru 2 layers", kind="adamw", shape="gru", layers=2, width=256, bits=32, dtype="float32"),
        # 200 tensors of odd sizes, 16-bit weights with 8-bit moments
        dict(name="adamw8 200 odd tensors", kind="adamw", shape="odd", layers=200, width=600011, bits=8, dtype="bfloat16"),
        # a model's worth of weights: the step is bound by memory
        dict(name="adamw 200M", kind="adamw", shape="blocks", layers=16, width=1024, bits=32, dtype="float32"),
        dict(name="adamw8 200M", kind="adamw", shape="blocks", layers=16, width=1024, bits=8, dtype="float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "forward", "train", "train", "adamw"])
    if kind == "adamw":
        bits, dtype = rng.choice([32, 8]), rng.choice(["float32", "bfloat16"])
        shape = rng.choice(["gru", "odd", "blocks"])
        if shape == "gru":
            return dict(kind=kind, shape=shape, layers=rng.randint(1, 6), width=rng.randint(33, 256), bits=bits, dtype=dtype)
        if shape == "odd":
            return dict(kind=kind, shape=shape, layers=_log(rng, 10, 400), width=_log(rng, 50, 1000000), bits=bits, dtype=dtype)
        return dict(kind=kind, shape=shape, layers=rng.randint(2, 16), width=8 * rng.randint(16, 128), bits=bits, dtype=dtype)
    dtype = rng.choice(["float32", "bfloat16"])
    Hk = rng.choice([1, 2, 4, 8])
    Hv = Hk * rng.choice([1, 1, 2, 3])
    if rng.random() < 0.5:
        dk = dv = rng.choice([64, 128])
    else:
        dk, dv = rng.randint(16, 128), rng.randint(16, 128)
    case = dict(kind=kind, B=1, Hk=Hk, Hv=Hv, dk=dk, dv=dv, dtype=dtype)
    if kind == "step":
        case["B"] = _log(rng, 1, 80)
        return case
    most = 500_000 if kind == "forward" else 120_000     # tokens x value heads
    case["T"] = max(1, min(_log(rng, 1, 16384 if kind == "forward" else 4096), most // Hv))
    case["B"] = _log(rng, 1, max(1, min(64, most // (Hv * case["T"]))))
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------


def _tensor_sizes(case):
    n, w = case["layers"], case["width"]
    if case["shape"] == "gru":
        sizes = [s for _ in range(n) for s in (3 * w * w, 3 * w * w, 3 * w, 3 * w)]
        return sizes + [w]
    if case["shape"] == "odd":
        # sizes over three orders of magnitude, from single elements up; odd ones mostly
        return [1 + (7919 * (i + 1) * (i + 3)) % max(2, w // (1 + i % 17) ** 2) for i in range(n)]
    # a block: four w x w projections, a gated 4 w wide pair and its way back, two norms
    return [s for _ in range(n) for s in (w * w, w * w, w * w, w * w, 4 * w * w, 4 * w * w, w, w)]


def _spans(sizes):
    """(start, size) of each tensor in a buffer where every tensor starts a block, and the buffer's length."""
    at, spans = 0, []
    for s in sizes:
        spans.append((at, s))
        at += -(-s // BLOCK) * BLOCK
    return spans, at


def _delta_inputs(case, seed, T):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, B, Hk, Hv, dk, dv = TYPES[case["dtype"]], case["B"], case["Hk"], case["Hv"], case["dk"], case["dv"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    q = F.normalize(normal(B, T, Hk, dk), dim=-1).to(dt)
    k = F.normalize(normal(B, T, Hk, dk) + 0.5 * normal(B, 1, Hk, dk), dim=-1).to(dt)
    v = normal(B, T, Hv, dv).to(dt)
    # per-head decay rates from long memory to a few tokens, as a layer learns them
    rate = torch.exp(torch.rand(Hv, device="cuda", generator=gen) * 5.0 - 5.0)
    g = -rate * F.softplus(normal(B, T, Hv))
    beta = torch.sigmoid(normal(B, T, Hv))
    s0 = 0.3 * normal(B, Hv, dk, dv)
    return gen, q, k, v, g, beta, s0


def prepare(case, seed):
    if case["kind"] == "adamw":
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        spans, n = _spans(_tensor_sizes(case))
        dt = TYPES[case["dtype"]]
        real = torch.zeros(n, dtype=torch.bool, device="cuda")
        for a, s in spans:
            real[a:a + s] = True
        flat = torch.where(real, 0.05 * torch.randn(n, device="cuda", generator=gen), 0.0).to(dt)
        # gradients spread over some decades inside a tensor, a few exactly zero
        mag = torch.exp(2.0 * torch.randn(n, device="cuda", generator=gen) - 7.0)
        grad = torch.randn(n, device="cuda", generator=gen) * mag
        grad = torch.where(real & (torch.rand(n, device="cuda", generator=gen) > 0.01), grad, 0.0).to(dt)
        del mag, real
        state = dict(case=case, flat=flat, grad=grad)
        if own:
            from rnn_kernel_b200 import AdamW

            params = []
            for a, s in spans:
                p = torch.nn.Parameter(flat[a:a + s])
                p.grad = grad[a:a + s]
                params.append(p)
            state["opt"] = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"], seed=SEED)
        else:
            state.update(step=0, m=torch.zeros(n, device="cuda"), v=torch.zeros(n, device="cuda"))
            if case["bits"] == 8:
                state.update(m=torch.zeros(n, dtype=torch.uint8, device="cuda"), v=torch.zeros(n, dtype=torch.uint8, device="cuda"),
                             sm=torch.zeros(n // BLOCK, device="cuda"), sv=torch.zeros(n // BLOCK, device="cuda"))
        return state
    if case["kind"] == "step":
        _, q, k, v, g, beta, s0 = _delta_inputs(case, seed, 1)
        return dict(case=case, q=q[:, 0], k=k[:, 0], v=v[:, 0], g=g[:, 0], beta=beta[:, 0], state=s0)
    gen, q, k, v, g, beta, s0 = _delta_inputs(case, seed, case["T"])
    state = dict(case=case, q=q, k=k, v=v, g=g, beta=beta, s0=s0)
    if case["kind"] == "train":
        for name in ("q", "k", "v", "g", "beta", "s0"):
            state[name].requires_grad_(True)
        state["do"] = torch.randn(v.shape, device="cuda", generator=gen).to(v.dtype)
        state["ds"] = 0.3 * torch.randn(s0.shape, device="cuda", generator=gen)
    return state


# ---- plain forms --------------------------------------------------------------------------------------------------


def _plain_rule(q, k, v, g, beta, s0):
    """The rule over chunks; returns out [B, T, Hv, dv] in v's type and the last state."""
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2], v.shape[3]
    C, n = CHUNK, -(-T // CHUNK)
    scale = dk ** -0.5

    def chunks(x):
        # [B, T, H, ...] -> [n, B * Hv, C, ...] in 32 bits, zeros after the last token
        x = x.float()
        if x.shape[2] != Hv:
            x = x.repeat_interleave(Hv // Hk, dim=2)
        x = F.pad(x, (0, 0) * (x.dim() - 2) + (0, n * C - T))
        x = x.reshape((B, n, C) + x.shape[2:])
        return x.movedim(3, 1).transpose(1, 2).movedim(1, 0).flatten(1, 2)

    q, k, v, g, beta = chunks(q), chunks(k), chunks(v), chunks(g), chunks(beta)
    gc = g.cumsum(-1)
    lower = torch.ones(C, C, dtype=torch.bool, device=q.device).tril()
    strict = lower.tril(-1)
    decay = (gc[..., :, None] - gc[..., None, :]).masked_fill(~lower, -math.inf).exp()
    a = (k @ k.transpose(-1, -2)) * decay * beta[..., None] * strict
    # (I + a)^-1 by doubling the size of the inverted diagonal blocks
    inv = torch.eye(C, device=q.device).expand_as(a)
    i = torch.arange(C, device=q.device)
    size = 1
    while size < C:
        below = ((i[:, None] // size) % 2 == 1) & (i[:, None] // size == i[None, :] // size + 1)
        inv = inv - inv @ (a * below) @ inv
        size *= 2
    p = (q @ k.transpose(-1, -2)) * decay * scale
    up = gc.exp()[..., None]
    rest = (gc[..., -1:] - gc).exp()[..., None]
    bv, bk = beta[..., None] * v, beta[..., None] * up * k
    u0, w = inv @ bv, inv @ bk
    s, outs = s0.flatten(0, 1), []
    for c in range(n):
        u = u0[c] - w[c] @ s
        outs.append((scale * up[c] * q[c]) @ s + p[c] @ u)
        s = up[c][:, -1:] * s + (rest[c] * k[c]).transpose(-1, -2) @ u
    out = torch.stack(outs, 1).reshape(B, Hv, n * C, dv)[:, :, :T].transpose(1, 2)
    return out, s.reshape(B, Hv, dk, dv)


def _plain_step(st):
    s, q, k, v = st["state"], st["q"].float(), st["k"].float(), st["v"].float()
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, dim=1), k.repeat_interleave(rep, dim=1)
    new = s * st["g"].exp()[..., None, None]
    u = st["beta"][..., None] * (v - (new * k[..., None]).sum(-2))
    new = new + k[..., None] * u[..., None, :]
    s.copy_(new)
    return ((new * q[..., None]).sum(-2) * q.shape[-1] ** -0.5).to(st["v"].dtype)


def _u(x, bits):
    """x, an int32 tensor, shifted right by `bits` as an unsigned number."""
    return (x >> bits) & ((1 << (32 - bits)) - 1)


def _wrap(c):
    return c - (1 << 32) if c >= 1 << 31 else c


def _noise(n, step, device):
    """32 random bits per element from (seed, step, position): the definition of the 8-bit moments' rounding."""
    key = (SEED * 0x8DA6B343 + step * 0xD8163841) & 0xFFFFFFFF
    h = torch.arange(n, dtype=torch.int32, device=device) * _wrap(0x9E3779B1) + _wrap(key)
    h = (h ^ _u(h, 15)) * _wrap(0xB5297A4D)
    h = (h ^ _u(h, 13)) * 0x68E31DA5
    return h ^ _u(h, 16)


def _decode(code, scale, exponent_bits):
    """8-bit codes as numbers: 3 mantissa bits, the largest code 1.875 times the block's scale, code 0 zero."""
    code = code.to(torch.int32)
    low = code & 0x7F if exponent_bits == 4 else code
    x = ((low << 20) + ((128 - (1 << exponent_bits)) << 23)).view(torch.float32)
    x = torch.where(low == 0, 0.0, x)
    if exponent_bits == 4:
        x = torch.where(code > 127, -x, x)
    return (x.reshape(-1, BLOCK) * scale[:, None]).reshape(-1)


def _encode(x, noise16, exponent_bits):
    """Numbers as 8-bit codes and block scales, rounded up or down at random in proportion to the distance."""
    x = x.reshape(-1, BLOCK)
    a = x.abs()
    scale = a.amax(1) * torch.tensor(1.0 / 1.875, device=x.device)
    scale = torch.where(scale < 2.0 ** -100, 0.0, scale)
    inv = torch.where(scale == 0, 0.0, 1.0 / scale)
    r = (a * inv[:, None]).reshape(-1)
    least = 2.0 ** (1 - (1 << exponent_bits)) * 1.125
    low = ((r.view(torch.int32) + (noise16 << 4)) >> 20) - ((128 - (1 << exponent_bits)) << 3)
    low = low.clamp(max=(1 << (exponent_bits + 3)) - 1)
    if exponent_bits == 4:      # first moment: below the least code to it or to zero, at random
        low = torch.where(r < least, (r > noise16.float() * (least / 65536.0)).int(), low)
        code = torch.where(x.reshape(-1) < 0, low + 128, low)
    else:                       # second moment: never rounded to zero, it divides
        low = low.clamp(min=1)
        code = torch.where(r > 0, low, 0)
    return code.to(torch.uint8), scale


def _plain_adamw(st):
    bits = st["case"]["bits"]
    st["step"] += 1
    t = st["step"]
    b1, b2 = BETAS
    g, p = st["grad"].float(), st["flat"].float()
    m, v = st["m"], st["v"]
    if bits == 8:
        m, v = _decode(m, st["sm"], 4), _decode(v, st["sv"], 5)
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    step = LR / (1.0 - b1 ** t)
    den = v.sqrt() * (1.0 / math.sqrt(1.0 - b2 ** t)) + EPS
    p = p * (1.0 - LR * DECAY) - (m * step) / den
    st["flat"].copy_(p)
    if bits == 32:
        st["m"], st["v"] = m, v
        return st["flat"], m, v
    noise = _noise(m.numel(), t, m.device)
    st["m"], st["sm"] = _encode(m, _u(noise, 16), 4)
    st["v"], st["sv"] = _encode(v, noise & 0xFFFF, 5)
    return st["flat"], _decode(st["m"], st["sm"], 4), _decode(st["v"], st["sv"], 5)


# ---- one pass -----------------------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if kind == "adamw":
        if own:
            state["opt"].step()
            m, v = state["opt"].moments()
            return state["flat"], m, v
        return _plain_adamw(state)
    if kind == "step":
        if own:
            from rnn_kernel_b200 import gated_delta_step

            o = gated_delta_step(state["q"], state["k"], state["v"], state["g"], state["beta"], state["state"])
        else:
            o = _plain_step(state)
        return o, state["state"]
    args = [state[n] for n in ("q", "k", "v", "g", "beta", "s0")]
    if kind == "forward":
        with torch.no_grad():
            if own:
                from rnn_kernel_b200 import gated_delta_rule

                return gated_delta_rule(*args[:5], initial_state=args[5])
            o, s = _plain_rule(*args)
            return o.to(state["v"].dtype), s
    if own:
        from rnn_kernel_b200 import gated_delta_rule

        o, s = gated_delta_rule(*args[:5], initial_state=args[5])
        grads = torch.autograd.grad((o, s), args, (state["do"], state["ds"]))
    else:
        # inputs widened first, so that every gradient is rounded to its input's type once, at the end
        wide = [a.detach().float().requires_grad_(True) for a in args]
        o, s = _plain_rule(*wide)
        grads = torch.autograd.grad((o, s), wide, (state["do"].float(), state["ds"]))
        grads = [d.to(a.dtype) for d, a in zip(grads, args)]
        o = o.detach().to(state["v"].dtype)
    return (o.detach(), s.detach(), *grads)


# ---- 64 bits ------------------------------------------------------------------------------------------------------


def _exact_rule(q, k, v, g, beta, s0, do=None, ds=None):
    """Token by token in 64 bits; with `do` and `ds` the gradients too, by the reversed recurrence."""
    B, T, Hk, dk = q.shape
    Hv = v.shape[2]
    rep, scale = Hv // Hk, dk ** -0.5
    q, k = (x.double().repeat_interleave(rep, dim=2) for x in (q, k))
    v, g, beta, s = v.double(), g.double(), beta.double(), s0.double()

    def token(s, t):
        kt = k[:, t, :, :, None]
        sd = s * g[:, t].exp()[..., None, None]
        e = v[:, t] - (sd * kt).sum(-2)
        return sd, e, sd + kt * (beta[:, t, :, None] * e)[..., None, :]

    out, marks, seg = torch.empty_like(v), [], 32
    for t in range(T):
        if do is not None and t % seg == 0:
            marks.append(s)
        _, _, s = token(s, t)
        out[:, t] = (s * q[:, t, :, :, None]).sum(-2) * scale
    if do is None:
        return out, s
    d, last = ds.double(), s
    dq, dkk, dvv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dg, db = torch.zeros_like(g), torch.zeros_like(beta)
    for first in reversed(range(0, T, seg)):
        s, kept = marks[first // seg], []
        for t in range(first, min(T, first + seg)):
            kept.append(token(s, t))
            s = kept[-1][2]
        for t in reversed(range(first, min(T, first + seg))):
            sd, e, s = kept[t - first]
            dot = do[:, t].double() * scale
            dq[:, t] = (s * dot[..., None, :]).sum(-1)
            d = d + q[:, t, :, :, None] * dot[..., None, :]
            du = (d * k[:, t, :, :, None]).sum(-2)
            b = beta[:, t, :, None]
            dvv[:, t] = b * du
            db[:, t] = (du * e).sum(-1)
            dkk[:, t] = (d * (b * e)[..., None, :]).sum(-1) - (sd * (b * du)[..., None, :]).sum(-1)
            d = d - k[:, t, :, :, None] * (b * du)[..., None, :]
            dg[:, t] = (d * sd).sum((-1, -2))
            d = d * g[:, t].exp()[..., None, None]
    dq, dkk = (x.reshape(B, T, Hk, rep, dk).sum(3) for x in (dq, dkk))
    return out, last, dq, dkk, dvv, dg, db, d


def exact(case, seed):
    global own
    was, own = own, False      # the inputs alone: no handle of the framework's
    try:
        st = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        if case["kind"] == "adamw":
            p, g = st["flat"].double(), st["grad"].double()
            b1, b2 = BETAS
            m, v = (1 - b1) * g, (1 - b2) * g * g
            p = p - LR * DECAY * p - LR * (m / (1 - b1)) / ((v / (1 - b2)).sqrt() + EPS)
            return (p, m, v) if case["bits"] == 32 else (p, None, None)
        if case["kind"] == "step":
            one = [st[n].unsqueeze(1) for n in ("q", "k", "v", "g", "beta")]
            out, s = _exact_rule(*one, st["state"])
            return out[:, 0], s
        args = [st[n].detach() for n in ("q", "k", "v", "g", "beta", "s0")]
        return _exact_rule(*args, *((st["do"], st["ds"]) if case["kind"] == "train" else ()))


# ---- work ---------------------------------------------------------------------------------------------------------


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "adamw":
        n = sum(_tensor_sizes(case))
        # weight read and written, gradient read, moments read and written; 8-bit ones are also written out widened,
        # since a pass returns the values that they stand for
        states = 16 if case["bits"] == 32 else 4 + 16.0 / BLOCK + 8
        return {"bytes": n * (3 * e + states), "flops": 14 * n}
    B, Hk, Hv, dk, dv = (case[x] for x in ("B", "Hk", "Hv", "dk", "dv"))
    T = case.get("T", 1)
    state = 4 * B * Hv * dk * dv
    qk, vo, gb = 2 * B * T * Hk * dk * e, 2 * B * T * Hv * dv * e, 8 * B * T * Hv
    if case["kind"] != "train":
        return {"bytes": qk + vo + gb + 2 * state, "flops": 7 * B * T * Hv * dk * dv}
    # forward, then: out's gradient read, every input's written, and the states' both
    return {"bytes": (qk + vo + gb + 2 * state) + (qk + vo + gb + 2 * state), "flops": 21 * B * T * Hv * dk * dv}
