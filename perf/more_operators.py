"""Measured cases of the selective state space scan (all tokens, gradient, single-token step), of the short causal
convolution in front of it (the same three), and of layer normalisation with the residual sum (forward, gradient).

The scan keeps N numbers per sequence and channel d; group g = d // (D / G) shares B and C.  Token t, with dt_t[d] > 0:

    h[n] = exp(dt_t A[d, n]) h[n] + dt_t x_t[d] B_t[g, n];   y_t[d] = sum_n C_t[g, n] h[n] + skip[d] x_t[d]

and y_t[d] silu(z_t[d]) leaves where a gate z is given; dt_t = softplus(raw_t + bias[d]).  The convolution of width W is
y_t = silu(bias + sum_j w[:, j] x_(t - W + 1 + j)), tokens before the first from a state of the last W - 1 inputs.  Layer
normalisation takes s = x + residual, in the residual's type, and gives (s - mean) / sqrt(variance + eps) w + b beside s.

``own`` selects the framework's calls; otherwise the plain form in elementary 32-bit torch operations runs: the scan by
doubling inside chunks of 64 tokens and over the chunks one after another, autograd for the gradients.
"""
import math

import torch
import torch.nn.functional as F

own = False

CHUNK = 64          # tokens per chunk of the plain scan
EPS = 1e-5

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one user's token through a layer of 2048 channels: latency of a serving step
        dict(name="scan step one sequence", kind="scan step", B=1, D=2048, N=16, G=1, gate=True, dtype="bfloat16"),
        # a serving batch's token: the states are read and written once
        dict(name="scan step batch of 256", kind="scan step", B=256, D=4096, N=16, G=1, gate=True, dtype="bfloat16"),
        # a short prompt through a narrow layer
        dict(name="scan prompt of 77", kind="scan forward", B=1, T=77, D=512, N=16, G=1, gate=True, dtype="bfloat16"),
        # a long document's prompt: one sequence, parallelism from channels and pieces of the time
        dict(name="scan prompt of 16384", kind="scan forward", B=1, T=16384, D=2048, N=16, G=1, gate=True, dtype="bfloat16"),
        # the framework's benchmark sequence (batch 64, 512 steps, width 256, here doubled inside the layer) in 32 bits
        dict(name="scan train 64 x 512", kind="scan train", B=64, T=512, D=512, N=16, G=1, gate=True, dtype="float32"),
        # a language model's layer, 16-bit activations
        dict(name="scan train 4 x 2048", kind="scan train", B=4, T=2048, D=2048, N=16, G=1, gate=True, dtype="bfloat16"),
        # nothing a multiple of anything: odd tokens, states, channels per group, no gate
        dict(name="scan train odd 3 x 333", kind="scan train", B=3, T=333, D=141, N=10, G=3, gate=False, dtype="float32"),
        # the convolution of a serving batch's token
        dict(name="conv step batch of 256", kind="conv step", B=256, D=4096, W=4, wtype="float32", dtype="bfloat16"),
        # the convolution of a language model's layer
        dict(name="conv train 4 x 2048", kind="conv train", B=4, T=2048, D=4096, W=4, wtype="float32", dtype="bfloat16"),
        # one user's token through the norm in front of a layer: latency
        dict(name="norm one token", kind="norm forward", R=1, D=1024, residual="bfloat16", wtype="bfloat16", dtype="bfloat16"),
        # the framework's benchmark activations (64 x 512 rows of 256)
        dict(name="norm train 32768 x 256", kind="norm train", R=32768, D=256, residual=None, wtype="float32", dtype="float32"),
        # a language model's block: 16-bit activations, the sum of the residual stream beside the norm
        dict(name="norm train 8192 x 2048", kind="norm train", R=8192, D=2048, residual="bfloat16", wtype="float32",
             dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan step", "scan forward", "scan train", "scan train", "conv step", "conv forward", "conv train",
                       "norm forward", "norm train"])
    dtype = rng.choice(["float32", "bfloat16"])
    wtype = rng.choice(["float32", dtype])
    if kind.startswith("norm"):
        D = rng.choice([_log(rng, 8, 8192), 8 * _log(rng, 2, 1024)])
        R = max(1, min(_log(rng, 1, 100_000), 16_000_000 // D))
        return dict(kind=kind, R=R, D=D, residual=rng.choice([None, dtype, "float32"]), wtype=wtype, dtype=dtype)
    if kind.startswith("conv"):
        D, W = rng.choice([_log(rng, 1, 6000), 8 * _log(rng, 2, 512)]), rng.choice([2, 3, 4, 4, 4, rng.randint(5, 8)])
        case = dict(kind=kind, B=_log(rng, 1, 256), D=D, W=W, wtype=wtype, dtype=dtype)
        if kind != "conv step":
            case["T"] = max(1, min(_log(rng, 1, 16384), 32_000_000 // D))
            case["B"] = _log(rng, 1, max(1, min(64, 32_000_000 // (D * case["T"]))))
        return case
    N = rng.choice([16, 16, rng.randint(1, 64)])
    G = rng.choice([1, 1, 2, 3, 4])
    D = G * rng.choice([_log(rng, 8, 1000), 32 * rng.randint(1, 32)])
    case = dict(kind=kind, B=_log(rng, 1, 256), D=D, N=N, G=G, gate=rng.random() < 0.7, dtype=dtype)
    if kind == "scan step":
        case["B"] = max(1, min(case["B"], 16_000_000 // (D * N)))
        return case
    most = (500_000_000 if kind == "scan forward" else 130_000_000) // (D * N)      # tokens
    case["T"] = max(1, min(_log(rng, 1, 16384 if kind == "scan forward" else 4096), most))
    case["B"] = _log(rng, 1, max(1, min(64, most // case["T"])))
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------


def _direction(case):
    return case["kind"].split()[1]


def _norm_inputs(case, gen, normal):
    R, D, dt = case["R"], case["D"], TYPES[case["dtype"]]
    # rows of different sizes, each with an offset of its own
    x = (torch.exp(normal(R, 1)) * normal(R, D) + 0.5 * normal(R, 1)).to(dt)
    w, b = ((one + 0.1 * normal(D)).to(TYPES[case["wtype"]]) for one in (1.0, 0.0))
    state = dict(x=x, weight=w, bias=b)
    if case["residual"]:
        state["residual"] = (2.0 * normal(R, D)).to(TYPES[case["residual"]])
    if _direction(case) == "train":
        state["dy"] = normal(R, D).to(dt)
        if case["residual"]:
            state["ds"] = normal(R, D).to(TYPES[case["residual"]])
    return state


def _conv_inputs(case, gen, normal):
    B, D, W, dt, wt = case["B"], case["D"], case["W"], TYPES[case["dtype"]], TYPES[case["wtype"]]
    T = () if _direction(case) == "step" else (case["T"],)
    state = dict(x=normal(B, *T, D).to(dt), weight=(W ** -0.5 * normal(D, W)).to(wt), bias=(0.1 * normal(D)).to(wt),
                 state=normal(B, W - 1, D).to(dt))
    if _direction(case) == "train":
        state.update(dy=normal(B, *T, D).to(dt), ds=normal(B, W - 1, D).to(dt))
    return state


def _scan_inputs(case, gen, normal):
    B, D, N, G, dt = case["B"], case["D"], case["N"], case["G"], TYPES[case["dtype"]]
    T = () if _direction(case) == "step" else (case["T"],)
    # channels that remember from ten tokens to a thousand, decay rates that grow with the state's index
    start = torch.exp(torch.rand(D, device="cuda", generator=gen) * math.log(100.0) + math.log(1e-3))
    state = dict(x=normal(B, *T, D).to(dt), dt=(0.7 * normal(B, *T, D)).to(dt), bm=normal(B, *T, G, N).to(dt),
                 cm=normal(B, *T, G, N).to(dt), a=-torch.arange(1, N + 1, device="cuda") * torch.exp(0.3 * normal(D, N)),
                 skip=1.0 + 0.1 * normal(D), bias=torch.log(torch.expm1(start)), s0=normal(B, D, N))
    if case["gate"]:
        state["z"] = normal(B, *T, D).to(dt)
    if _direction(case) == "train":
        state.update(dy=normal(B, *T, D).to(dt), ds=0.3 * normal(B, D, N))
    return state


LEAVES = {"norm": ("x", "residual", "weight", "bias"), "conv": ("x", "weight", "bias", "state"),
          "scan": ("x", "dt", "a", "bm", "cm", "skip", "z", "bias", "s0")}


def _leaves(state):
    return [n for n in LEAVES[state["case"]["kind"].split()[0]] if n in state]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    make = {"norm": _norm_inputs, "conv": _conv_inputs, "scan": _scan_inputs}[case["kind"].split()[0]]
    state = dict(make(case, gen, normal), case=case)
    if _direction(case) == "train":
        for n in _leaves(state):
            state[n].requires_grad_(True)
    return state


# ---- plain forms ----------------------------------------------------------------------------------------------------


def _plain_norm(x, residual, weight, bias, kept):
    """The norm of s, and s as the residual stream of type `kept` has it (None: no residual, s is x)."""
    s = x
    if kept is not None:
        s = x + residual
        s = s + (s.to(kept).float() - s).detach()       # the stream's rounding, which a gradient passes as it is
    c = s - s.mean(-1, keepdim=True)
    y = c / (c.square().mean(-1, keepdim=True) + EPS).sqrt() * weight + bias
    return (y,) if kept is None else (y, s)


def _plain_conv(x, weight, bias, state):
    """All tokens; also the state after them, as it is stored."""
    T, W = x.shape[1], weight.shape[1]
    padded = torch.cat([state, x], 1)
    windows = padded.unfold(1, W, 1)                            # [B, T, D, W], a view
    y = (windows * weight).sum(-1) + bias
    return y * torch.sigmoid(y), padded[:, T:]


def _plain_scan(x, dt, a, bm, cm, skip, z, bias, s0):
    B, T, D = x.shape
    G, N = bm.shape[2:]
    C = min(CHUNK, 1 << (T - 1).bit_length())
    n, R = -(-T // C), D // G
    raw = dt + bias
    step = torch.where(raw > 20.0, raw, torch.log1p(torch.exp(raw.clamp(max=20.0))))

    def chunks(t, *last):
        return F.pad(t, (0, 0) * (t.dim() - 2) + (0, n * C - T)).reshape(B, n, C, G, *last)

    sc = chunks(step, R, 1)
    h = chunks(step * x, R, 1) * chunks(bm, 1, N)               # what each token adds
    p = torch.exp(sc * a.reshape(G, R, N))                      # and leaves of what was
    size = 1
    while size < C:         # h, p: of the last 2 size tokens
        h = torch.cat([h[:, :, :size], h[:, :, size:] + p[:, :, size:] * h[:, :, :-size]], 2)
        p = torch.cat([p[:, :, :size], p[:, :, size:] * p[:, :, :-size]], 2)
        size *= 2
    s, starts = s0.reshape(B, G, R, N), []
    for c in range(n):
        starts.append(s)
        s = p[:, c, -1] * s + h[:, c, -1]
    h = h + p * torch.stack(starts, 1)[:, :, None]
    y = (h * chunks(cm, 1, N)).sum(-1).reshape(B, n * C, D)[:, :T] + skip * x
    if z is not None:
        y = y * z * torch.sigmoid(z)
    return y, s.reshape(B, D, N)


def _second(state):
    """The type of the output beside y: the sum, or the last state."""
    return state["residual"].dtype if "residual" in state else state["state"].dtype if "state" in state else torch.float32


def _plain(state, get):
    """The operator's outputs in 32 bits from `get(name)`: a tensor in 32 bits, or None."""
    kind = state["case"]["kind"]
    if kind.startswith("norm"):
        return _plain_norm(*(get(n) for n in LEAVES["norm"]), _second(state) if "residual" in state else None)
    if kind.startswith("conv"):
        return _plain_conv(*(get(n) for n in LEAVES["conv"]))
    return _plain_scan(*(get(n) for n in LEAVES["scan"]))


def _plain_run(state):
    dtypes = (state["x"].dtype, _second(state))
    if _direction(state["case"]) == "train":
        # inputs widened first, so that every gradient is rounded to its input's type once, at the end
        wide = {n: state[n].detach().float().requires_grad_(True) for n in _leaves(state)}
        outs = _plain(state, wide.get)
        got = torch.autograd.grad(outs, list(wide.values()), [state[n].float() for n in ("dy", "ds") if n in state])
        return (*(o.detach().to(t) for o, t in zip(outs, dtypes)), *(g.to(state[n].dtype) for g, n in zip(got, wide)))
    with torch.no_grad():
        wide = {n: state[n].float() for n in _leaves(state)}
        if _direction(state["case"]) == "forward":
            return tuple(o.to(t) for o, t in zip(_plain(state, wide.get), dtypes))
        # one token is a sequence of one; the state is updated where it is
        wide.update({n: wide[n].unsqueeze(1) for n in ("x", "dt", "bm", "cm", "z") if n in wide})
        y, s = _plain(state, wide.get)
        held = state["state" if "state" in state else "s0"]
        held.copy_(s)
        return y[:, 0].to(dtypes[0]), held


# ---- one pass -----------------------------------------------------------------------------------------------------


def _own_forward(state):
    from rnn_kernel_b200 import causal_conv, layer_norm, selective_scan

    kind = state["case"]["kind"]
    if kind.startswith("norm"):
        got = layer_norm(state["x"], state["weight"], state["bias"], eps=EPS, residual=state.get("residual"))
        return got if "residual" in state else (got,)
    if kind.startswith("conv"):
        return causal_conv(state["x"], state["weight"], state["bias"], activation="silu", initial_state=state["state"])
    return selective_scan(state["x"], state["dt"], state["a"], state["bm"], state["cm"], skip=state["skip"], z=state.get("z"),
                          dt_bias=state["bias"], dt_softplus=True, initial_state=state["s0"])


def _own_run(state):
    from rnn_kernel_b200 import causal_conv_step, selective_step

    kind, case = state["case"]["kind"], state["case"]
    if kind == "conv step":
        y = causal_conv_step(state["x"], state["weight"], state["state"], state["bias"], activation="silu")
        return y, state["state"]
    if kind == "scan step":
        y = selective_step(state["x"], state["dt"], state["a"], state["bm"], state["cm"], state["s0"], skip=state["skip"],
                           z=state.get("z"), dt_bias=state["bias"], dt_softplus=True)
        return y, state["s0"]
    if _direction(case) == "forward":
        with torch.no_grad():
            return _own_forward(state)
    outs = _own_forward(state)
    grads = [state[n] for n in ("dy", "ds") if n in state]
    got = torch.autograd.grad(outs, [state[n] for n in _leaves(state)], grads)
    return (*(o.detach() for o in outs), *got)


def run(state):
    return _own_run(state) if own else _plain_run(state)


# ---- 64 bits ------------------------------------------------------------------------------------------------------


def _exact_norm(st):
    x, w, b = st["x"].double(), st["weight"].double(), st["bias"].double()
    kept = st["residual"].dtype if "residual" in st else None
    s = (x + st["residual"].double()).to(kept).double() if kept else x
    c = s - s.mean(-1, keepdim=True)
    r = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
    y = c * r * w + b
    outs = (y, s) if kept else (y,)
    if "dy" not in st:
        return outs
    dy, n = st["dy"].double(), c * r
    g = dy * w
    d = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    if kept:
        d = d + st["ds"].double()
    return (*outs, d, *((d,) if kept else ()), (dy * n).sum(0), dy.sum(0))


def _exact_conv(st):
    step = st["x"].dim() == 2
    x, w, b, s = st["x"].double(), st["weight"].double(), st["bias"].double(), st["state"].double()
    x = x.unsqueeze(1) if step else x
    T, W = x.shape[1], w.shape[1]
    padded = torch.cat([s, x], 1)
    pre = b + sum(w[:, j] * padded[:, j:j + T] for j in range(W))
    gate = torch.sigmoid(pre)
    y, last = pre * gate, padded[:, T:]
    if step:
        return y[:, 0], last
    if "dy" not in st:
        return y, last
    d = st["dy"].double() * gate * (1.0 + pre * (1.0 - gate))
    dp = torch.zeros_like(padded)
    for j in range(W):
        dp[:, j:j + T] += w[:, j] * d
    dp[:, T:] += st["ds"].double()
    dw = torch.stack([(d * padded[:, j:j + T]).sum((0, 1)) for j in range(W)], -1)
    return y, last, dp[:, W - 1:], dw, d.sum((0, 1)), dp[:, :W - 1]


def _exact_scan(st):
    """Token by token; the gradients by the reversed recurrence."""
    one = {n: (st[n].double() if n in st else None) for n in (*LEAVES["scan"], "dy", "ds")}
    step = one["x"].dim() == 2
    if step:
        one.update({n: one[n].unsqueeze(1) for n in ("x", "dt", "bm", "cm", "z") if one[n] is not None})
    x, dt, a, bm, cm, skip, z, bias, s0, dy, ds = (one[n] for n in (*LEAVES["scan"], "dy", "ds"))
    B, T, D = x.shape
    G, N = bm.shape[2:]
    R, raw = D // G, dt + bias
    sp = F.softplus(raw, threshold=60.0)
    h, y, marks, seg = s0, torch.empty_like(x), [], 32

    def shared(t, i):           # [B, D, N] of what a group's channels share
        return t[:, i].repeat_interleave(R, dim=1) if G > 1 else t[:, i]

    def token(h, i):
        return torch.exp(sp[:, i, :, None] * a) * h + (sp[:, i] * x[:, i])[..., None] * shared(bm, i)

    for i in range(T):
        if i % seg == 0:
            marks.append(h)
        h = token(h, i)
        y[:, i] = (h * shared(cm, i)).sum(-1) + skip * x[:, i]
    last, gate = h, None
    out = y
    if z is not None:
        gate = torch.sigmoid(z)
        out = y * z * gate
    if step:
        return out[:, 0], last
    if dy is None:
        return out, last
    g = dy if z is None else dy * z * gate
    dx, dsp, da = skip * g, torch.zeros_like(x), torch.zeros_like(a)
    db, dc = torch.zeros_like(bm), torch.zeros_like(cm)
    dh = ds
    for first in reversed(range(0, T, seg)):
        h, kept = marks[first // seg], []
        for i in range(first, min(T, first + seg)):
            kept.append(h)
            h = token(h, i)
        after = h
        for i in reversed(range(first, min(T, first + seg))):
            before = kept[i - first]
            b, u = shared(bm, i), (sp[:, i] * x[:, i])[..., None]
            dh = dh + g[:, i, :, None] * shared(cm, i)
            dc[:, i] = (g[:, i, :, None] * after).reshape(B, G, R, N).sum(2)
            db[:, i] = (dh * u).reshape(B, G, R, N).sum(2)
            du = (dh * b).sum(-1)
            decay = torch.exp(sp[:, i, :, None] * a)
            w = dh * decay * before
            dx[:, i] += sp[:, i] * du
            dsp[:, i] = x[:, i] * du + (w * a).sum(-1)
            da += (w * sp[:, i, :, None]).sum(0)
            dh, after = dh * decay, before
    dr = dsp * torch.sigmoid(raw)
    dz = () if z is None else (dy * y * gate * (1.0 + z * (1.0 - gate)),)
    return (out, last, dx, dr, da, db, dc, (g * x).sum((0, 1)), *dz, dr.sum((0, 1)), dh)


def exact(case, seed):
    st = prepare(case, seed)
    st = {n: (v.detach() if isinstance(v, torch.Tensor) else v) for n, v in st.items()}
    with torch.no_grad():
        return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan}[case["kind"].split()[0]](st)


# ---- work ---------------------------------------------------------------------------------------------------------


def work(case):
    size = {"float32": 4, "bfloat16": 2, None: 0}
    what, way = case["kind"].split()
    e, D = size[case["dtype"]], case["D"]
    if what == "norm":
        r, w, n = size[case["residual"]], 2 * D * size[case["wtype"]], case["R"] * D
        once = n * (2 * e + 2 * r) + w              # x, residual; the norm, the sum
        if way == "forward":
            return {"bytes": once, "flops": 8 * n}
        return {"bytes": 2 * once, "flops": 20 * n}     # their gradients, with the weights' own
    B, T = case["B"], case.get("T", 1)
    if what == "conv":
        W = case["W"]
        once = 2 * B * T * D * e + 2 * B * (W - 1) * D * e + (W + 1) * D * size[case["wtype"]]
        flops = (2 * W + 5) * B * T * D
        return {"bytes": 2 * once, "flops": 3 * flops} if way == "train" else {"bytes": once, "flops": flops}
    N, G = case["N"], case["G"]
    wide, few = B * T * D * e, 2 * B * T * G * N * e
    once = (4 if case["gate"] else 3) * wide + few + 2 * 4 * B * D * N + 4 * D * (N + 2)
    if way != "train":
        return {"bytes": once, "flops": 7 * B * T * D * N}
    return {"bytes": 2 * once, "flops": 24 * B * T * D * N}
