"""Plain 64-bit gated delta rule, token by token, for the tests (torch, any device; differentiable by autograd)."""
import torch


def rule(q, k, v, g, beta, state=None, scale=None):
    """``(out [B, T, Hv, dv], last state)`` in float64 from inputs of any type."""
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2:]
    scale = dk ** -0.5 if scale is None else scale
    q, k = (x.double().repeat_interleave(Hv // Hk, dim=2) for x in (q, k))
    v, g, beta = v.double(), g.double(), beta.double()
    s = torch.zeros(B, Hv, dk, dv, dtype=torch.float64, device=q.device) if state is None else state.double()
    outs = []
    for t in range(T):
        s = s * g[:, t].exp()[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (s * k[:, t, :, :, None]).sum(-2))
        s = s + k[:, t, :, :, None] * u[..., None, :]
        outs.append((s * q[:, t, :, :, None]).sum(-2) * scale)
    out = torch.stack(outs, 1) if outs else v.new_zeros(B, T, Hv, dv)
    return out, s


def inputs(B, T, Hk, Hv, dk, dv, dtype=torch.float32, seed=0, device="cuda", unit_keys=True):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=device, generator=gen)

    q, k = normal(B, T, Hk, dk), normal(B, T, Hk, dk)
    if unit_keys:
        q, k = (torch.nn.functional.normalize(x, dim=-1) for x in (q, k))
    rate = torch.exp(torch.rand(Hv, device=device, generator=gen) * 5 - 5)
    g = -rate * torch.nn.functional.softplus(normal(B, T, Hv))
    return (q.to(dtype), k.to(dtype), normal(B, T, Hv, dv).to(dtype), g, torch.sigmoid(normal(B, T, Hv)),
            0.5 * normal(B, Hv, dk, dv))
