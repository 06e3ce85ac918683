"""The gated-recurrence block's operators in 64 bits on the CPU, step by step and row by row
(test infrastructure): what ``delrec.gated`` and ``delrec.checkpoint8`` compute, by definition."""

import torch

BLOCK = GROUP = 64


def round8(x):
    """The values an 8-bit copy of x stands for, with the stored arithmetic's 32-bit roundings
    (x must hold fp32 values): (values in 64 bits, integers, scales)."""
    n = x.shape[-1]
    p = torch.nn.functional.pad(x.detach().to(torch.float32), (0, -n % GROUP)).unflatten(-1, (-1, GROUP))
    amax = p.abs().amax(-1, keepdim=True)
    scale = torch.maximum(amax * torch.tensor(1.0 / 127, dtype=torch.float32), torch.tensor(2.0 ** -126))
    scale = torch.where(torch.isfinite(p).all(-1, keepdim=True), scale, torch.nan)
    q = (p * (1.0 / scale)).round()
    value = (q.double() * scale.double()).flatten(-2)[..., :n]
    return value, q.flatten(-2)[..., :n], scale[..., 0]


def scan(z, f, bias=None, h0=None, starts=None, lengths=None, kept=None):
    """(h, last, states): the recurrence over (T, B, N) in 64 bits, differentiable. ``kept``:
    the states to go on from every 64 steps (a backward pass from 8-bit inputs)."""
    T, B, N = z.shape
    h = torch.zeros(B, N, dtype=torch.float64) if h0 is None else h0
    ys, states = [], []
    for t in range(T):
        if t % BLOCK == 0:
            if kept is not None:
                # the value of the kept state, the derivative of the recurrence
                h = h + (kept[t // BLOCK] - h).detach()
            states.append(h.detach())
        prev = h
        if starts is not None:
            prev = torch.where(starts[t][:, None], torch.zeros_like(h), h)
        k = torch.sigmoid(-(f[t] if bias is None else f[t] + bias))
        new = prev + k * (z[t] - prev)
        if lengths is not None:
            live = (t < lengths)[:, None]
            ys.append(torch.where(live, new, torch.zeros_like(new)))
            h = torch.where(live, new, h)
        else:
            ys.append(new)
            h = new
    return torch.stack(ys), h, torch.stack(states)


def scan_grads(z, f, bias, h0, starts, lengths, dh, dlast, checkpoint=False):
    """(h, last, dz, df, db, dh0) of 64-bit inputs."""
    bias = torch.zeros(z.shape[-1], dtype=torch.float64) if bias is None else bias
    h0 = torch.zeros(z.shape[1:], dtype=torch.float64) if h0 is None else h0
    leaves = [t.detach().clone().requires_grad_(True) for t in (z, f, bias, h0)]
    h, last, states = scan(*leaves, starts, lengths)
    if not checkpoint:
        return (h.detach(), last.detach(), *torch.autograd.grad((h, last), leaves, (dh, dlast)))
    with torch.no_grad():
        leaves[0].copy_(round8(z)[0])
        leaves[1].copy_(round8(f)[0])
    h2, last2, _ = scan(*leaves, starts, lengths, kept=states)
    return (h.detach(), last.detach(), *torch.autograd.grad((h2, last2), leaves, (dh, dlast)))


def _rms(v, eps):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def norm_gate(o, g, x, w, scale, w2, eps):
    """(x', u) in 64 bits, differentiable; o None: the norm of x alone; w2 None: no u."""
    if o is not None:
        x = x + scale * _rms(o, eps) * w * g * torch.sigmoid(g)
    return x, None if w2 is None else _rms(x, eps) * w2


def norm_gate_grads8(o, g, x, w, scale, w2, eps, dxo, du):
    """Gradients (do, dg, dx, dw, dscale, dw2) at the 8-bit copies of o, g and x, the norms
    those of the 64-bit inputs."""
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    r = 1 / torch.sqrt(mean(o * o) + eps)
    new = norm_gate(o, g, x, w, scale, None, eps)[0]
    r2 = 1 / torch.sqrt(mean(new * new) + eps)
    o, g, x = (round8(t)[0] for t in (o, g, x))
    sg = torch.sigmoid(g)
    e = o * r
    e2 = (x + scale * e * w * g * sg) * r2
    v2 = w2 * du
    dx = dxo + r2 * (v2 - e2 * mean(v2 * e2))
    v = w * scale * dx * g * sg
    rows = tuple(range(x.dim() - 1))
    return (r * (v - e * mean(v * e)), scale * dx * e * w * (sg + g * sg * (1 - sg)), dx,
            (scale * dx * g * sg * e).sum(rows), (dx * e * w * g * sg).sum(rows), (du * e2).sum(rows))
