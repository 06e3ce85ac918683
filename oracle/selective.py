"""The selective state-space block's operators in 64 bits on the CPU, step by step (test
infrastructure): what ``delrec.selective`` and ``delrec.gated.add_norm`` compute, by definition."""

import torch


def _fresh(starts, lengths, t):
    """(B,) rows whose sequence starts at step t, and rows that have a step t."""
    live = None if lengths is None else t < lengths
    start = None if starts is None else (starts[t] if live is None else starts[t] & live)
    return start, live


def conv(x, weight, bias=None, state=None, starts=None, lengths=None, silu=True):
    """(y, state after) over (T, B, N), differentiable."""
    T, B, N = x.shape
    W = weight.shape[1]
    zero = torch.zeros(B, N, dtype=torch.float64)
    window = [zero] * (W - 1) if state is None else [state[:, k] for k in range(W - 1)]
    ys = []
    for t in range(T):
        start, live = _fresh(starts, lengths, t)
        if start is not None:
            window = [torch.where(start[:, None], zero, v) for v in window]
        now = window + [x[t] if live is None else torch.where(live[:, None], x[t], zero)]
        y = sum(v * weight[:, i] for i, v in enumerate(now))
        if bias is not None:
            y = y + bias
        if silu:
            y = y * torch.sigmoid(y)
        if live is None:
            window = now[1:]
        else:
            y = torch.where(live[:, None], y, zero)
            window = [torch.where(live[:, None], a, b) for a, b in zip(now[1:], window)]
        ys.append(y)
    return torch.stack(ys), torch.stack(window, 1)


def softplus(x):
    return torch.nn.functional.softplus(x, threshold=700.0)


def scan(x, dt, A, B, C, D=None, g=None, dt_bias=None, h0=None, starts=None, lengths=None):
    """(y, last) over (T, B, N), differentiable."""
    T, R, N = x.shape
    zero = torch.zeros(R, N, A.shape[1], dtype=torch.float64)
    h, ys = zero if h0 is None else h0, []
    for t in range(T):
        start, live = _fresh(starts, lengths, t)
        d = softplus(dt[t] if dt_bias is None else dt[t] + dt_bias)
        before = h if start is None else torch.where(start[:, None, None], zero, h)
        new = torch.exp(d[..., None] * A) * before + (d * x[t])[..., None] * B[t][:, None]
        y = (new * C[t][:, None]).sum(-1)
        if D is not None:
            y = y + D * x[t]
        if g is not None:
            y = y * g[t] * torch.sigmoid(g[t])
        if live is not None:
            y = torch.where(live[:, None], y, zero[..., 0])
            new = torch.where(live[:, None, None], new, h)
        h = new
        ys.append(y)
    return torch.stack(ys), h


def scan_grads(x, dt, A, B, C, D, g, dt_bias, h0, starts, lengths, dy, dlast):
    """The gradients by their formulas, the carry walked back from the last step: a dict, and for
    those that are sums the largest sum of magnitudes."""
    T, R, N = x.shape
    zero = torch.zeros(R, N, A.shape[1], dtype=torch.float64)
    D = torch.zeros(N, dtype=torch.float64) if D is None else D
    raw = dt if dt_bias is None else dt + dt_bias
    delta, slope = softplus(raw), torch.sigmoid(raw)
    befores, h = [], zero if h0 is None else h0
    for t in range(T):
        start, live = _fresh(starts, lengths, t)
        before = h if start is None else torch.where(start[:, None, None], zero, h)
        new = torch.exp(delta[t][..., None] * A) * before + (delta[t] * x[t])[..., None] * B[t][:, None]
        befores.append(before)
        h = new if live is None else torch.where(live[:, None, None], new, h)
    out = {k: torch.zeros_like(v) for k, v in dict(x=x, dt=dt, A=A, B=B, C=C, D=D, g=x, dt_bias=D).items()}
    mass = {k: torch.zeros_like(out[k]) for k in ('A', 'B', 'C', 'D', 'dt_bias')}
    carry = dlast
    for t in reversed(range(T)):
        start, live = _fresh(starts, lengths, t)
        on = torch.ones(R, dtype=torch.bool) if live is None else live
        a, u = torch.exp(delta[t][..., None] * A), delta[t] * x[t]
        h = a * befores[t] + u[..., None] * B[t][:, None]
        core = (h * C[t][:, None]).sum(-1) + D * x[t]
        w = dy[t]
        if g is not None:
            sg = torch.sigmoid(g[t])
            out['g'][t] = torch.where(on[:, None], dy[t] * core * sg * (1 + g[t] * (1 - sg)), 0.0)
            w = dy[t] * g[t] * sg
        lam = w[..., None] * C[t][:, None] + carry
        k = a * lam
        q = k * befores[t]
        lb = (lam * B[t][:, None]).sum(-1)
        draw = ((A * q).sum(-1) + x[t] * lb) * slope[t]
        live3, live2 = on[:, None, None], on[:, None]
        out['x'][t] = torch.where(live2, delta[t] * lb + D * w, 0.0)
        out['dt'][t] = torch.where(live2, draw, 0.0)
        for name, terms, dims in (('A', delta[t][..., None] * q, 0), ('D', w * x[t], 0), ('dt_bias', draw, 0)):
            terms = torch.where(live3 if terms.dim() == 3 else live2, terms, 0.0)
            out[name] += terms.sum(dims)
            mass[name] += terms.abs().sum(dims)
        for name, terms in (('B', lam * u[..., None]), ('C', w[..., None] * h)):
            terms = torch.where(live3, terms, 0.0)
            out[name][t] = terms.sum(1)
            mass[name][t] = terms.abs().sum(1)
        if start is not None:
            k = torch.where(start[:, None, None], zero, k)
        carry = torch.where(live3, k, carry)
    out['h0'] = carry
    if g is None:
        del out['g']
    return out, {k: float(v.max()) if v.numel() else 0.0 for k, v in mass.items()}


def add_norm(x, y, w, eps):
    new = x + y
    return new, new / torch.sqrt((new * new).mean(-1, keepdim=True) + eps) * w
