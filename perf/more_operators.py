"""Workloads for the selective state-space block's operators: the short causal convolution and the
selective scan over (T, B, N) sequences, both for one time step, and the residual addition with its
norm, whose output also comes in 8 bits.

A case is a dict of plain values; ``kind`` names the operator:

  conv   ``causal_conv``: forward, and with ``mode`` 'train' its backward pass
  scan   ``selective_scan``: the same
  step   ``conv_step`` and ``selective_step``: one time step of streaming input (a Linear stands between
         the two, so the second has inputs of its own)
  add    ``add_norm``: forward, and with ``mode`` 'train' its backward pass; with ``pack`` the
         norm's output in 8 bits too, returned as the values they stand for

With ``joint`` the inputs are column slices of one projection's output, as the block makes them.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16}
GROUP = 64       # channels of a row that share an 8-bit scale
EPS = 1e-6


def _conv(name, T, B, N, W, dtype, **more):
    return dict(dict(name=name, kind='conv', mode='train', T=T, B=B, N=N, W=W, dtype=dtype, joint=dtype == 'bf16',
                     masks=False), **more)


def _scan(name, T, B, N, S, dtype, **more):
    return dict(dict(name=name, kind='scan', mode='train', T=T, B=B, N=N, S=S, dtype=dtype, joint=dtype == 'bf16',
                     masks=False), **more)


def _add(name, R, N, dtype, resid, **more):
    return dict(dict(name=name, kind='add', mode='train', R=R, N=N, dtype=dtype, resid=resid, pack=False), **more)


def listed():
    return [
        # streaming inference of a few sessions, one time step: latency
        dict(name='step_small', kind='step', B=4, N=256, S=16, W=4, dtype='bf16'),
        # the same for many sessions of a wide model
        dict(name='step_large', kind='step', B=512, N=2048, S=16, W=4, dtype='bf16'),
        # speech commands: 250 steps, batch 128, 512 channels, slices of the block's projection
        _conv('conv_ordinary', 250, 128, 512, 4, 'bf16'),
        # packed and padded streams of an odd width in 32 bits
        _conv('conv_ragged', 1000, 50, 333, 3, 'fp32', masks=True),
        # the memorisation task's layer (64 neurons, 32 steps, batch 64): launches and host path count
        _scan('scan_small', 32, 64, 64, 16, 'fp32'),
        # speech commands
        _scan('scan_ordinary', 250, 128, 512, 16, 'bf16'),
        # packed and padded streams of an odd width
        _scan('scan_ragged', 1000, 50, 333, 8, 'bf16', masks=True),
        # a long recording read in before streaming: one row of the widest layer
        _scan('scan_prompt', 8192, 1, 2048, 16, 'bf16', mode='infer'),
        # the most states a channel, few rows, in 32 bits
        _scan('scan_states', 512, 4, 1024, 64, 'fp32'),
        # the widest layer's training step
        _scan('scan_large', 1024, 8, 2048, 16, 'bf16'),
        # evaluating a small model of an odd width: forward only
        _add('add_eval', 5000, 700, 'fp32', 'fp32', mode='infer'),
        # the widest block's, residual stream in 32 bits, the next Linear's input kept in 8 bits
        _add('add_pack', 65536, 2048, 'bf16', 'fp32', pack=True),
    ]


def draw(rng):
    """A case of the listed ones' ranges: sizes spread over their logarithms, odd ones too."""
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return min(hi, v if rng.random() < 0.5 else max(lo, v // 20 * 20))

    kind = rng.choice(['scan', 'scan', 'scan', 'conv', 'conv', 'add', 'add', 'step'])
    dtype = rng.choice(['bf16', 'bf16', 'fp32'])
    W = rng.choice([2, 3, 4, 4, 4, 5, 8])
    S = rng.choice([16, 16, 16, size(1, 64)])
    if kind == 'step':
        return dict(kind=kind, B=size(1, 512), N=size(32, 2048), S=min(S, 16), W=W, dtype=dtype)
    mode = rng.choice(['train', 'train', 'infer'])
    if kind == 'add':
        return dict(kind=kind, mode=mode, R=size(200, 65536), N=size(32, 2048), dtype=dtype, resid=rng.choice(['fp32', dtype]),
                    pack=rng.random() < 0.5)
    N, joint, masks = size(32, 2048), rng.random() < 0.5, rng.random() < 0.4
    if kind == 'conv':
        T = size(16, 8192)
        B = size(1, max(2, min(512, (1 << 24) // (T * N))))
        return dict(kind=kind, mode=mode, T=T, B=B, N=N, W=W, dtype=dtype, joint=joint, masks=masks)
    T = size(16, 8192 if mode == 'infer' else 2048)
    B = size(1, max(1, min(256, (1 << 28) // (T * N * S))))
    return dict(kind=kind, mode=mode, T=T, B=B, N=N, S=S, dtype=dtype, joint=joint, masks=masks)


# ---------------------------------------------------------------- inputs --------------------

def _leaf(t):
    return t.detach().requires_grad_(True)


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case['dtype']]

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * std).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=gen, device=dev) * (hi - lo) + lo

    def state_space(N, S):
        # step sizes from 1e-3 to 1e-1 where dt is 0, decay rates 1 .. S with some spread
        step = torch.exp(uniform(N, lo=math.log(1e-3), hi=math.log(1e-1)))
        rates = torch.arange(1, S + 1, device=dev, dtype=torch.float32) * torch.exp(normal(N, S, std=0.1))
        return -rates, 1 + normal(N, std=0.1), torch.log(torch.expm1(step))

    s = {'case': case}
    kind = case['kind']
    if kind == 'add':
        R, N = case['R'], case['N']
        rt = DTYPES[case['resid']]
        s.update(x=_leaf(normal(R, N, dtype=rt)), y=_leaf(normal(R, N, dtype=dt, std=0.5)), weight=_leaf(1 + normal(N, std=0.1)))
        if case['mode'] == 'train':
            s.update(dx=normal(R, N, dtype=rt), du=normal(R, N, dtype=dt))
        return s
    if kind == 'step':
        B, N, S, W = case['B'], case['N'], case['S'], case['W']
        A, D, bias = state_space(N, S)
        proj, low = normal(B, 2 * N, dtype=dt), normal(B, 2 * S, dtype=dt)
        s.update(x=proj[:, :N], g=proj[:, N:], conv=normal(B, W - 1, N, dtype=dt), weight=normal(N, W, std=W ** -0.5),
                 bias=normal(N, std=0.1), xc=normal(B, N, dtype=dt), dt=normal(B, N, dtype=dt), A=A, D=D, dt_bias=bias, b=low[:, :S], c=low[:, S:],
                 h=normal(B, N, S, std=0.5))
        s.update(conv_out=torch.empty_like(s['conv']), h_out=torch.empty_like(s['h']))
        return s
    T, B, N = case['T'], case['B'], case['N']
    train = case['mode'] == 'train'
    s.update(starts=None, lengths=None)
    if case['masks']:
        s['starts'] = uniform(T, B) < 1.0 / 128
        lengths = (uniform(B) * (T + 1)).to(torch.int64).clamp_(max=T)
        lengths[0] = T
        if B > 1:
            lengths[-1] = 0
        s['lengths'] = lengths
    if case['joint']:
        proj = normal(T, B, 2 * N, dtype=dt)
        x, g = proj[..., :N], proj[..., N:]
    else:
        x, g = normal(T, B, N, dtype=dt), normal(T, B, N, dtype=dt)
    s['x'] = _leaf(x)
    if kind == 'conv':
        W = case['W']
        s.update(weight=_leaf(normal(N, W, std=W ** -0.5)), bias=_leaf(normal(N, std=0.1)),
                 state=_leaf(normal(B, W - 1, N, dtype=dt)))
        if train:
            s.update(dy=normal(T, B, N, dtype=dt), dstate=normal(B, W - 1, N, dtype=dt))
        return s
    S = case['S']
    A, D, bias = state_space(N, S)
    if case['joint']:
        low = normal(T, B, 2 * S, dtype=dt)
        b, c = low[..., :S], low[..., S:]
    else:
        b, c = normal(T, B, S, dtype=dt), normal(T, B, S, dtype=dt)
    s.update(g=_leaf(g), dt=_leaf(normal(T, B, N, dtype=dt)), A=_leaf(A), b=_leaf(b), c=_leaf(c), D=_leaf(D),
             dt_bias=_leaf(bias), h0=_leaf(normal(B, N, S, std=0.5)))
    if train:
        s.update(dy=normal(T, B, N, dtype=dt), dlast=normal(B, N, S))
    return s


# ---------------------------------------------------------------- the framework's calls -----

CONV_LEAVES = ('x', 'weight', 'bias', 'state')
SCAN_LEAVES = ('x', 'dt', 'A', 'b', 'c', 'D', 'g', 'dt_bias', 'h0')
ADD_LEAVES = ('x', 'y', 'weight')


def _ops():
    pkg = str(Path(__file__).resolve().parent.parent / 'snn-delays_amd')
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from delrec import checkpoint8, gated, selective
    return selective, gated, checkpoint8


def _run_own(s):
    case = s['case']
    selective, gated, checkpoint8 = _ops()
    kind = case['kind']
    if kind == 'step':
        with torch.no_grad():
            u, conv = selective.conv_step(s['x'], s['conv'], s['weight'], s['bias'], state_out=s['conv_out'])
            y, h = selective.selective_step(s['xc'], s['dt'], s['A'], s['b'], s['c'], s['h'], D=s['D'], g=s['g'],
                                            dt_bias=s['dt_bias'], h_out=s['h_out'])
        return {'u': u, 'conv': conv, 'y': y, 'h': h}
    if kind == 'conv':
        def call():
            return selective.causal_conv(s['x'], s['weight'], s['bias'], s['state'], starts=s['starts'], lengths=s['lengths'])
        names, outs, cots = CONV_LEAVES, ('y', 'state'), ('dy', 'dstate')
    elif kind == 'scan':
        def call():
            return selective.selective_scan(s['x'], s['dt'], s['A'], s['b'], s['c'], D=s['D'], g=s['g'], dt_bias=s['dt_bias'],
                                            h0=s['h0'], starts=s['starts'], lengths=s['lengths'])
        names, outs, cots = SCAN_LEAVES, ('y', 'last'), ('dy', 'dlast')
    else:
        def call():
            return gated.add_norm(s['x'], s['y'], s['weight'], eps=EPS, pack=case['pack'])
        names, outs, cots = ADD_LEAVES, ('x', 'u'), ('dx', 'du')
    if case['mode'] == 'infer':
        with torch.no_grad():
            res = call()
        out = dict(zip(outs, res))
    else:
        res = call()
        out = dict(zip(outs, res))
        grads = torch.autograd.grad(res[:2], [s[n] for n in names], [s[n] for n in cots])
        out.update(('d_' + n, t) for n, t in zip(names, grads))
    if case.get('pack'):
        out['u8'] = checkpoint8.unpack8(res[2])
    return out


# ---------------------------------------------------------------- plain forms ---------------

def _silu(x):
    return x * torch.sigmoid(x)


def _silu_slope(x):
    sig = torch.sigmoid(x)
    return sig * (1 + x * (1 - sig))


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _segments(starts, lengths, T, B, dev):
    """(T, B): the number of the sequence that a step belongs to, and whether it is padding."""
    seg = starts.to(torch.int64).cumsum(0)
    return seg, torch.arange(T, device=dev)[:, None] >= lengths


def _plain_conv(s):
    case = s['case']
    T, B, W = case['T'], case['B'], case['W']
    x, w, bias, state = s['x'].float(), s['weight'], s['bias'], s['state'].float()
    dt = DTYPES[case['dtype']]
    pad = seg = None
    if case['masks']:
        seg, pad = _segments(s['starts'], s['lengths'], T, B, x.device)
        x = torch.where(pad[..., None], 0.0, x)
        seg = torch.cat([torch.zeros(W - 1, B, dtype=seg.dtype, device=x.device), seg])
    ext = torch.cat([state.transpose(0, 1), x])            # step t is row t + W - 1
    taps = []
    for i in range(W):
        tap = ext[i:i + T]
        if seg is not None:
            tap = torch.where((seg[i:i + T] == seg[W - 1:])[..., None], tap, 0.0)
        taps.append(tap)
    pre = bias + sum(t * w[:, i] for i, t in enumerate(taps))
    y = _silu(pre)
    if pad is not None:
        y = torch.where(pad[..., None], 0.0, y)
    out = {'y': y.to(dt)}
    # the rows that the next call starts from
    if pad is None:
        out['state'] = ext[T:].transpose(0, 1).contiguous().to(dt)
    else:
        rows = s['lengths'][:, None] + torch.arange(W - 1, device=x.device)             # (B, W - 1)
        cols = torch.arange(B, device=x.device)[:, None].expand_as(rows)
        kept = seg[rows, cols] == seg[s['lengths'] + W - 2, cols[:, 0]][:, None]
        out['state'] = torch.where(kept[..., None], ext[rows, cols], 0.0).to(dt)
    if case['mode'] == 'infer':
        return out
    dpre = s['dy'].float() * _silu_slope(pre)
    if pad is not None:
        dpre = torch.where(pad[..., None], 0.0, dpre)
    dw = torch.stack([(dpre * t).sum((0, 1)) for t in taps], 1)
    dext = torch.zeros_like(ext)
    for i in range(W):
        part = dpre * w[:, i]
        if seg is not None:
            part = torch.where((seg[i:i + T] == seg[W - 1:])[..., None], part, 0.0)
        dext[i:i + T] += part
    if pad is None:
        dext[T:] += s['dstate'].float().transpose(0, 1)
    else:
        dext[rows, cols] += torch.where(kept[..., None], s['dstate'].float(), 0.0)
    dx = dext[W - 1:]
    if pad is not None:
        dx = torch.where(pad[..., None], 0.0, dx)
    out.update(d_x=dx.to(dt), d_weight=dw, d_bias=dpre.sum((0, 1)), d_state=dext[:W - 1].transpose(0, 1).contiguous().to(dt))
    return out


def _affine_scan(a, b):
    """All prefixes of h <- a h + b along the first axis, by doubling, in b's place."""
    a = a.clone()
    n, s = a.shape[0], 1
    while s < n:
        b[s:] += a[s:] * b[:n - s]
        if 2 * s < n:
            a[s:] = a[s:] * a[:n - s]
        s *= 2
    return b


def _plain_scan(s):
    case = s['case']
    T, B = case['T'], case['B']
    dt = DTYPES[case['dtype']]
    x, raw, g = s['x'].float(), s['dt'].float() + s['dt_bias'], s['g'].float()
    A, b, c, D = s['A'], s['b'].float(), s['c'].float(), s['D']
    delta = _softplus(raw)
    pad = starts = None
    if case['masks']:
        starts = s['starts'][..., None, None]
        _, pad = _segments(s['starts'], s['lengths'], T, B, x.device)
        delta = torch.where(pad[..., None], 0.0, delta)    # the state stays as it is
    a = torch.exp(delta[..., None] * A)
    if starts is not None:
        a = torch.where(starts & ~pad[..., None, None], 0.0, a)
    h = (delta * x)[..., None] * b[:, :, None, :]
    h[0] += a[0] * s['h0']
    h = _affine_scan(a, h)
    core = (h * c[:, :, None, :]).sum(-1) + D * x
    y = core * _silu(g)
    if pad is not None:
        y = torch.where(pad[..., None], 0.0, y)
    out = {'y': y.to(dt), 'last': h[-1].clone()}
    if case['mode'] == 'infer':
        return out
    dy = s['dy'].float()
    if pad is not None:
        dy = torch.where(pad[..., None], 0.0, dy)
    dg = dy * core * _silu_slope(g)
    dcore = dy * _silu(g)
    dc = (dcore[..., None] * h).sum(2)
    # lam_t = c_t dcore_t + a_{t+1} lam_{t+1}, latest step first
    lam = dcore[..., None] * c[:, :, None, :]
    lam[-1] += s['dlast']
    back = torch.cat([torch.zeros_like(a[:1]), a[1:].flip(0)])
    lam = _affine_scan(back, lam.flip(0)).flip(0)
    del back
    d0 = a[0] * lam[0]
    db = (lam * (delta * x)[..., None]).sum(2)
    lb = (lam * b[:, :, None, :]).sum(-1)
    lam *= a
    lam[0] *= s['h0']
    lam[1:] *= h[:-1]
    dA = (lam * delta[..., None]).sum((0, 1))
    ddelta = (lam * A).sum(-1) + x * lb
    draw = ddelta * torch.sigmoid(raw)
    dx = delta * lb + D * dcore
    if pad is not None:
        draw, dg = (torch.where(pad[..., None], 0.0, t) for t in (draw, dg))
    out.update(d_x=dx.to(dt), d_dt=draw.to(dt), d_A=dA, d_b=db.to(dt), d_c=dc.to(dt), d_D=(dcore * x).sum((0, 1)), d_g=dg.to(dt),
               d_dt_bias=draw.sum((0, 1)), d_h0=d0)
    return out


def _plain_step(s):
    dt = DTYPES[s['case']['dtype']]
    rows = torch.cat([s['conv'], s['x'][:, None]], 1)
    u = _silu((rows.float() * s['weight'].t()).sum(1) + s['bias']).to(dt)
    x = s['xc'].float()
    delta = _softplus(s['dt'].float() + s['dt_bias'])[..., None]
    h = torch.exp(delta * s['A']) * s['h'] + delta * x[..., None] * s['b'].float()[:, None, :]
    y = ((h * s['c'].float()[:, None, :]).sum(-1) + s['D'] * x) * _silu(s['g'].float())
    return {'u': u, 'conv': rows[:, 1:].contiguous(), 'y': y.to(dt), 'h': h}


def _round8(x):
    """The values that groups of 64 channels of a row stand for in 8 bits."""
    n = x.shape[-1]
    p = torch.nn.functional.pad(x, (0, -n % GROUP)).unflatten(-1, (-1, GROUP))
    scale = (p.abs().amax(-1, keepdim=True) * (1.0 / 127)).clamp(min=2.0 ** -126)
    return ((p * scale.reciprocal()).round() * scale).flatten(-2)[..., :n]


def _plain_add(s):
    case = s['case']
    dt, rt = DTYPES[case['dtype']], DTYPES[case['resid']]
    new = s['x'].float() + s['y'].float()
    r = (new.square().mean(-1, keepdim=True) + EPS).rsqrt()
    unit = new * r
    out = {'x': new.to(rt), 'u': (unit * s['weight']).to(dt)}
    if case['mode'] == 'train':
        du = s['du'].float()
        v = s['weight'] * du
        dx = s['dx'].float() + r * (v - unit * (v * unit).mean(-1, keepdim=True))
        out.update(d_x=dx.to(rt), d_y=dx.to(dt), d_weight=(du * unit).sum(0))
    if case['pack']:
        out['u8'] = _round8(out['u'].float()).to(dt)
    return out


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {'conv': _plain_conv, 'scan': _plain_scan, 'step': _plain_step, 'add': _plain_add}[state['case']['kind']](state)


# ---------------------------------------------------------------- work ----------------------

def work(case):
    size = {'fp32': 4, 'bf16': 2}
    e = size[case['dtype']]
    train = case.get('mode') == 'train'
    if case['kind'] == 'add':
        n, r = case['R'] * case['N'], size[case['resid']]
        # x, y, x', u and, in training, dx', du, dx, dy; a byte a value more and the groups' scales
        bytes_ = n * (4 * (e + r) if train else 2 * (e + r)) + case['N'] * (8 if train else 4)
        if case['pack']:
            bytes_ += n + case['R'] * -(-case['N'] // GROUP) * 4
        return {'bytes': bytes_, 'flops': n * (16 if train else 6)}
    if case['kind'] == 'step':
        n, S, W = case['B'] * case['N'], case['S'], case['W']
        return {'bytes': n * (8 * S + e * (2 * W + 4)) + case['B'] * 2 * S * e + case['N'] * 4 * (S + W + 3),
                'flops': n * (7 * S + 2 * W + 25)}
    n = case['T'] * case['B'] * case['N']
    if case['kind'] == 'conv':
        W = case['W']
        # x, y and, in training, dy and dx (x is read again); the states at both ends
        rows = case['B'] * case['N'] * (W - 1) * e * (4 if train else 2)
        return {'bytes': n * e * (4 if train else 2) + rows, 'flops': n * (6 * W + 20 if train else 2 * W + 6)}
    S = case['S']
    low = case['T'] * case['B'] * S * e
    rows = case['B'] * case['N'] * S * 4
    # x, dt, g, y and, in training, dy, dx, ddt, dg; B, C and their gradients; the states at both ends
    return {'bytes': n * e * (8 if train else 4) + low * (4 if train else 2) + rows * (4 if train else 2),
            'flops': n * ((25 if train else 7) * S + (60 if train else 20))}


# ---------------------------------------------------------------- 64 bits -------------------

def _exact_conv(x, weight, bias, state, starts, lengths):
    """Step by step: a window of the last rows, emptied by a start."""
    W = weight.shape[1]
    window = [state[:, k] for k in range(W - 1)]
    ys = []
    for t in range(x.shape[0]):
        if starts is not None:
            window = [torch.where(starts[t][:, None], torch.zeros_like(v), v) for v in window] if lengths is None else [
                torch.where((starts[t] & (t < lengths))[:, None], torch.zeros_like(v), v) for v in window]
        now = window + [x[t]]
        pre = bias
        for i, v in enumerate(now):
            pre = pre + v * weight[:, i]
        y = pre / (1 + torch.exp(-pre))
        if lengths is None:
            window = now[1:]
        else:
            live = (t < lengths)[:, None]
            y = torch.where(live, y, torch.zeros_like(y))
            window = [torch.where(live, new, old) for new, old in zip(now[1:], window)]
        ys.append(y)
    return torch.stack(ys), torch.stack(window, 1)


def _exact_scan(x, dt, A, b, c, D, g, dt_bias, h0, starts, lengths):
    """Step by step."""
    h, ys = h0, []
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    for t in range(x.shape[0]):
        delta = torch.nn.functional.softplus(dt[t] + dt_bias, threshold=700.0)
        before = h
        if starts is not None:
            before = torch.where(starts[t][:, None, None], zero, h)
        new = torch.exp(delta.unsqueeze(-1) * A) * before + (delta * x[t]).unsqueeze(-1) * b[t].unsqueeze(1)
        y = (torch.matmul(new, c[t].unsqueeze(-1)).squeeze(-1) + D * x[t]) * g[t] / (1 + torch.exp(-g[t]))
        if lengths is not None:
            live = (t < lengths)[:, None]
            y = torch.where(live, y, zero)
            new = torch.where(live.unsqueeze(-1), new, h)
        h = new
        ys.append(y)
    return torch.stack(ys), h


def _exact_add(x, y, weight):
    new = x + y
    return new, new / torch.sqrt((new * new).sum(-1, keepdim=True) / new.shape[-1] + EPS) * weight


def _kept8(x):
    """8-bit values by their definition, one group of columns at a time."""
    parts = []
    for col in range(0, x.shape[-1], GROUP):
        part = x[..., col:col + GROUP]
        step = torch.maximum(part.abs().max(-1, keepdim=True).values / 127, torch.full((), 2.0 ** -126, dtype=x.dtype, device=x.device))
        parts.append(torch.round(part / step) * step)
    return torch.cat(parts, -1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind == 'step':
        with torch.no_grad():
            d = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
            u, conv = _exact_conv(d['x'][None], d['weight'], d['bias'], d['conv'], None, None)
            y, h = _exact_scan(d['xc'][None], d['dt'][None], d['A'], d['b'][None], d['c'][None], d['D'], d['g'][None], d['dt_bias'], d['h'],
                               None, None)
        return {'u': u[0], 'conv': conv, 'y': y[0], 'h': h}
    if kind == 'conv':
        names, outs, cots = CONV_LEAVES, ('y', 'state'), ('dy', 'dstate')
        call = lambda *a: _exact_conv(*a, s['starts'], s['lengths'])  # noqa: E731
    elif kind == 'scan':
        names, outs, cots = SCAN_LEAVES, ('y', 'last'), ('dy', 'dlast')
        call = lambda *a: _exact_scan(*a, s['starts'], s['lengths'])  # noqa: E731
    else:
        names, outs, cots = ADD_LEAVES, ('x', 'u'), ('dx', 'du')
        call = _exact_add
    train = case['mode'] == 'train'
    with torch.set_grad_enabled(train):
        leaves = [s[n].detach().double().requires_grad_(train) for n in names]
        res = call(*leaves)
        out = {n: t.detach() for n, t in zip(outs, res)}
        if train:
            grads = torch.autograd.grad(res, leaves, [s[n].double() for n in cots])
            out.update(('d_' + n, t) for n, t in zip(names, grads))
    if case.get('pack'):
        out['u8'] = _kept8(out['u'].to(DTYPES[case['dtype']]).double())
    return out
