"""The causal convolution, the selective scan and its step, and the residual addition with its norm
against their definitions in 64 bits.

Tolerances. In fp32 a step of the recurrence multiplies the state by a decay that is off by at most
3e-7 of itself (the exponent's two roundings, 2^y to 1 ulp, softplus) and adds a product of three
roundings: over the 300 steps here at most 300 * 3e-7 = 9e-5 of the largest value, random signs far
less. Rows of a convolution or a norm lose a few roundings and the gate's error: 1e-5 of the largest
value. bf16 outputs add half a unit in the 8th bit, 2^-8 of their own size at most. Sums over rows or
channels carry the same relative errors on the sum of magnitudes."""

import pytest
import torch

from oracle import gated as og
from oracle import selective as osel

BF16, FP32 = torch.bfloat16, torch.float32
SCAN_TOL, ROW_TOL = 1e-4, 1e-5
LEAVES = ('x', 'dt', 'A', 'B', 'C', 'D', 'g', 'dt_bias', 'h0')


@pytest.fixture
def dev():
    return torch.device('cuda')


def close(got, ref, tol, what, mass=None):
    """|got - ref| <= tol * largest magnitude (or ``mass``), plus a bf16 output's rounding."""
    got64 = got.detach().double().cpu()
    assert got64.shape == ref.shape, what
    big = (float(ref.abs().max()) if ref.numel() else 0.0) if mass is None else mass
    bound = tol * big + (2.0 ** -8 * ref.abs() if got.dtype == BF16 else 0.0) + 1e-30
    bad = ~((got64 - ref).abs() <= bound)
    assert int(bad.sum()) == 0, f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got64 - ref).abs().max()):.3e}, largest {big:.3e}'


def rnd(gen, *shape, dtype=FP32, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def masks_of(gen, T, B, masks):
    if not masks:
        return dict(starts=None, lengths=None)
    lengths = torch.randint(0, T + 1, (B,), generator=gen)
    lengths[0] = 0
    if B > 1:
        lengths[1] = T
    return dict(starts=torch.rand(T, B, generator=gen) < 0.1, lengths=lengths)


def put(c, dev):
    return {k: None if v is None else v.to(dev) for k, v in c.items()}


# ---------------------------------------------------------------- the recurrence ------------

def scan_case(T, B, N, S, dtype, masks, seed=0, rate=3.0):
    g = torch.Generator().manual_seed(seed)
    c = dict(x=rnd(g, T, B, N, dtype=dtype), dt=rnd(g, T, B, N, dtype=dtype), A=-torch.rand(N, S, generator=g) * rate,
             B=rnd(g, T, B, S, dtype=dtype), C=rnd(g, T, B, S, dtype=dtype), D=rnd(g, N), g=rnd(g, T, B, N, dtype=dtype),
             dt_bias=rnd(g, N) - 2, h0=rnd(g, B, N, S), dy=rnd(g, T, B, N, dtype=dtype), dlast=rnd(g, B, N, S))
    c.update(masks_of(g, T, B, masks))
    return c


def run_scan(c, dev):
    from delrec.selective import selective_scan
    d = put(c, dev)
    leaves = {k: d[k].requires_grad_(True) for k in LEAVES if d[k] is not None}
    y, last = selective_scan(*[leaves.get(k) for k in LEAVES], starts=d['starts'], lengths=d['lengths'])
    grads = torch.autograd.grad((y, last), list(leaves.values()), (d['dy'], d['dlast']))
    return dict(y=y.detach(), last=last.detach(), **dict(zip(leaves, grads)))


def check_scan(c, dev):
    got = run_scan(c, dev)
    d = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}
    y, last = osel.scan(*[d[k] for k in LEAVES], d['starts'], d['lengths'])
    ref, mass = osel.scan_grads(*[d[k] for k in LEAVES], d['starts'], d['lengths'], d['dy'], d['dlast'])
    close(got['y'], y, SCAN_TOL, 'y')
    close(got['last'], last, SCAN_TOL, 'last')
    for k in LEAVES:
        if c[k] is not None:
            close(got[k], ref[k], SCAN_TOL, 'd' + k, mass.get(k))
    return got


SCAN_SIZES = [(1, 1, 1, 1), (1, 3, 65, 16), (2, 2, 3, 5), (15, 2, 5, 3), (16, 1, 64, 16), (17, 3, 70, 8), (33, 2, 130, 17),
              (50, 2, 20, 33), (40, 1, 17, 64), (300, 2, 96, 16), (130, 5, 33, 4), (31, 33, 16, 2), (40, 530, 8, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize('masks', [False, True])
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('T,B,N,S', SCAN_SIZES)
def test_scan_forward_and_gradients(dev, T, B, N, S, dtype, masks):
    check_scan(scan_case(T, B, N, S, dtype, masks), dev)


@pytest.mark.gpu
@pytest.mark.parametrize('gone', [('g',), ('D', 'dt_bias'), ('h0',), ('g', 'D', 'dt_bias', 'h0')])
def test_scan_without_optional_inputs(dev, gone):
    c = scan_case(40, 3, 40, 16, FP32, True)
    c.update((k, None) for k in gone)
    check_scan(c, dev)


@pytest.mark.gpu
@pytest.mark.parametrize('S', [4, 16, 64])
def test_scan_gradients_are_differences(dev, S):
    """The loss' change along a direction, from its values in 64 bits, is the gradients' product."""
    c = scan_case(37, 2, 20, S, FP32, True)
    got = run_scan(c, dev)
    d = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}
    gen = torch.Generator().manual_seed(7)

    def loss(v):
        y, last = osel.scan(*[v[k] for k in LEAVES], v['starts'], v['lengths'])
        return float((y * d['dy']).sum() + (last * d['dlast']).sum())
    for k in LEAVES:
        way = torch.randn(d[k].shape, generator=gen, dtype=torch.float64)
        up, down, e = dict(d), dict(d), 1e-5
        up[k], down[k] = d[k] + e * way, d[k] - e * way
        terms = got[k].double().cpu() * way
        assert abs((loss(up) - loss(down)) / (2 * e) - float(terms.sum())) <= SCAN_TOL * float(terms.abs().sum()), k


@pytest.mark.gpu
@pytest.mark.parametrize('S', [3, 16, 40])
def test_scan_masked_places_may_hold_anything(dev, S):
    """Padding holds NaN and infinities, and a state before a start is infinite: neither reaches an
    output or a gradient."""
    T, B, N = 40, 4, 24
    c = scan_case(T, B, N, S, FP32, True)
    want = run_scan(c, dev)
    pad = (torch.arange(T)[:, None] >= c['lengths'])[..., None]
    for k, bad in (('x', float('nan')), ('dt', float('inf')), ('g', float('nan')), ('B', float('inf')), ('C', float('nan')),
                   ('dy', float('nan'))):
        c[k] = torch.where(pad, bad, c[k])
    got = run_scan(c, dev)
    for k in want:
        assert torch.equal(got[k], want[k]), k
    c['starts'][0] = True
    c['lengths'][0] = T
    pad = (torch.arange(T)[:, None] >= c['lengths'])[..., None]
    for k in ('x', 'dt', 'g', 'B', 'C', 'dy'):
        c[k] = torch.nan_to_num(c[k], 0.0, 0.0, 0.0)
    c['dlast'][c['lengths'] == 0] = 0.0
    c['h0'].fill_(float('inf'))
    got = run_scan(c, dev)
    for k in got:
        if k != 'last':
            assert torch.isfinite(got[k]).all(), k
    assert torch.isinf(got['last'][c['lengths'].to(dev) == 0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [FP32, BF16])
def test_scan_strides(dev, dtype):
    """Column slices of projections, batch-first tensors, one value for all steps, a last axis that is
    not contiguous, B and C of one row broadcast over rows."""
    from delrec.selective import selective_scan
    T, B, N, S = 35, 3, 68, 16
    c = scan_case(T, B, N, S, dtype, False)
    want = run_scan(c, dev)
    d = put(c, dev)
    proj = torch.cat([d['x'], d['g']], -1).requires_grad_(True)
    low = torch.cat([d['dt'], d['B'], d['C']], -1).requires_grad_(True)
    x, g = proj.chunk(2, -1)
    dt, Bm, C = low.split([N, S, S], -1)
    y, last = selective_scan(x, dt, d['A'], Bm, C, d['D'], g, d['dt_bias'], d['h0'])
    first = d['dy'].transpose(0, 1).contiguous().transpose(0, 1)
    dp, dl = torch.autograd.grad((y, last), (proj, low), (first, d['dlast']))
    assert torch.equal(y, want['y']) and torch.equal(last, want['last'])
    assert torch.equal(dp, torch.cat([want['x'], want['g']], -1)) and torch.equal(dl, torch.cat([want['dt'], want['B'], want['C']], -1))
    bf = {k: d[k].transpose(0, 1).contiguous().transpose(0, 1) for k in ('x', 'dt', 'g', 'B', 'C')}
    y, last = selective_scan(bf['x'], bf['dt'], d['A'].t().contiguous().t(), bf['B'], bf['C'], d['D'], bf['g'], d['dt_bias'], d['h0'])
    assert torch.equal(y, want['y']) and torch.equal(last, want['last'])
    wide = torch.stack([d['x'], d['x']], -1)[..., 0]
    y, _ = selective_scan(wide, d['dt'], d['A'], d['B'], d['C'], d['D'], d['g'], d['dt_bias'], d['h0'])
    assert torch.equal(y, want['y'])
    one = d['B'][:, :1].clone().requires_grad_(True)
    y, _ = selective_scan(d['x'], d['dt'], d['A'], one.expand(T, B, S), d['C'], d['D'], d['g'], d['dt_bias'], d['h0'])
    full = d['B'][:, :1].repeat(1, B, 1).requires_grad_(True)
    y2, _ = selective_scan(d['x'], d['dt'], d['A'], full, d['C'], d['D'], d['g'], d['dt_bias'], d['h0'])
    assert torch.equal(y, y2)
    (a,), (b,) = torch.autograd.grad(y, one, d['dy']), torch.autograd.grad(y2, full, d['dy'])
    torch.testing.assert_close(a, b.sum(1, keepdim=True))


@pytest.mark.gpu
def test_scan_in_parts_and_steps(dev):
    """A sequence in two calls, and step by step, is the sequence in one call."""
    from delrec.selective import selective_scan, selective_step
    for S in (1, 7, 16, 24, 64):
        c = put(scan_case(37, 3, 50, S, FP32, False), dev)
        args = lambda a, b: [c[k][a:b] if k in ('x', 'dt', 'B', 'C', 'g') else c[k] for k in LEAVES[:-1]]  # noqa: E731
        y, last = selective_scan(*args(0, 37), c['h0'])
        y1, h = selective_scan(*args(0, 20), c['h0'])
        y2, h = selective_scan(*args(20, 37), h)
        close(torch.cat([y1, y2]), y.double().cpu(), SCAN_TOL, 'parts')
        close(h, last.double().cpu(), SCAN_TOL, 'state')
        h = c['h0'].clone()
        for t in range(37):
            yt, h2 = selective_step(c['x'][t], c['dt'][t], c['A'], c['B'][t], c['C'][t], h, c['D'], c['g'][t], c['dt_bias'], h_out=h)
            assert h2.data_ptr() == h.data_ptr()
            close(yt, y[t].double().cpu(), SCAN_TOL, f'step {t}')
        close(h, last.double().cpu(), SCAN_TOL, 'stepped state')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('B,N,S', [(1, 1, 1), (5, 70, 16), (3, 130, 5), (2, 33, 64), (300, 16, 24)])
def test_step(dev, B, N, S, dtype):
    from delrec.selective import selective_step
    c = scan_case(1, B, N, S, dtype, False)
    d = put(c, dev)
    y, h = selective_step(d['x'][0], d['dt'][0], d['A'], d['B'][0], d['C'][0], d['h0'], d['D'], d['g'][0], d['dt_bias'])
    r = {k: v.double() if v is not None else None for k, v in c.items()}
    ry, rh = osel.scan(*[r[k] for k in LEAVES])
    close(y, ry[0], ROW_TOL, 'y')
    close(h, rh, ROW_TOL, 'h')
    bare, _ = selective_step(d['x'][0], d['dt'][0], d['A'], d['B'][0], d['C'][0], d['h0'])
    rb, _ = osel.scan(r['x'], r['dt'], r['A'], r['B'], r['C'], h0=r['h0'])
    close(bare, rb[0], ROW_TOL, 'bare')


@pytest.mark.gpu
def test_scan_extreme_step_sizes(dev):
    """Step sizes of e^-20 keep their digits, large ones forget the state, growing states follow the
    formula."""
    T, B, N, S = 20, 2, 32, 16
    c = scan_case(T, B, N, S, FP32, False)
    c['dt'] = torch.linspace(-20, 20, N).expand(T, B, N).contiguous()
    c['dt_bias'].zero_()
    check_scan(c, dev)
    from delrec.selective import selective_scan
    d = put(c, dev)
    d['dt'].fill_(-15.0)
    d['h0'].zero_()
    y, last = selective_scan(*[d[k] for k in LEAVES])
    r = {k: v.cpu().double() if v is not None else None for k, v in d.items()}
    _, rl = osel.scan(*[r[k] for k in LEAVES])
    # against each state's own sum of magnitudes, not the largest value
    mags = (osel.softplus(r['dt'] + r['dt_bias']) * r['x'].abs())[..., None] * r['B'].abs()[:, :, None]
    assert ((last.double().cpu() - rl).abs() <= 1e-5 * mags.sum(0)).all()
    c = scan_case(T, B, N, S, FP32, False)
    c['A'] = c['A'].abs() * 0.2
    check_scan(c, dev)


@pytest.mark.gpu
def test_scan_offsets_past_32_bits(dev):
    """Rows of a tensor of more than 2^32 elements, forward and backward."""
    from delrec.selective import selective_scan
    T, B, N, S = 17, 2, 64, 4
    c = scan_case(T, B, N, S, BF16, False)
    want = run_scan(c, dev)
    big = torch.empty(T * 260_000_000 + 4096, dtype=BF16, device=dev)
    d = put(c, dev)
    far = big.as_strided((T, B, N), (260_000_000, N, 1)).copy_(d['x'])
    leaves = {k: d[k].requires_grad_(True) for k in LEAVES}
    leaves['x'] = far.requires_grad_(True)
    y, last = selective_scan(*[leaves[k] for k in LEAVES])
    (dx,) = torch.autograd.grad((y, last), (leaves['x'],), (d['dy'], d['dlast']))
    assert torch.equal(y, want['y']) and torch.equal(last, want['last']) and torch.equal(dx, want['x'])


@pytest.mark.gpu
@pytest.mark.parametrize('S', [2, 40])
def test_scan_ranges_of_time(dev, S):
    """Long sequences of few channels are cut into ranges of time: starts and row ends anywhere, in the
    first and last steps of a range too, rows that end before a range begins."""
    T, B, N = 513, 6, 20
    c = scan_case(T, B, N, S, FP32, True, rate=0.3)
    c['lengths'] = torch.tensor([T, 0, 1, 255, 256, 257])
    c['starts'] = torch.zeros(T, B, dtype=torch.bool)
    for t in (31, 32, 33, 255, 256, 512):
        c['starts'][t] = True
    c['starts'][:, 0] = False
    check_scan(c, dev)
    c['starts'] = c['lengths'] = None
    check_scan(c, dev)


@pytest.mark.gpu
def test_more_rows_than_one_launch_holds(dev):
    """Past 2^20 workgroups the launches are repeated: the last rows are computed as the first."""
    from delrec.selective import causal_conv, conv_step, selective_scan, selective_step
    B, N, S = (1 << 20) + 70, 1, 2
    c = put(scan_case(1, 3, N, S, FP32, False), dev)
    wide = {k: c[k].repeat(*([1] * (c[k].dim() - 2)), (B + 2) // 3, 1)[:, :B] if k in ('x', 'dt', 'B', 'C', 'g', 'dy') else c[k] for k in c}
    for k in ('h0', 'dlast'):
        wide[k] = c[k].repeat((B + 2) // 3, 1, 1)[:B]
    want = run_scan({k: v if v is None else v.cpu() for k, v in c.items()}, dev)
    leaves = {k: wide[k].contiguous().requires_grad_(True) for k in LEAVES}
    y, last = selective_scan(*[leaves[k] for k in LEAVES])
    dx, dB, dh = torch.autograd.grad((y, last), (leaves['x'], leaves['B'], leaves['h0']), (wide['dy'], wide['dlast']))
    for got, k in ((y, 'y'), (dx, 'x'), (dB, 'B')):
        assert torch.equal(got[:, :3], want[k]) and torch.equal(got[:, B - 1], want[k][:, (B - 1) % 3])
    assert torch.equal(last[B - 1], want['last'][(B - 1) % 3]) and torch.equal(dh[B - 1], want['h0'][(B - 1) % 3])
    with torch.no_grad():
        ys, hs = selective_step(*[wide[k][0] if k in ('x', 'dt', 'B', 'C') else wide[k] for k in ('x', 'dt', 'A', 'B', 'C')], wide['h0'],
                                wide['D'], wide['g'][0], wide['dt_bias'])
        close(ys, y[0].double().cpu(), ROW_TOL, 'step')
        close(hs, last.double().cpu(), ROW_TOL, 'state')
    e = put(conv_case(1, 3, 125, 4, BF16, False), dev)
    B = (1 << 23) + 9                    # eight rows a workgroup
    x, state = (e[k].repeat(1, (B + 2) // 3, 1)[:, :B] if k == 'x' else e[k].repeat((B + 2) // 3, 1, 1)[:B] for k in ('x', 'state'))
    with torch.no_grad():
        y0, s0 = causal_conv(e['x'], e['weight'], e['bias'], e['state'])
        y, s = causal_conv(x, e['weight'], e['bias'], state)
        assert torch.equal(y[0, B - 3:], y0[0, [(B - 3 + i) % 3 for i in range(3)]]) and torch.equal(s[B - 1], s0[(B - 1) % 3])
        y, s = conv_step(x[0], state, e['weight'], e['bias'])
        assert torch.equal(y[B - 1], y0[0, (B - 1) % 3]) and torch.equal(s[B - 1], s0[(B - 1) % 3])


@pytest.mark.gpu
def test_parameters_of_other_types_and_saved_tensor_hooks(dev):
    """Parameters in bf16 count as their fp32 values and get their gradients in bf16; what the graph
    keeps may go through the host."""
    from delrec.gated import add_norm
    from delrec.selective import causal_conv, selective_scan
    c = put(scan_case(30, 2, 24, 16, FP32, False), dev)
    half = {k: c[k].bfloat16() for k in ('A', 'D', 'dt_bias')}
    outs = []
    for cast in (lambda t: t, lambda t: t.float()):
        p = {k: cast(v).detach().requires_grad_(True) for k, v in half.items()}
        y, last = selective_scan(c['x'], c['dt'], p['A'], c['B'], c['C'], p['D'], c['g'], p['dt_bias'], c['h0'])
        outs.append((y, *torch.autograd.grad((y, last), list(p.values()), (c['dy'], c['dlast']))))
    assert torch.equal(outs[0][0], outs[1][0])
    for a, b in zip(outs[0][1:], outs[1][1:]):
        assert a.dtype == BF16 and torch.equal(a, b.bfloat16())
    e = put(conv_case(30, 2, 24, 4, BF16, True), dev)
    n = put(add_case((6, 5, 24), BF16, FP32), dev)

    def grads():
        d = {k: c[k].detach().requires_grad_(True) for k in LEAVES}
        y, last = selective_scan(*[d[k] for k in LEAVES])
        f = {k: e[k].detach().requires_grad_(True) for k in CONV_LEAVES}
        yc, after = causal_conv(*[f[k] for k in CONV_LEAVES], starts=e['starts'], lengths=e['lengths'])
        v = [n[k].detach().requires_grad_(True) for k in ('x', 'y', 'w')]
        x, u = add_norm(*v)
        return lambda: torch.autograd.grad((y, last, yc, after, x, u), [*d.values(), *f.values(), *v],
                                           (c['dy'], c['dlast'], e['dy'], e['dstate'], n['dx'], n['du']))
    plain = grads()()
    with torch.autograd.graph.save_on_cpu():
        later = grads()
    assert all(torch.equal(a, b) for a, b in zip(plain, later()))


@pytest.mark.gpu
def test_results_do_not_change_from_call_to_call(dev):
    c = scan_case(70, 9, 150, 16, BF16, True)
    a, b = run_scan(c, dev), run_scan(c, dev)
    assert all(torch.equal(a[k], b[k]) for k in a)


# ---------------------------------------------------------------- the convolution -----------

CONV_LEAVES = ('x', 'weight', 'bias', 'state')


def conv_case(T, B, N, W, dtype, masks, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = dict(x=rnd(g, T, B, N, dtype=dtype), weight=rnd(g, N, W), bias=rnd(g, N), state=rnd(g, B, W - 1, N, dtype=dtype),
             dy=rnd(g, T, B, N, dtype=dtype), dstate=rnd(g, B, W - 1, N, dtype=dtype))
    c.update(masks_of(g, T, B, masks))
    return c


def run_conv(c, dev, silu=True):
    from delrec.selective import causal_conv
    d = put(c, dev)
    leaves = {k: d[k].requires_grad_(True) for k in CONV_LEAVES if d[k] is not None}
    y, state = causal_conv(*[leaves.get(k) for k in CONV_LEAVES], starts=d['starts'], lengths=d['lengths'], silu=silu)
    grads = torch.autograd.grad((y, state), list(leaves.values()), (d['dy'], d['dstate']))
    return dict(y=y.detach(), after=state.detach(), **dict(zip(leaves, grads)))


def check_conv(c, dev, silu=True):
    got = run_conv(c, dev, silu)
    d = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}
    leaves = {k: d[k].clone().requires_grad_(True) for k in CONV_LEAVES if d[k] is not None}
    y, state = osel.conv(*[leaves.get(k) for k in CONV_LEAVES], d['starts'], d['lengths'], silu)
    ref = dict(zip(leaves, torch.autograd.grad((y, state), list(leaves.values()), (d['dy'], d['dstate']), allow_unused=True)))
    close(got['y'], y.detach(), ROW_TOL, 'y')
    assert torch.equal(got['after'].cpu().double(), state.detach())
    n = c['x'].shape[0] * c['x'].shape[1]
    for k in leaves:
        r = torch.zeros_like(leaves[k]) if ref[k] is None else ref[k]
        # sums of n products of gradients (slopes are at most 1.1) and inputs
        mass = {'weight': 4.0 * n, 'bias': 2.0 * n}.get(k)
        close(got[k], r, ROW_TOL, 'd' + k, mass)


CONV_SIZES = [(1, 1, 1, 4), (2, 3, 5, 4), (3, 2, 7, 8), (7, 2, 64, 2), (32, 1, 333, 3), (33, 3, 66, 4), (100, 2, 130, 5), (31, 40, 12, 6),
              (65, 1, 8, 7), (64, 2, 1, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize('masks', [False, True])
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('T,B,N,W', CONV_SIZES)
def test_conv_forward_and_gradients(dev, T, B, N, W, dtype, masks):
    check_conv(conv_case(T, B, N, W, dtype, masks), dev)


@pytest.mark.gpu
@pytest.mark.parametrize('masks', [False, True])
def test_conv_without_optional_inputs_and_activation(dev, masks):
    c = conv_case(40, 3, 70, 4, FP32, masks)
    check_conv(c, dev, silu=False)
    c.update(bias=None, state=None)
    check_conv(c, dev)


@pytest.mark.gpu
def test_conv_masked_places_strides_parts_and_steps(dev):
    from delrec.selective import causal_conv, conv_step
    T, B, N, W = 41, 4, 37, 4
    c = conv_case(T, B, N, W, FP32, True)
    want = run_conv(c, dev)
    pad = (torch.arange(T)[:, None] >= c['lengths'])[..., None]
    c['x'], c['dy'] = torch.where(pad, float('nan'), c['x']), torch.where(pad, float('inf'), c['dy'])
    got = run_conv(c, dev)
    assert all(torch.equal(got[k], want[k]) for k in want)
    # infinities before a start go no further, NaN of a state that a start drops neither
    c = conv_case(T, B, N, W, FP32, False)
    c['starts'] = torch.zeros(T, B, dtype=torch.bool)
    c['starts'][0] = c['starts'][20] = True
    c['state'].fill_(float('nan'))
    c['x'][19] = float('inf')
    got = run_conv(c, dev, silu=False)
    assert torch.isfinite(got['y'][20:]).all() and torch.isfinite(got['y'][:19]).all() and torch.isfinite(got['x']).all()
    assert float(got['state'].abs().max()) == 0.0
    for dtype in (FP32, BF16):
        c = put(conv_case(T, B, N, W, dtype, False), dev)
        y, after = causal_conv(c['x'], c['weight'], c['bias'], c['state'])
        part = torch.cat([c['x'], c['x']], -1)[..., :N]
        assert torch.equal(causal_conv(part, c['weight'], c['bias'], c['state'])[0], y)
        first = c['x'].transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(causal_conv(first, c['weight'], c['bias'], c['state'])[0], y)
        y1, mid = causal_conv(c['x'][:2], c['weight'], c['bias'], c['state'])
        y2, end = causal_conv(c['x'][2:], c['weight'], c['bias'], mid)
        assert torch.equal(torch.cat([y1, y2]), y) and torch.equal(end, after)
        state = c['state'].clone()
        for t in range(T):
            yt, s2 = conv_step(c['x'][t], state, c['weight'], c['bias'], state_out=state)
            assert s2.data_ptr() == state.data_ptr() and torch.equal(yt, y[t])
        assert torch.equal(state, after)
        yt, s2 = conv_step(c['x'][0], c['state'], c['weight'], c['bias'])
        assert torch.equal(yt, y[0]) and torch.equal(s2[:, :-1], c['state'][:, 1:]) and torch.equal(s2[:, -1], c['x'][0])


# ---------------------------------------------------------------- addition and norm ---------

def run_add(c, dev, pack=False, eps=1e-6):
    from delrec.gated import add_norm
    leaves = [c[k].to(dev).requires_grad_(True) for k in ('x', 'y', 'w')]
    out = add_norm(*leaves, eps=eps, pack=pack)
    grads = torch.autograd.grad(out[:2], leaves, (c['dx'].to(dev), c['du'].to(dev)))
    return out, grads


def add_case(shape, dtype, resid, seed=0):
    g = torch.Generator().manual_seed(seed)
    return dict(x=rnd(g, *shape, dtype=resid), y=rnd(g, *shape, dtype=dtype), w=1 + rnd(g, shape[-1], std=0.3),
                dx=rnd(g, *shape, dtype=resid), du=rnd(g, *shape, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,resid', [(FP32, FP32), (BF16, BF16), (BF16, FP32)])
@pytest.mark.parametrize('shape', [(1, 2), (5, 3), (3, 4), (7, 64), (33, 65), (5, 3, 130), (200, 255), (9, 513), (3, 1001), (2, 3, 2048),
                                   (3, 4097), (2, 8192), (2, 8193), (1300, 4), (700, 320)])
def test_add_norm(dev, shape, dtype, resid):
    from delrec.checkpoint8 import pack8, unpack8
    c = add_case(shape, dtype, resid)
    (x, u, p), grads = run_add(c, dev, pack=True)
    d = {k: v.double() for k, v in c.items()}
    leaves = [d[k].clone().requires_grad_(True) for k in ('x', 'y', 'w')]
    rx, ru = osel.add_norm(*leaves, 1e-6)
    ref = torch.autograd.grad((rx, ru), leaves, (d['dx'], d['du']))
    close(x, rx.detach(), ROW_TOL, "x'")
    close(u, ru.detach(), ROW_TOL, 'u')
    rows = d['x'].numel() // shape[-1]
    for name, got, r in zip(('dx', 'dy', 'dw'), grads, ref):
        assert got.dtype == dict(dx=resid, dy=dtype, dw=FP32)[name]
        close(got, r, ROW_TOL, name, mass=8.0 * rows if name == 'dw' else None)
    own = pack8(u)
    assert torch.equal(p.q, own.q) and torch.equal(p.scale, own.scale)
    assert torch.equal(unpack8(p).cpu().double(), og.round8(u.cpu())[0].to(dtype).double())
    (x2, u2), grads2 = run_add(c, dev)
    assert torch.equal(x, x2) and torch.equal(u, u2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


@pytest.mark.gpu
def test_add_norm_strides_and_single_gradients(dev):
    from delrec.gated import add_norm
    for dtype, resid in ((FP32, FP32), (BF16, FP32), (BF16, BF16)):
        c = add_case((6, 5, 96), dtype, resid)
        (x, u), grads = run_add(c, dev)
        d = put(c, dev)
        xt = d['x'].transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True)
        yw = torch.cat([d['y'], d['y']], -1)[..., :96].detach().requires_grad_(True)
        x2, u2 = add_norm(xt, yw, d['w'])
        g2 = torch.autograd.grad((x2, u2), (xt, yw), (d['dx'].transpose(0, 1).contiguous().transpose(0, 1), d['du']))
        assert torch.equal(x, x2) and torch.equal(u, u2) and torch.equal(g2[0], grads[0]) and torch.equal(g2[1], grads[1])
        # one output used, the other not
        leaves = [d[k].detach().requires_grad_(True) for k in ('x', 'y', 'w')]
        x2, u2 = add_norm(*leaves)
        gx = torch.autograd.grad(x2, leaves, d['dx'], retain_graph=True)
        assert torch.equal(gx[0], d['dx']) and torch.equal(gx[1], d['dx'].to(dtype)) and float(gx[2].abs().max()) == 0.0
        gu = torch.autograd.grad(u2, leaves, d['du'])
        r = [c[k].double().requires_grad_(True) for k in ('x', 'y', 'w')]
        ref = torch.autograd.grad(osel.add_norm(*r, 1e-6)[1], r, c['du'].double())
        close(gu[0], ref[0], ROW_TOL, 'dx of u')
        # an input added to itself
        s = d['y'].detach().requires_grad_(True)
        x2, u2 = add_norm(s, s, d['w'])
        (gs,) = torch.autograd.grad((x2, u2), s, (d['dx'].to(dtype), d['du']))
        t = c['y'].double().requires_grad_(True)
        (rs,) = torch.autograd.grad(osel.add_norm(t, t, c['w'].double(), 1e-6), t, (c['dx'].to(dtype).double(), c['du'].double()))
        # (the engine adds the two gradients in their type: a rounding of each and of the sum)
        close(gs, rs, ROW_TOL + (2.0 ** -8 if dtype == BF16 else 0.0), 'twice')


@pytest.mark.gpu
def test_changes_in_place_are_noticed(dev):
    from delrec.gated import add_norm
    from delrec.selective import causal_conv, conv_step, selective_scan, selective_step
    for shape, dtype, resid in (((3, 8), FP32, FP32), ((2, 3, 8), BF16, FP32), ((2, 3, 8), BF16, BF16), ((2, 2, 3, 8), FP32, FP32),
                                ((8,), FP32, FP32)):
        c = put(add_case(shape, dtype, resid), dev)
        for which in (0, 1, 2):
            x, y = c['x'].clone(), c['y'].clone()
            w = c['w'].clone().requires_grad_(True)
            xo, u = add_norm(x, y, w)
            hit = (x, y, xo)[which]
            kept = which == 2 if resid == FP32 else which < 2
            with torch.no_grad():
                hit.add_(1)
            if kept:
                with pytest.raises(RuntimeError, match='modified by an inplace'):
                    u.sum().backward()
            else:
                u.sum().backward()
    c = put(scan_case(5, 2, 8, 4, FP32, False), dev)
    for k in ('x', 'dt', 'B', 'C', 'g'):
        d = {n: v.clone() if v is not None else None for n, v in c.items()}
        d['A'].requires_grad_(True)
        y, _ = selective_scan(*[d[n] for n in LEAVES])
        d[k].add_(1)
        with pytest.raises(RuntimeError, match='modified by an inplace'):
            y.sum().backward()
    # a step in place counts as a change of the state
    d = put(scan_case(5, 2, 8, 4, FP32, False), dev)
    v = d['h0']._version
    with torch.no_grad():
        selective_step(d['x'][0], d['dt'][0], d['A'], d['B'][0], d['C'][0], d['h0'], h_out=d['h0'])
    assert d['h0']._version > v
    e = put(conv_case(5, 2, 8, 4, FP32, False), dev)
    v = e['state']._version
    conv_step(e['x'][0], e['state'], e['weight'], state_out=e['state'])
    assert e['state']._version > v
    x = e['x'].clone()
    y, _ = causal_conv(x, e['weight'].requires_grad_(True))
    x.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        y.sum().backward()


# ---------------------------------------------------------------- streams, graphs, refusals -

@pytest.mark.gpu
def test_on_another_stream_and_captured(dev):
    from delrec.gated import add_norm
    from delrec.selective import causal_conv, conv_step, selective_scan, selective_step
    c = scan_case(50, 3, 70, 16, BF16, True)
    e = conv_case(50, 3, 70, 4, BF16, True)
    a = add_case((150, 70), BF16, FP32)
    want = run_scan(c, dev), run_conv(e, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_scan(c, dev), run_conv(e, dev)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(g[k], w[k]) for k in w)
    d, f, s = put(c, dev), put(e, dev), put(a, dev)
    h, cs = d['h0'].clone(), f['state'].clone()

    def forward():
        with torch.no_grad():
            y, last = selective_scan(*[d[k] for k in LEAVES], starts=d['starts'], lengths=d['lengths'])
            yc, after = causal_conv(f['x'], f['weight'], f['bias'], f['state'], f['starts'], f['lengths'])
            x, u, p = add_norm(s['x'], s['y'], s['w'], pack=True)
            ys, _ = selective_step(d['x'][0], d['dt'][0], d['A'], d['B'][0], d['C'][0], h, d['D'], d['g'][0], d['dt_bias'], h_out=h)
            yt, _ = conv_step(f['x'][0], cs, f['weight'], f['bias'], state_out=cs)
        return y, last, yc, after, x, u, p.q, p.scale, ys, yt
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        forward()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = forward()
    for i in range(3):
        for t in (d['x'], f['x'], s['y']):
            t.mul_(-0.5)
        h.copy_(d['h0']), cs.copy_(f['state'])
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in (*outs, h, cs)]
        h.copy_(d['h0']), cs.copy_(f['state'])
        eager = forward()
        assert all(torch.equal(x, y) for x, y in zip(kept, (*eager, h, cs))), i


@pytest.mark.gpu
def test_refusals(dev):
    from delrec.checkpoint8 import linear8
    from delrec.gated import add_norm
    from delrec.selective import causal_conv, conv_step, selective_scan, selective_step
    x, low, A = torch.zeros(3, 2, 4, device=dev), torch.zeros(3, 2, 5, device=dev), torch.zeros(4, 5, device=dev)
    h = torch.zeros(2, 4, 5, device=dev)
    bad = [lambda: selective_scan(x[0], x[0], A, low, low), lambda: selective_scan(x, x[:2], A, low, low),
           lambda: selective_scan(x, x.bfloat16(), A, low, low), lambda: selective_scan(x, x, A, low.bfloat16(), low),
           lambda: selective_scan(x, x, A, low, low[..., :4]), lambda: selective_scan(x, x, A[:3], low, low),
           lambda: selective_scan(x, x, torch.zeros(4, 65, device=dev), torch.zeros(3, 2, 65, device=dev), torch.zeros(3, 2, 65, device=dev)),
           lambda: selective_scan(x, x, A[:, :0], low[..., :0], low[..., :0]), lambda: selective_scan(x.half(), x.half(), A, low.half(), low.half()),
           lambda: selective_scan(x, x, A, low, low, D=torch.zeros(5, device=dev)), lambda: selective_scan(x, x, A, low, low, g=x[:, :1]),
           lambda: selective_scan(x, x, A, low, low, h0=h.double()), lambda: selective_scan(x, x, A, low, low, h0=h.cpu()),
           lambda: selective_scan(x, x, A, low, low, starts=torch.zeros(2, 2, device=dev)),
           lambda: selective_scan(x, x, A, low, low, lengths=torch.zeros(2, device=dev)),
           lambda: selective_scan(x, x, A.cpu(), low, low), lambda: selective_scan(x[:, :0], x[:, :0], A, low[:, :0], low[:, :0]),
           lambda: selective_step(x[0], x[0], A, low[0], low[0], h[:1]), lambda: selective_step(x[0], x[0], A, low[0, :1], low[0], h),
           lambda: selective_step(x[0], x[0], A, low[0], low[0], h, h_out=h.transpose(0, 1).contiguous().transpose(0, 1)),
           lambda: causal_conv(x, torch.zeros(4, 9, device=dev)), lambda: causal_conv(x, torch.zeros(4, 1, device=dev)),
           lambda: causal_conv(x, torch.zeros(5, 4, device=dev)), lambda: causal_conv(x, torch.zeros(4, 4, device=dev), state=x),
           lambda: causal_conv(x, torch.zeros(4, 4, device=dev), state=torch.zeros(2, 3, 4, device=dev, dtype=BF16)),
           lambda: causal_conv(x[0], torch.zeros(4, 4, device=dev)), lambda: causal_conv(x.double(), torch.zeros(4, 4, device=dev)),
           lambda: conv_step(x[0], x[:, :, :3], torch.zeros(4, 4, device=dev)), lambda: add_norm(x, x[:2], torch.ones(4, device=dev)),
           lambda: add_norm(x.bfloat16(), x, torch.ones(4, device=dev)), lambda: add_norm(x, x, torch.ones(5, device=dev)),
           lambda: add_norm(x, x, None), lambda: add_norm(x[..., :1], x[..., :1], torch.ones(1, device=dev))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print(i)
    w = torch.zeros(4, 4, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match='no backward'):
        conv_step(x[0], torch.zeros(2, 3, 4, device=dev), w)
    with pytest.raises(RuntimeError, match='no backward'):
        selective_step(x[0], x[0], A.clone().requires_grad_(True), low[0], low[0], h)
    y, _ = causal_conv(x, w)
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(y.sum(), w, create_graph=True)
    y, _ = causal_conv(x, w)
    y.sum().backward()
    with pytest.raises(RuntimeError, match='second time'):
        y.sum().backward()
    _, u, p = add_norm(x, x, torch.ones(4, device=dev), pack=True)
    with pytest.raises(ValueError, match='packed'):
        linear8(u[:2], w, packed=p)


@pytest.mark.gpu
def test_no_steps(dev):
    from delrec.selective import causal_conv, selective_scan
    c = put(scan_case(4, 2, 8, 4, FP32, False), dev)
    leaves = {k: c[k].clone().requires_grad_(True) for k in LEAVES}
    args = [leaves[k][:0] if k in ('x', 'dt', 'B', 'C', 'g') else leaves[k] for k in LEAVES]
    y, last = selective_scan(*args)
    assert y.shape == (0, 2, 8) and torch.equal(last, c['h0'])
    for g in torch.autograd.grad((y, last), list(leaves.values()), (torch.zeros_like(y), torch.zeros_like(last))):
        assert float(g.abs().sum()) == 0.0
    e = put(conv_case(4, 2, 8, 4, BF16, False), dev)
    y, state = causal_conv(e['x'][:0], e['weight'], e['bias'], e['state'])
    assert y.shape == (0, 2, 8) and y.dtype == BF16 and torch.equal(state, e['state'])


# ---------------------------------------------------------------- the block and the model ---

class Config:
    input_size, hidden_layers, output_size, bias = 8, [32, 32], 4, True


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [False, True])
def test_model_gradients_against_the_definitions(dev, checkpoint):
    """The whole model in 64 bits on the CPU from the definitions. 8-bit inputs change the gradients of
    what keeps them: of a Linear's weight, and of the first norm and, through it, the embedding. A kept
    value is off by at most 0.502 / 127 of its group's largest, which for a normed row of 32 is at most
    sqrt(32) = 5.7: each term of those sums by at most 0.023 of the gradient that it multiplies."""
    from delrec.networks import RNN_selective
    torch.manual_seed(0)
    cfg = type('C', (Config,), dict(checkpoint8=checkpoint))
    m = RNN_selective(cfg).to(dev)
    ref = RNN_selective(Config).double()
    ref.load_state_dict({k: v.double().cpu() for k, v in m.state_dict().items()})
    g = torch.Generator().manual_seed(1)
    T, B = 21, 3
    x = torch.randn(T, B, 8, generator=g)
    starts = torch.rand(T, B, generator=g) < 0.1
    lengths = torch.tensor([T, 9, 0])
    dy = torch.randn(T, B, 4, generator=g)
    y = m(x.to(dev), starts=starts.to(dev), lengths=lengths.to(dev))
    y.backward(dy.to(dev))
    r = ref.embed(x.double())
    u = og.norm_gate(None, None, r, None, None, ref.norm_weight, 1e-6)[1]
    for b in ref.blocks:
        c, gate = b.proj(u).chunk(2, -1)
        c, _ = osel.conv(c, b.conv_weight, b.conv_bias, None, starts, lengths)
        low, Bm, C = b.low(c).split([b.rank, b.S, b.S], -1)
        h, _ = osel.scan(c, b.dt(low), -torch.exp(b.A_log), Bm, C, b.D, gate, b.dt_bias, None, starts, lengths)
        r, u = osel.add_norm(r, b.out(h), b.next_weight, 1e-6)
    out = ref.readout(u)
    out.backward(dy.double())
    close(y, out.detach(), SCAN_TOL, 'y')
    for (name, p), q in zip(m.named_parameters(), ref.parameters()):
        eight = checkpoint and (name.endswith('proj.weight') or name in ('readout.weight', 'norm_weight') or name.startswith('embed'))
        close(p.grad, q.grad, 0.023 if eight else 1e-3, name)


@pytest.mark.gpu
def test_model_streams_where_the_prompt_ended(dev):
    """``step`` by step from the state that a prompt left equals the whole sequence at once."""
    from delrec.networks import RNN_selective
    torch.manual_seed(0)
    m = RNN_selective(Config).to(dev)
    x = torch.randn(30, 5, 8, device=dev)
    with torch.no_grad():
        full = m(x)
        _, state = m(x[:17], return_state=True)
        for t in range(17, 30):
            y, state = m.step(x[t], state)
            close(y, full[t].double().cpu(), 1e-3, f'step {t}')
        y, _ = m.step(x[0])
        close(y, full[0].double().cpu(), 1e-3, 'first')
        with torch.autocast('cuda', BF16):
            half = m(x)
            state = None
            for t in range(3):
                y, state = m.step(x[t], state)
    assert half.dtype == BF16 and float((half.float() - full).norm() / full.norm()) < 0.05
    assert float((y.float() - full[2]).norm() / full[2].norm()) < 0.05


@pytest.mark.gpu
def test_model_trains_on_the_memorisation_task(dev):
    from configs.perf_MEM import Config as Mem
    from delrec.training import mem
    cfg = Mem()
    cfg.model, cfg.hidden_layers, cfg.epochs, cfg.num_samples, cfg.checkpoint8 = 'RNN_selective', [32, 32], 2, 64, True
    history, final = mem.run(cfg, 'cuda')
    assert len(history) == 2 and final['num_samples'] == 64
