"""The gated recurrence, the norms with gate and residual, and the 8-bit checkpoints against
their definitions in 64 bits.

Tolerances. In fp32 a state takes one rounding per step (6e-8 of its size) and the gate's error
(at most 1e-6 relative for gates up to 16 in magnitude), and keeps them for at most the steps a
leak remembers: over the 300 steps here at most 3e-5 of the largest value, random signs far
less. Row operations lose a few roundings and the gate's error: 1e-5 of the largest value.
bf16 outputs add half a unit in the 8th bit, 2^-8 of their own size at most. Sums over rows
carry the same relative errors on the sum of magnitudes."""

import pytest
import torch

from oracle import gated as og

BF16, FP32 = torch.bfloat16, torch.float32


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
    assert int(bad.sum()) == 0, f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got64 - ref).abs().max()):.3e}, largest {ref.abs().max():.3e}'


def rnd(gen, *shape, dtype=FP32, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def scan_case(T, B, N, dtype, masks, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = dict(z=rnd(g, T, B, N, dtype=dtype), f=rnd(g, T, B, N, dtype=dtype), bias=torch.rand(N, generator=g) * 6,
             h0=rnd(g, B, N), dh=rnd(g, T, B, N, dtype=dtype), dlast=rnd(g, B, N), starts=None, lengths=None)
    if masks:
        c['starts'] = torch.rand(T, B, generator=g) < 0.1
        c['lengths'] = torch.randint(0, T + 1, (B,), generator=g)
        c['lengths'][0] = 0
        if B > 1:
            c['lengths'][1] = T
    return c


def run_scan(c, dev, checkpoint=False):
    from delrec.gated import gated_scan
    leaves = [c[k].to(dev).requires_grad_(True) for k in ('z', 'f', 'bias', 'h0')]
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    h, last = gated_scan(*leaves, starts=to(c['starts']), lengths=to(c['lengths']), checkpoint=checkpoint)
    grads = torch.autograd.grad((h, last), leaves, (c['dh'].to(dev), c['dlast'].to(dev)))
    return h, last, *grads


def check_scan(c, dev, checkpoint=False):
    got = run_scan(c, dev, checkpoint)
    d = {k: v.double() for k, v in c.items() if k not in ('starts', 'lengths')}
    ref = og.scan_grads(d['z'], d['f'], d['bias'], d['h0'], c['starts'], c['lengths'], d['dh'], d['dlast'], checkpoint)
    for name, x, y in zip(('h', 'last', 'dz', 'df', 'db', 'dh0'), got, ref):
        close(x, y, 3e-5, name, mass=float(ref[3].abs().sum((0, 1)).max()) if name == 'db' else None)


SCAN_SIZES = [(1, 1, 1), (1, 3, 65), (2, 2, 3), (63, 2, 5), (64, 3, 64), (65, 1, 130), (130, 4, 333), (300, 2, 256),
              (257, 5, 7), (40, 33, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [False, True])
@pytest.mark.parametrize('masks', [False, True])
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('T,B,N', SCAN_SIZES)
def test_scan_forward_and_gradients(dev, T, B, N, dtype, masks, checkpoint):
    check_scan(scan_case(T, B, N, dtype, masks), dev, checkpoint)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('T,B,N', [(130, 3, 68), (65, 2, 33)])
def test_scan_strides(dev, T, B, N, dtype):
    """Column slices of one projection, batch-first tensors and their gradients, reversed time."""
    from delrec.gated import gated_scan
    c = scan_case(T, B, N, dtype, False)
    want = run_scan(c, dev)
    proj = torch.cat([c['z'], c['f'], c['z']], -1).to(dev).requires_grad_(True)
    first = c['dh'].to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    z, f, _ = proj.chunk(3, -1)
    h, last = gated_scan(z, f, c['bias'].to(dev), c['h0'].to(dev))
    (dp,) = torch.autograd.grad((h, last), (proj,), (first, c['dlast'].to(dev)))
    assert torch.equal(h, want[0]) and torch.equal(last, want[1])
    assert torch.equal(dp[..., :N], want[2]) and torch.equal(dp[..., N:2 * N], want[3])
    bf = [c[k].to(dev).transpose(0, 1).contiguous().transpose(0, 1) for k in ('z', 'f')]
    h, last = gated_scan(*bf, c['bias'].to(dev), c['h0'].to(dev))
    assert torch.equal(h, want[0]) and torch.equal(last, want[1])
    # a last axis that is not contiguous, and one value for every step
    wide = torch.stack([c['z'], c['z']], -1).to(dev)[..., 0]
    assert torch.equal(gated_scan(wide, c['f'].to(dev), c['bias'].to(dev), c['h0'].to(dev))[0], want[0])
    one = c['f'][:1].to(dev).expand(T, B, N)
    assert torch.equal(gated_scan(c['z'].to(dev), one)[0], gated_scan(c['z'].to(dev), one.contiguous())[0])


@pytest.mark.gpu
@pytest.mark.parametrize('T,B,N', [(20, 3, 5), (130, 4, 64)])
def test_scan_masked_places_may_hold_anything(dev, T, B, N):
    """Padding holds NaN and infinities, and a state before a start is infinite: neither reaches
    an output or a gradient."""
    c = scan_case(T, B, N, FP32, True)
    want = run_scan(c, dev)
    pad = torch.arange(T)[:, None] >= c['lengths']
    for k, bad in (('z', float('nan')), ('f', float('inf')), ('dh', float('nan'))):
        c[k] = torch.where(pad[..., None], bad, c[k])
    for a, b in zip(run_scan(c, dev), want):
        assert torch.equal(a, b)
    for checkpoint in (False, True):
        assert all(torch.isfinite(t).all() for t in run_scan(c, dev, checkpoint))
    c['starts'][0] = True
    c['lengths'][:] = T
    c['z'], c['f'], c['dh'] = (scan_case(T, B, N, FP32, True)[k] for k in ('z', 'f', 'dh'))
    want = run_scan(c, dev)
    c['h0'][:] = float('inf')
    got = run_scan(c, dev)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not got[5].any()


@pytest.mark.gpu
def test_scan_nan_spreads_to_its_own_channel_only(dev):
    c = scan_case(200, 2, 70, FP32, False)
    c['z'][10, 1, 3] = float('nan')
    h, last, dz, df, db, dh0 = run_scan(c, dev)
    bad = torch.zeros(200, 2, 70, dtype=torch.bool)
    bad[10:, 1, 3] = True
    assert torch.equal(torch.isnan(h).cpu(), bad) and torch.equal(torch.isnan(last).cpu(), bad[-1])
    assert torch.isfinite(dz).all() and torch.isnan(db).sum() == 1


@pytest.mark.gpu
def test_scan_saturated_gates(dev):
    """Gates that keep everything or take everything."""
    from delrec.gated import gated_scan
    z = torch.randn(100, 2, 8, generator=torch.Generator().manual_seed(1)).to(dev)
    h0 = torch.ones(2, 8, device=dev)
    h, last = gated_scan(z, torch.full_like(z, 200.0), h0=h0)
    assert torch.equal(h, torch.ones_like(h)) and torch.equal(last, h0)
    h, _ = gated_scan(z, torch.full_like(z, -200.0), h0=h0)
    torch.testing.assert_close(h, z, rtol=0, atol=2.0 ** -22 * float(z.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize('T,B,N,dtype', [(5000, 1, 8, FP32), (3001, 2, 70, BF16), (4096, 1, 300, FP32)])
@pytest.mark.parametrize('masks', [False, True])
def test_scan_long(dev, T, B, N, dtype, masks):
    """Long sequences of few channels. Leaks here remember at most a few hundred steps, so the
    errors stay those of 300 steps."""
    check_scan(scan_case(T, B, N, dtype, masks, seed=5), dev)
    check_scan(scan_case(T, B, N, dtype, masks, seed=6), dev, checkpoint=True)


@pytest.mark.gpu
def test_scan_gradient_against_differences(dev):
    """Directional central differences of the 64-bit forward: their own error is below 1e-7 of
    the sum of magnitudes, the kernel's gradients' 3e-5."""
    c = scan_case(90, 2, 12, FP32, True, seed=3)
    got = run_scan(c, dev)
    d = {k: v.double() for k, v in c.items() if k not in ('starts', 'lengths')}
    g = torch.Generator().manual_seed(8)

    def loss(z, f, bias, h0):
        h, last, _ = og.scan(z, f, bias, h0, c['starts'], c['lengths'])
        return float((h * d['dh']).sum() + (last * d['dlast']).sum())
    base = [d[k] for k in ('z', 'f', 'bias', 'h0')]
    for k in range(4):
        way = torch.randn(base[k].shape, generator=g, dtype=torch.float64)
        hi, lo = ([t + s * way if i == k else t for i, t in enumerate(base)] for s in (1e-5, -1e-5))
        diff = (loss(*hi) - loss(*lo)) / 2e-5
        grad = got[2 + k].double().cpu()
        assert abs(float((grad * way).sum()) - diff) <= 1e-4 * float((grad * way).abs().sum())


@pytest.mark.gpu
def test_scan_empty_and_partial_gradients(dev):
    from delrec.gated import gated_scan
    h0 = torch.randn(3, 4, device=dev, requires_grad=True)
    h, last = gated_scan(torch.empty(0, 3, 4, device=dev), torch.empty(0, 3, 4, device=dev), h0=h0)
    assert h.shape == (0, 3, 4) and torch.equal(last, h0)
    z = torch.randn(70, 3, 4, device=dev, requires_grad=True)
    f = torch.randn(70, 3, 4, device=dev)
    h, last = gated_scan(z, f)
    (dz,) = torch.autograd.grad(last.sum(), z, retain_graph=True)
    (dy,) = torch.autograd.grad(h[-1].sum(), z)
    torch.testing.assert_close(dz, dy, rtol=1e-6, atol=0)
    with torch.no_grad():
        h2, last2 = gated_scan(z, f)
    assert torch.equal(h, h2) and torch.equal(last, last2) and not h2.requires_grad


@pytest.mark.gpu
def test_scan_in_pieces_is_the_scan(dev):
    """The state handed on between two calls, and one step at a time."""
    from delrec.gated import gated_scan
    c = scan_case(130, 3, 68, FP32, False)
    z, f, b = (c[k].to(dev) for k in ('z', 'f', 'bias'))
    h, last = gated_scan(z, f, b)
    a, s = gated_scan(z[:50], f[:50], b)
    e, s = gated_scan(z[50:], f[50:], b, h0=s)
    big = float(h.abs().max())
    torch.testing.assert_close(torch.cat([a, e]), h, rtol=0, atol=3e-5 * big)
    torch.testing.assert_close(s, last, rtol=0, atol=3e-5 * big)


@pytest.mark.gpu
def test_scan_refusals(dev):
    from delrec.gated import gated_scan
    z = torch.zeros(4, 2, 8, device=dev)
    for kw in (dict(f=z[:3]), dict(f=z.to(BF16)), dict(f=z.cpu()), dict(bias=torch.zeros(7, device=dev)),
               dict(bias=torch.zeros(8)), dict(h0=torch.zeros(2, 7, device=dev)),
               dict(h0=torch.zeros(2, 8, device=dev, dtype=BF16)), dict(starts=torch.zeros(4, 3, device=dev)),
               dict(lengths=torch.zeros(2, device=dev)), dict(lengths=torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            gated_scan(z, **{'f': z, **kw})
    with pytest.raises(ValueError):
        gated_scan(z.half(), z.half())
    with pytest.raises(ValueError):
        gated_scan(z[0], z[0])
    # lengths past the end count as the end, below zero as empty
    o = torch.ones_like(z)
    h, _ = gated_scan(o, o, lengths=torch.tensor([1 << 40, -5], device=dev))
    assert (h[:, 0] > 0).all() and not h[:, 1].any()


# ---------------------------------------------------------------- norms ---------------------

def norm_case(shape, dtype, resid, seed=0):
    g = torch.Generator().manual_seed(seed)
    N = shape[-1]
    return dict(o=rnd(g, *shape, dtype=dtype, std=0.5), g=rnd(g, *shape, dtype=dtype), x=rnd(g, *shape, dtype=resid),
                w=1 + rnd(g, N, std=0.1), scale=torch.rand(N, generator=g), w2=1 + rnd(g, N, std=0.1),
                dxo=rnd(g, *shape, dtype=resid), du=rnd(g, *shape, dtype=dtype))


NAMES = ('o', 'g', 'x', 'w', 'scale', 'w2')


def run_norm(c, dev, checkpoint=False, eps=1e-6):
    from delrec.gated import norm_gate_residual
    leaves = [c[k].to(dev).requires_grad_(True) for k in NAMES]
    xo, u = norm_gate_residual(*leaves, eps=eps, checkpoint=checkpoint)
    return xo, u, *torch.autograd.grad((xo, u), leaves, (c['dxo'].to(dev), c['du'].to(dev)))


def ref_norm(c, checkpoint=False, eps=1e-6):
    d = {k: v.double() for k, v in c.items()}
    leaves = [d[k].requires_grad_(True) for k in NAMES]
    xo, u = og.norm_gate(*leaves, eps)
    if checkpoint:
        grads = og.norm_gate_grads8(*(t.detach() for t in leaves), eps, d['dxo'], d['du'])
    else:
        grads = torch.autograd.grad((xo, u), leaves, (d['dxo'], d['du']))
    return xo.detach(), u.detach(), *grads


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [False, True])
@pytest.mark.parametrize('dtype,resid', [(FP32, FP32), (BF16, BF16), (BF16, FP32)])
@pytest.mark.parametrize('shape', [(3, 2), (5, 3), (7, 64), (33, 65), (4, 5, 127), (9, 3, 256), (600, 260),
                                   (17, 700), (6, 1500), (5, 2049), (3, 5000), (4, 4099), (9, 4096), (2, 17000)])
def test_norm_gate_forward_and_gradients(dev, shape, dtype, resid, checkpoint):
    c = norm_case(shape, dtype, resid)
    got, ref = run_norm(c, dev, checkpoint), ref_norm(c, checkpoint)
    rows = c['x'].numel() // shape[-1]
    for name, a, b in zip(('xo', 'u') + NAMES, got, ref):
        mass = None
        if name in ('w', 'scale', 'w2'):
            mass = 16.0 * rows       # terms are products of values of order one, each below 16
        close(a, b, 1e-5 if mass is None else 1e-6, name, mass)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('shape', [(3, 64), (40, 130), (2, 3, 1000)])
def test_rms_norm(dev, shape, dtype):
    from delrec.gated import rms_norm
    for checkpoint in (False, True):
        c = norm_case(shape, dtype, dtype, seed=2)
        x, w = c['x'].to(dev).requires_grad_(True), c['w2'].to(dev).requires_grad_(True)
        u = rms_norm(x, w, checkpoint=checkpoint)
        dx, dw = torch.autograd.grad(u, (x, w), c['du'].to(dev))
        X, W = c['x'].double().requires_grad_(True), c['w2'].double().requires_grad_(True)
        U = og.norm_gate(None, None, X, None, None, W, 1e-6)[1]
        close(u, U.detach(), 1e-5, 'u')
        if checkpoint:
            zero, one = torch.zeros_like(X.detach()), torch.zeros_like(W.detach())
            g = og.norm_gate_grads8(zero, zero, X.detach(), one, one, W.detach(), 1e-6, zero, c['du'].double())
            RX, RW = g[2], g[5]
        else:
            RX, RW = torch.autograd.grad(U, (X, W), c['du'].double())
        close(dx, RX, 1e-5, 'dx')
        close(dw, RW, 1e-6, 'dw', mass=16.0 * x.numel() / shape[-1])


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [False, True])
def test_norm_gate_without_next_norm_and_partial_gradients(dev, checkpoint):
    from delrec.gated import norm_gate_residual
    c = norm_case((50, 130), FP32, FP32, seed=4)
    L = {k: c[k].to(dev).requires_grad_(True) for k in NAMES}
    xo, u = norm_gate_residual(L['o'], L['g'], L['x'], L['w'], L['scale'], checkpoint=checkpoint)
    assert u is None
    got = torch.autograd.grad(xo, [L[k] for k in NAMES[:5]], c['dxo'].to(dev))
    c0 = dict(c, du=torch.zeros_like(c['du']))
    ref = ref_norm(c0, checkpoint)
    for name, a, b in zip(NAMES, got, ref[2:]):
        close(a, b, 1e-5 if a.dim() == 2 else 1e-6, name, None if a.dim() == 2 else 16.0 * 50)
    # only u is used
    xo, u = norm_gate_residual(*(L[k] for k in NAMES), checkpoint=checkpoint)
    got = torch.autograd.grad(u, [L[k] for k in NAMES], c['du'].to(dev))
    ref = ref_norm(dict(c, dxo=torch.zeros_like(c['dxo'])), checkpoint)
    for name, a, b in zip(NAMES, got, ref[2:]):
        close(a, b, 1e-5 if a.dim() == 2 else 1e-6, name, None if a.dim() == 2 else 16.0 * 50)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [FP32, BF16])
def test_norm_gate_strides_and_zero_rows(dev, dtype):
    from delrec.gated import norm_gate_residual
    c = norm_case((6, 7, 68), dtype, FP32, seed=5)
    c['o'][2] = 0                       # a padded row's output
    got, ref = run_norm(c, dev), ref_norm(c)
    for name, a, b in zip(('xo', 'u') + NAMES, got, ref):
        big = None if a.dim() == 3 else 16.0 * 42
        # do of a zero row is scaled by 1/sqrt(eps)
        close(a, b, 1e-5 if a.dim() == 3 else 1e-6, name, big)
    t = {k: c[k].to(dev) for k in NAMES}
    joint = torch.cat([t['o'], t['g']], -1)
    swapped = t['x'].transpose(0, 1).contiguous().transpose(0, 1)
    o, g = joint.chunk(2, -1)
    xo, u = norm_gate_residual(o, g, swapped, t['w'], t['scale'], t['w2'])
    assert torch.equal(xo, got[0]) and torch.equal(u, got[1])
    four = norm_gate_residual(*(t[k].reshape(2, 3, 7, 68) for k in 'ogx'), t['w'], t['scale'], t['w2'])
    assert four[0].shape == (2, 3, 7, 68) and torch.equal(four[0].reshape(6, 7, 68), got[0])


@pytest.mark.gpu
def test_norm_gate_gradient_against_differences(dev):
    c = norm_case((11, 37), FP32, FP32, seed=6)
    got = run_norm(c, dev, eps=1e-3)[2:]
    d = {k: v.double() for k, v in c.items()}
    g = torch.Generator().manual_seed(9)

    def loss(*args):
        xo, u = og.norm_gate(*args, 1e-3)
        return float((xo * d['dxo']).sum() + (u * d['du']).sum())
    base = [d[k] for k in NAMES]
    for k in range(6):
        way = torch.randn(base[k].shape, generator=g, dtype=torch.float64)
        hi, lo = ([t + s * way if i == k else t for i, t in enumerate(base)] for s in (1e-5, -1e-5))
        diff = (loss(*hi) - loss(*lo)) / 2e-5
        grad = got[k].double().cpu()
        assert abs(float((grad * way).sum()) - diff) <= 1e-4 * float((grad * way).abs().sum())


@pytest.mark.gpu
def test_norm_gate_empty_and_refusals(dev):
    from delrec.gated import norm_gate_residual, rms_norm
    x = torch.zeros(0, 8, device=dev, requires_grad=True)
    w = torch.ones(8, device=dev, requires_grad=True)
    xo, u = norm_gate_residual(x, x, x, w, w, w)
    assert xo.shape == u.shape == (0, 8)
    (dw,) = torch.autograd.grad(u.sum(), w)
    assert not dw.any()
    x, w = torch.zeros(3, 8, device=dev), torch.ones(8, device=dev)
    for bad in ((x, x[:2], x, w, w), (x, x.to(BF16), x, w, w), (x, x, x.to(BF16), w, w), (x, x, x[:2], w, w),
                (x, x, x, w[:7], w), (x[:, :1], x[:, :1], x[:, :1], w[:1], w[:1]), (x, x, x, w, w.cpu()), (x, x, x, None, w), (x.half(), x.half(), x, w, w)):
        with pytest.raises(ValueError):
            norm_gate_residual(*bad)
    with pytest.raises(ValueError):
        rms_norm(x, w[:3])
    with pytest.raises(RuntimeError):
        rms_norm(x.cpu(), w)
    with pytest.raises(ValueError):                 # the norm of one column is its sign
        rms_norm(x[:, :1], w[:1])


# ---------------------------------------------------------------- 8 bits --------------------

@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('shape', [(1, 1), (3, 63), (5, 64), (4, 65), (2, 3, 700), (1000, 130), (70,), (2, 2, 3, 200)])
def test_pack8_is_its_definition(dev, shape, dtype):
    from delrec.checkpoint8 import pack8, unpack8
    x = rnd(torch.Generator().manual_seed(3), *shape, dtype=dtype) * 3
    x.view(-1)[0] = 0
    p = pack8(x.to(dev))
    value, q, scale = og.round8(x)
    assert torch.equal(p.q.cpu().float().reshape(shape), q)
    assert torch.equal(p.scale.cpu().reshape(scale.shape), scale)
    back = unpack8(p)
    assert back.dtype == dtype and back.shape == x.shape
    assert torch.equal(back.cpu(), value.float().to(dtype))


@pytest.mark.gpu
def test_pack8_strides_zeros_and_non_finite(dev):
    from delrec.checkpoint8 import pack8, unpack8
    x = torch.randn(6, 5, 200, device=dev)
    for v in (x.transpose(0, 1), x[..., 3:131], x[::2], x.transpose(1, 2), x[:1].expand(6, 5, 200)):
        want = unpack8(pack8(v.contiguous()))
        assert torch.equal(unpack8(pack8(v)), want)
    z = torch.zeros(3, 130, device=dev)
    assert not unpack8(pack8(z)).any()
    z[0, 5], z[1, 70], z[2, 129] = float('nan'), float('inf'), 1e-40
    got = torch.isnan(unpack8(pack8(z))).cpu()
    want = torch.zeros(3, 130, dtype=torch.bool)
    want[0, :64] = want[1, 64:128] = True
    assert torch.equal(got, want)
    big = torch.full((1, 64), 3.4e38, device=dev)
    assert torch.isfinite(unpack8(pack8(big))).all()
    assert unpack8(pack8(torch.empty(0, 8, device=dev))).shape == (0, 8)
    for bad in (torch.zeros(3, 8), torch.zeros(3, 8, device=dev).half(), torch.zeros(3, 0, device=dev)):
        with pytest.raises((ValueError, RuntimeError)):
            pack8(bad)


@pytest.mark.gpu
def test_linear8_gradients(dev):
    """The weight's gradient is that of the 8-bit input; the others are a Linear's."""
    from delrec.checkpoint8 import Linear8
    torch.manual_seed(0)
    lin = Linear8(70, 33).to(dev)
    x = torch.randn(5, 4, 70, device=dev, requires_grad=True)
    g = torch.randn(5, 4, 33, device=dev)
    y = lin(x)
    torch.testing.assert_close(y, torch.nn.functional.linear(x, lin.weight, lin.bias))
    dx, dw, db = torch.autograd.grad(y, (x, lin.weight, lin.bias), g)
    x8 = og.round8(x.cpu())[0].reshape(-1, 70)
    g64 = g.double().cpu().reshape(-1, 33)
    close(dw, g64.t() @ x8, 1e-5, 'dw')
    close(dx.reshape(-1, 70), g64 @ lin.weight.detach().double().cpu(), 1e-5, 'dx')
    close(db, g64.sum(0), 1e-5, 'db')


# ---------------------------------------------------------------- one step, block, model ----

@pytest.mark.gpu
@pytest.mark.parametrize('dtype,resid', [(FP32, FP32), (BF16, BF16), (BF16, FP32)])
@pytest.mark.parametrize('B,N', [(1, 2), (1, 64), (3, 70), (2, 333), (70, 256), (2, 2050), (1, 9000)])
def test_step(dev, B, N, dtype, resid):
    from delrec.gated import gated_step
    c = norm_case((B, N), dtype, resid, seed=7)
    g = torch.Generator().manual_seed(1)
    f, h, bias = rnd(g, B, N, dtype=dtype), rnd(g, B, N), torch.rand(N, generator=g) * 6
    t = {k: v.to(dev) for k, v in c.items()}
    state = h.to(dev)
    joint = torch.cat([t['o'], f.to(dev), t['g']], -1)
    zz, ff, gg = joint.chunk(3, -1)
    xo, u, hn = gated_step(zz, ff, gg, t['x'], state, t['w'], t['scale'], t['w2'], bias.to(dev))
    H = og.scan(c['o'].double()[None], f.double()[None], bias.double(), h.double())[1]
    X, U = og.norm_gate(H, c['g'].double(), c['x'].double(), c['w'].double(), c['scale'].double(), c['w2'].double(), 1e-6)
    for name, a, b in (('h', hn, H), ('xo', xo, X), ('u', u, U)):
        close(a, b, 1e-5, name)
    assert torch.equal(state.cpu(), h)
    again = gated_step(zz, ff, gg, t['x'], state, t['w'], t['scale'], t['w2'], bias.to(dev), h_out=state)
    assert again[2] is state and torch.equal(state, hn) and torch.equal(again[0], xo) and torch.equal(again[1], u)


@pytest.mark.gpu
def test_step_refusals(dev):
    from delrec.gated import gated_step
    x, w = torch.zeros(2, 8, device=dev), torch.ones(8, device=dev)
    for bad in ((x, x[:1], x, x, x, w, w), (x, x, x, x, x[:1], w, w), (x, x, x, x, x.to(BF16), w, w),
                (x, x, x, x, x, w, None), (x[None], x[None], x[None], x[None], x[None], w, w)):
        with pytest.raises(ValueError):
            gated_step(*bad)
    with pytest.raises(RuntimeError):
        gated_step(x, x, x, x, x, w.clone().requires_grad_(True), w)


@pytest.mark.gpu
def test_operators_on_another_stream(dev):
    """A side stream's results, gradients among them, are the default stream's."""
    from delrec.gated import gated_scan, norm_gate_residual
    c, n = scan_case(130, 2, 72, FP32, True), norm_case((130, 2, 72), FP32, FP32)
    t = {k: (None if v is None else v.to(dev)) for k, v in c.items()}
    w = {k: v.to(dev) for k, v in n.items()}
    z, f, b = (t[k].requires_grad_(True) for k in ('z', 'f', 'bias'))

    def step():
        h, _ = gated_scan(z, f, b, t['h0'], t['starts'], t['lengths'])
        xo, u = norm_gate_residual(h, w['g'], w['x'], w['w'], w['scale'], w['w2'], checkpoint=True)
        return (xo, u, *torch.autograd.grad((xo, u), (z, f, b), (w['dxo'], w['du'])))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step() for _ in range(3)][-1]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@torch.no_grad()
def test_forward_calls_in_a_graph(dev):
    """Captured calls replay the eager results, with the inputs changed in place and eager calls
    in between. The long scan is the one that launches more than one kernel."""
    from delrec.checkpoint8 import pack8, unpack8
    from delrec.gated import gated_scan, gated_step, norm_gate_residual
    c, n = scan_case(3000, 2, 72, FP32, True), norm_case((3000, 2, 72), FP32, FP32)
    t = {k: (None if v is None else v.to(dev)) for k, v in c.items()}
    w = {k: v.to(dev) for k, v in n.items()}

    def call():
        h, last = gated_scan(t['z'], t['f'], t['bias'], t['h0'], t['starts'], t['lengths'])
        xo, u = norm_gate_residual(h, w['g'], w['x'], w['w'], w['scale'], w['w2'])
        s = gated_step(u[0], u[1], u[2], xo[0], last, w['w'], w['scale'], w['w2'], t['bias'])
        return (h, last, xo, u, unpack8(pack8(u)), *s)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(3):
        t['z'].mul_(0.5)
        want = [v.clone() for v in call()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


@pytest.mark.gpu
@pytest.mark.parametrize('masks', [False, True])
def test_scan_offsets_past_32_bits(dev, masks):
    """Rows of the batch so far apart that their distance in bytes does not fit 32 bits."""
    from delrec.gated import gated_scan
    T, B, N, far = 70, 2, 300, (1 << 30) + 512
    c = scan_case(T, B, N, BF16, masks, seed=11)
    want = run_scan(c, dev)
    big = torch.empty(far + T * N, dtype=BF16, device=dev)
    z = big.as_strided((T, B, N), (N, far, 1))
    with torch.no_grad():
        z.copy_(c['z'].to(dev))
    c2 = {k: (None if v is None else v.to(dev)) for k, v in c.items()}
    leaves = [z.detach().requires_grad_(True)] + [c2[k].requires_grad_(True) for k in ('f', 'bias', 'h0')]
    for checkpoint in (False, True):
        h, last = gated_scan(*leaves, starts=c2['starts'], lengths=c2['lengths'], checkpoint=checkpoint)
        got = (h, last, *torch.autograd.grad((h, last), leaves, (c2['dh'], c2['dlast'])))
        ref = want if not checkpoint else run_scan(c, dev, True)
        for name, a, b in zip(('h', 'last', 'dz', 'df', 'db', 'dh0'), got, ref):
            close(a, b.detach().double().cpu(), 3e-5, name, mass=float(ref[3].double().abs().sum((0, 1)).max()) if name == 'db' else None)


# ---------------------------------------------------------------- block and model -----------

def block_reference(block, x, u, dx, du):
    """A GatedBlock's outputs and gradients in 64 bits."""
    N = x.shape[-1]
    p = {k: v.detach().double().cpu() for k, v in block.named_parameters()}
    leaves = [t.double().cpu().requires_grad_(True) for t in (x, u)] + [v.requires_grad_(True) for v in p.values()]
    z, f, g = (leaves[1] @ p['proj.weight'].t()).split(N, -1)
    h, last, _ = og.scan(z, f, p['gate_bias'])
    xo, uo = og.norm_gate(h, g, leaves[0], p['weight'], p['scale'], p['next_weight'], block.eps)
    grads = torch.autograd.grad((xo, uo), leaves, (dx.double().cpu(), du.double().cpu()))
    return xo.detach(), uo.detach(), last.detach(), dict(zip(['x', 'u', *p], grads))


@pytest.mark.gpu
def test_block_forward_and_gradients(dev):
    """The block's fp32 projection adds a rounding per product (torch's GEMM): 1e-4 of the largest."""
    from delrec.gated import GatedBlock
    torch.manual_seed(2)
    block = GatedBlock(68).to(dev)
    x, u, dx, du = (torch.randn(90, 3, 68, device=dev) for _ in range(4))
    xl, ul = x.clone().requires_grad_(True), u.clone().requires_grad_(True)
    xo, uo, last = block(xl, ul)
    params = dict(block.named_parameters())
    grads = torch.autograd.grad((xo, uo), [xl, ul, *params.values()], (dx, du))
    X, U, L, G = block_reference(block, x, u, dx, du)
    for name, a, b in (('x', xo, X), ('u', uo, U), ('last', last, L), *((k, g, G[k]) for k, g in zip(['x', 'u', *params], grads))):
        close(a, b, 1e-4, name)


@pytest.mark.gpu
def test_block_keeps_less_in_8_bits(dev):
    """Between forward and backward a checkpointed block holds about 7 bytes a channel and step
    beside its outputs (u, z, f, o, g, x in 8 bits with their scales, the states), an fp32 one 24
    and more; its gradients stay within some percent."""
    from delrec.gated import GatedBlock
    T, B, N = 512, 8, 256
    held, grads = [], []
    for checkpoint in (False, True):
        torch.manual_seed(2)
        block = GatedBlock(N, checkpoint=checkpoint).to(dev)
        gen = torch.Generator(device=dev).manual_seed(1)
        x, u, dx, du = (torch.randn(T, B, N, device=dev, generator=gen) for _ in range(4))
        x.requires_grad_(True), u.requires_grad_(True)
        out = block(x * 1.0, u * 1.0)            # inputs that the block alone keeps alive
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        params = list(block.parameters())
        grads.append(torch.autograd.grad(out[:2], [x, u, *params], (dx, du)))
        size = sum(g.numel() * g.element_size() for g in grads[-1])
        torch.cuda.synchronize()
        held.append((base + size - torch.cuda.memory_allocated()) / (T * B * N))
    assert held[1] < 8.0 and held[0] > 20.0, held
    for a, b in zip(*grads):
        assert float((a - b).norm() / a.norm()) < 0.05


def gated_config(**kw):
    from configs.perf_MEM import Config
    cfg = Config()
    cfg.hidden_layers = [64, 64]
    cfg.model = 'RNN_gated'
    for k, v in kw.items():
        setattr(cfg, k, v)
    return cfg


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [False, True])
def test_model_learns_the_memorisation_task(dev, checkpoint):
    """The task's 256 random patterns of four classes, as the spiking models train on them."""
    from delrec.training import mem
    history, final = mem.run(gated_config(epochs=60, checkpoint8=checkpoint), dev)
    assert history[0]['loss'] > final['loss'] and final['accuracy_percent'] > 90.0, (history[0], final)


@pytest.mark.gpu
def test_model_steps_are_its_scan(dev):
    """Streaming gives the sequence's outputs (fp32, the errors of 40 steps and two blocks), also
    through a captured step."""
    from delrec.networks import RNN_gated
    torch.manual_seed(4)
    model = RNN_gated(gated_config(hidden_layers=[72, 72, 72])).to(dev)
    x = torch.randn(40, 5, 8, device=dev)
    with torch.no_grad():
        want = model(x)
        state, outs = None, []
        for t in range(40):
            y, state = model.step(x[t], state)
            outs.append(y)
        torch.testing.assert_close(torch.stack(outs), want, rtol=0, atol=1e-4 * float(want.abs().max()))
        state = [torch.zeros_like(s) for s in state]
        slot = x[0].clone()
        model.step(slot, [s.clone() for s in state])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, _ = model.step(slot, state)
        for s in state:
            s.zero_()
        for t in range(40):
            slot.copy_(x[t])
            graph.replay()
            torch.cuda.synchronize()
            torch.testing.assert_close(y, outs[t], rtol=0, atol=0)


@pytest.mark.gpu
def test_model_under_autocast_and_masks(dev):
    """bf16 activations, an fp32 residual stream, and rows of several lengths: each row's outputs
    are those of the row alone."""
    from delrec.networks import RNN_gated
    torch.manual_seed(5)
    model = RNN_gated(gated_config()).to(dev)
    x = torch.randn(50, 3, 8, device=dev)
    lengths = torch.tensor([50, 17, 1], device=dev)
    with torch.autocast('cuda', torch.bfloat16):
        y = model(x, lengths=lengths)
        y.float().square().mean().backward()
    full = model(x, lengths=lengths)
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert float((y.float() - full).norm() / full.norm()) < 0.05
    for b, n in enumerate(lengths.tolist()):
        alone = model(x[:n, b:b + 1])
        torch.testing.assert_close(full[:n, b:b + 1], alone, rtol=0, atol=1e-4 * float(full.abs().max()))


@pytest.mark.gpu
def test_graph_nodes_keep_and_release(dev):
    """A second backward needs retain_graph, a changed input is noticed, second derivatives are
    refused, and a parameter's own type comes back as its gradient's."""
    from delrec.gated import gated_scan, rms_norm
    z = torch.randn(70, 2, 8, device=dev, requires_grad=True)
    f = torch.randn(70, 2, 8, device=dev)
    bias = torch.zeros(8, device=dev, dtype=BF16, requires_grad=True)
    h, _ = gated_scan(z, f, bias)
    first = torch.autograd.grad(h.sum(), (z, bias), retain_graph=True)
    again = torch.autograd.grad(h.sum(), (z, bias))
    assert all(torch.equal(a, b) for a, b in zip(first, again)) and first[1].dtype == BF16
    with pytest.raises(RuntimeError, match='second time'):
        torch.autograd.grad(h.sum(), z)
    h, _ = gated_scan(z, f)
    f.add_(1.0)
    with pytest.raises(RuntimeError, match='inplace'):
        torch.autograd.grad(h.sum(), z)
    u = rms_norm(z, torch.ones(8, device=dev))
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(u.sum(), z, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [False, True])
def test_more_than_2_to_32_values(dev, checkpoint):
    """Tensors past 2^32 values (and bytes, and odd rows): the far end of each against the same
    channels or rows by themselves, bit for bit."""
    from delrec.checkpoint8 import pack8, unpack8
    from delrec.gated import gated_scan, norm_gate_residual
    T, B, N = 66, 2, 33_000_001
    cut = (N // 64 - 1) * 64                 # whole 8-bit groups
    gen = torch.Generator(device=dev).manual_seed(1)

    def fill(*shape):
        return torch.empty(*shape, dtype=BF16, device=dev).normal_(generator=gen)
    z, f, dh = (fill(T, B, N) for _ in range(3))
    bias = torch.rand(N, device=dev, generator=gen) * 6

    def both(z, f, bias, dh):
        leaves = [t.detach().requires_grad_(True) for t in (z, f)]
        h, last = gated_scan(*leaves, bias, checkpoint=checkpoint)
        return h.detach(), last.detach(), *torch.autograd.grad(h, leaves, dh)
    far = both(*(t[:, 1:, cut:].contiguous() for t in (z, f)), bias[cut:].contiguous(), dh[:, 1:, cut:].contiguous())
    whole = both(z, f, bias, dh)
    for a, b in zip(whole, far):
        assert torch.equal(a[..., 1:, cut:], b)
    del whole, z, f, dh
    R, N = 2_150_000, 2001
    o, g, x, dx = (fill(R, N) for _ in range(4))
    w = torch.rand(N, device=dev, generator=gen) + 0.5
    rows = slice(R - 5, R)

    def norms(o, g, x, dx):
        leaves = [t.detach().requires_grad_(True) for t in (o, g, x)]
        y, u = norm_gate_residual(*leaves, w, w, w, checkpoint=checkpoint)
        return y.detach(), u.detach(), *torch.autograd.grad((y, u), leaves, (dx, dx))
    far = norms(*(t[rows].clone() for t in (o, g, x, dx)))
    for a, b in zip(norms(o, g, x, dx), far):
        assert torch.equal(a[rows], b)
    assert torch.equal(unpack8(pack8(o))[rows], unpack8(pack8(o[rows].clone())))
