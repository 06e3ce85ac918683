"""The selective block's operators where they were wrong, or untested, before: last bits of a norm's factor,
growing states in ranges of time, every shape in ranges, long runs of the convolution's backward,
states that share memory with inputs.
Tolerances as in test_gpu_selective.py unless a test derives its own."""

import pytest
import torch

from oracle import selective as osel
from test_gpu_selective import (BF16, CONV_LEAVES, FP32, LEAVES, SCAN_TOL, add_case, check_conv, check_scan, close, conv_case, masks_of, put,
                                run_conv, run_scan, scan_case)

INF, NAN = float('inf'), float('nan')


@pytest.fixture
def dev():
    return torch.device('cuda')


def workspace(kind, T, B, N, L):
    import ctypes
    from delrec import _lib
    size = ctypes.c_size_t(0)
    assert _lib.load().delrec_query_workspace(kind, T, B, N, L, 0, ctypes.byref(size)) == 0
    return size.value


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,resid', [(FP32, FP32), (BF16, FP32)])
@pytest.mark.parametrize('shape', [(300, 2), (200, 37), (500, 64), (300, 128), (300, 333), (200, 1000), (5, 40, 2048), (50, 4000), (20, 8192),
                                   (20, 9000)])
def test_add_norm_to_its_last_bit(dev, shape, dtype, resid):
    """The mean of squares from a sum in 64 bits, its root and the products each rounded once: whatever the
    width, so that u and its 8-bit codes are those of the elementary operations. (Sums in 64 bits differ by
    1e-14 with their order, which moves one rounding to 32 bits in 10^7.)"""
    from delrec.checkpoint8 import unpack8
    from delrec.gated import add_norm
    from oracle import gated as og
    c = add_case(shape, dtype, resid)
    x, u, p = add_norm(*[c[k].to(dev) for k in ('x', 'y', 'w')], pack=True)
    N = shape[-1]
    new = c['x'].float() + c['y'].float()
    mean = new.square().double().sum(-1, keepdim=True).float() * torch.tensor(1.0 / N, dtype=FP32) + torch.tensor(1e-6, dtype=FP32)
    r = (1.0 / mean.double().sqrt()).float()
    want = (new * r * c['w']).to(dtype)
    assert torch.equal(x.cpu(), new.to(resid)) and torch.equal(u.cpu(), want)
    value, codes, scale = og.round8(want.float())
    assert torch.equal(p.q.cpu().float().reshape(codes.shape), codes) and torch.equal(p.scale.cpu().reshape(scale.shape), scale)
    assert torch.equal(unpack8(p).cpu(), value.to(dtype))


@pytest.mark.gpu
def test_add_norm_of_nothing_and_of_infinities(dev):
    """Rows of zeros with and without eps, of an infinity, of values whose squares leave fp32."""
    from delrec.gated import add_norm
    for N in (3, 64, 700, 9000):
        x = torch.zeros(5, N, device=dev)
        x[1, 1], x[2, 0], x[3] = INF, NAN, 1e25
        y, w = torch.zeros_like(x), torch.ones(N, device=dev)
        _, u = add_norm(x, y, w)
        assert float(u[0].abs().max()) == 0.0 and float(u[4].abs().max()) == 0.0
        assert torch.isnan(u[1, 1]) and float(u[1, 2:].abs().max()) == 0.0 and torch.isnan(u[2]).all() and float(u[3].abs().max()) == 0.0
        _, u = add_norm(x, y, w, eps=0.0)
        assert torch.isnan(u[0]).all()


# ---------------------------------------------------------------- ranges of time ------------

def growing_case(S, T=96, step=3.0):
    """Rates of about 1: a state grows by e^3 a step, over a range of 32 steps past the largest fp32 number.
    Six blocks of 16 steps and few rows: three ranges."""
    c = scan_case(T, 2, 20, S, FP32, False)
    c['A'] = 0.9 + 0.1 * torch.rand(20, S, generator=torch.Generator().manual_seed(5))
    c['dt'].fill_(step)
    c['dt_bias'].zero_()
    return c


@pytest.mark.gpu
@pytest.mark.parametrize('S', [2, 12, 24, 40])
def test_silent_stretches_of_growing_states(dev, S):
    """A state, or a carry, of 0 stays 0 over ranges whose growth leaves fp32."""
    c = growing_case(S)
    c['h0'] = None
    c['x'][:84] = 0.0
    d = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}
    y, last = osel.scan(*[d[k] for k in LEAVES])
    from delrec.selective import selective_scan
    g = put(c, dev)
    got, end = selective_scan(*[g[k] for k in LEAVES])
    close(got, y, SCAN_TOL, 'y')
    close(end, last, SCAN_TOL, 'last')
    # the carry, from the last step to the first
    c = growing_case(S)
    c['h0'].zero_()
    c['x'].zero_()
    c['dy'][12:] = 0.0
    c['dlast'].zero_()
    check_scan(c, dev)


@pytest.mark.gpu
@pytest.mark.parametrize('S', [2, 12, 24, 40])
def test_growing_states_in_ranges(dev, S):
    """Growth by some e^14 in all, and of a tiny state by e^90 over one range. (An exponent is off by 5e-7 of
    itself at most: 4.6e-5.)"""
    c = growing_case(S, step=0.0)
    c['A'] *= 0.2
    check_scan(c, dev)
    c = growing_case(S, T=64)
    c['x'].zero_()
    c['dt'][:32], c['dt'][32:] = 2.9, -30.0
    c['A'] = 0.95 + 0.01 * torch.rand_like(c['A'])
    c['h0'] = 2e-38 * (1 + torch.rand_like(c['h0']))
    d = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}
    _, last = osel.scan(*[d[k] for k in LEAVES])
    got = run_scan(c, dev)['last'].double().cpu()
    assert float(last.abs().max()) < 1e3 and ((got - last).abs() <= 1e-4 * last).all()


@pytest.mark.gpu
@pytest.mark.parametrize('S', [2, 40])
def test_infinite_states_in_ranges(dev, S):
    """An infinite state stays infinite however far its decay goes, as step by step; a row without steps keeps
    any state at any rate."""
    c = scan_case(96, 3, 20, S, FP32, False)
    c['dt'].fill_(3.0)
    c['A'].fill_(-1.0)
    c['h0'][0] = INF
    c['lengths'] = torch.tensor([96, 96, 0])
    c['h0'][2, 4] = -INF
    c['A'][7] = NAN
    from delrec.selective import selective_scan
    g = put(c, dev)
    _, end = selective_scan(*[g[k] for k in LEAVES], lengths=g['lengths'])
    rest = [n for n in range(20) if n != 7]
    assert (end[0, rest] == INF).all() and torch.isfinite(end[1, rest]).all() and torch.isnan(end[:2, 7]).all()
    assert torch.equal(end[2].cpu(), c['h0'][2])


@pytest.mark.gpu
def test_steps_of_size_zero_in_ranges(dev):
    """They leave a state as it is over a whole range, but for what 0 times infinity gives, as step by step."""
    from delrec.selective import selective_scan
    c = scan_case(96, 3, 20, 4, FP32, False)
    c['dt'][:64] = -INF
    c['B'][5, 1, 2] = INF
    d = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}
    _, last = osel.scan(*[d[k] for k in LEAVES])
    assert int(torch.isnan(last).sum()) == 20 and torch.isnan(last[1, :, 2]).all()
    g = put(c, dev)
    _, got = selective_scan(*[g[k] for k in LEAVES])
    assert torch.equal(torch.isnan(got).cpu(), torch.isnan(last))
    close(torch.nan_to_num(got), torch.nan_to_num(last), SCAN_TOL, 'last')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('S', [2, 12, 24, 40])
def test_every_shape_in_ranges(dev, S, dtype):
    """Up to 8, 16, 32 and 64 states, each with lanes and registers of its own: starts and row ends at the
    ranges' borders, rows that end before a range begins."""
    from delrec import _lib
    T, B, N = 513, 6, 20
    assert workspace(_lib.WS_SELECTIVE_FWD, T, B, N, S) > 0       # (the ranges' maps)
    c = scan_case(T, B, N, S, dtype, True, rate=0.3)
    c['lengths'] = torch.tensor([T, 0, 1, 255, 256, 257])
    c['starts'] = torch.zeros(T, B, dtype=torch.bool)
    for t in (31, 32, 33, 255, 256, 512):
        c['starts'][t] = True
    c['starts'][:, 0] = False
    check_scan(c, dev)
    c['starts'] = None
    check_scan(c, dev)
    c['lengths'] = None
    check_scan(c, dev)


@pytest.mark.gpu
def test_step_sizes_to_their_own_size(dev):
    """softplus, as the state that a step makes of ones. The exponent -|x| log2(e) is rounded (2^-24 of itself,
    6.0e-8 |x| in the value) and its factor is off by 1.34e-8 of itself; the hardware's power and reciprocal
    are good to 2^-23 each, and four operations round to 2^-24. A decay exp(-e), e > 0, is off by 5e-7 e of
    itself likewise: since e exp(-e) <= 1 / 2.7, by at most 2e-7 and a last place of 1 in all."""
    from delrec.selective import selective_step
    x = torch.linspace(-80.0, 60.0, 100_001)[None]
    one = lambda *s: torch.ones(*s, device=dev)  # noqa: E731
    N = x.shape[1]
    _, d = selective_step(one(1, N), x.to(dev), one(N, 1), one(1, 1), one(1, 1), torch.zeros(1, N, 1, device=dev))
    want = torch.log1p(torch.exp(-x.double().abs())) + x.double().clamp(min=0)
    assert (((d[0, :, 0].double().cpu() - want[0]) / want[0]).abs() <= 5e-7 + 7.4e-8 * x[0].double().abs()).all()
    _, h = selective_step(torch.zeros(1, N, device=dev), torch.full((1, N), 2.0, device=dev), -x.abs().t().contiguous().to(dev), one(1, 1),
                          one(1, 1), one(1, N, 1))
    e = torch.nn.functional.softplus(torch.tensor(2.0, dtype=torch.float64)) * x[0].double().abs()
    assert ((h[0, :, 0].double().cpu() - torch.exp(-e)).abs() <= 2e-7 + 2.0 ** -23 + 1e-30).all()


# ---------------------------------------------------------------- runs of the convolution ---

# steps of a run of the backward, without and with masks, each more than the shortest runs' 16 - (W - 1)
LONG_RUNS = [(120, 60, 400, 4, 17, 17), (97, 40, 1030, 5, 20, 20), (200, 64, 300, 7, 22, 22), (150, 50, 700, 8, 25, 25), (350, 32, 1000, 4, 45, 25),
             (300, 40, 1024, 2, 51, 27)]


def check_runs(T, B, N, W, steps, masked):
    """The workspace holds a set of sums for each workgroup of 256 lanes (32 of them side by side): as many
    as the stated runs make."""
    from delrec import _lib
    blocks = max(-(-(-(-T // s) * B) // 8) for s in (steps, masked))
    assert N >= 125 and workspace(_lib.WS_CAUSAL_CONV_BWD, T, B, N, W) // (4 * N * (W + 1)) == blocks
    assert min(steps, masked) > 16 - (W - 1)


@pytest.mark.gpu
@pytest.mark.parametrize('masks', [False, True])
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('T,B,N,W,steps,masked', LONG_RUNS)
def test_conv_long_runs_to_the_last_bit(dev, T, B, N, W, steps, masked, dtype, masks):
    """Small whole numbers and no activation: every product and sum is exact (gradients of weights are below
    2 * 3 * 13000 < 2^24, outputs below 2^8 in bf16), in any order."""
    check_runs(T, B, N, W, steps, masked)
    g = torch.Generator().manual_seed(T)
    whole = lambda most, *shape: torch.randint(-most, most + 1, shape, generator=g)  # noqa: E731
    c = dict(x=whole(3, T, B, N).to(dtype), weight=whole(2, N, W).float(), bias=whole(2, N).float(), state=whole(3, B, W - 1, N).to(dtype),
             dy=whole(2, T, B, N).to(dtype), dstate=whole(2, B, W - 1, N).to(dtype), **masks_of(g, T, B, masks))
    got = run_conv(c, dev, silu=False)
    d = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}
    leaves = {k: d[k].clone().requires_grad_(True) for k in CONV_LEAVES}
    y, state = osel.conv(*[leaves[k] for k in CONV_LEAVES], d['starts'], d['lengths'], False)
    ref = dict(zip(leaves, torch.autograd.grad((y, state), list(leaves.values()), (d['dy'], d['dstate']))), y=y.detach(), after=state.detach())
    for k, v in ref.items():
        assert torch.equal(got[k].double().cpu(), v), k


@pytest.mark.gpu
@pytest.mark.parametrize('masks', [False, True])
@pytest.mark.parametrize('T,B,N,W,steps,masked', LONG_RUNS)
def test_conv_long_runs(dev, T, B, N, W, steps, masked, masks):
    check_conv(conv_case(T, B, N, W, FP32 if W % 2 else BF16, masks), dev)


@pytest.mark.gpu
@pytest.mark.parametrize('silu', [False, True])
def test_conv_padding_has_no_gradient_whatever_the_weights(dev, silu):
    """Infinite and NaN weights: outputs and gradients of padded steps are 0, other channels unchanged."""
    T, B, N, W = 30, 4, 12, 4
    c = conv_case(T, B, N, W, FP32, True)
    want = run_conv(c, dev, silu)
    c['weight'][3], c['weight'][5] = INF, NAN
    got = run_conv(c, dev, silu)
    pad = (torch.arange(T)[:, None] >= c['lengths']).to(dev)
    assert int(pad.sum()) > T and float(got['x'][pad].abs().max()) == 0.0 and float(got['y'][pad].abs().max()) == 0.0
    rest = [n for n in range(N) if n not in (3, 5)]
    for k in ('y', 'x', 'state', 'after'):
        assert torch.equal(got[k][..., rest], want[k][..., rest]), k
    assert torch.equal(got['weight'][rest], want['weight'][rest]) and torch.equal(got['bias'][rest], want['bias'][rest])


# ---------------------------------------------------------------- states of steps -----------

def steps_of(dev, B, N, S, W):
    """name -> (call(state, out, x=...), the state's shape)"""
    from delrec.gated import gated_step
    from delrec.selective import conv_step, selective_step
    c, e = put(scan_case(1, B, N, S, FP32, False), dev), put(conv_case(1, B, N, W, FP32, False), dev)
    ones = torch.ones(N, device=dev)
    x0 = c['x'][0]
    return {
        'h_out': (lambda h, out, x=x0: selective_step(x, c['dt'][0], c['A'], c['B'][0], c['C'][0], h, c['D'], c['g'][0], c['dt_bias'], h_out=out),
                  (B, N, S)),
        'state_out': (lambda s, out, x=x0: conv_step(x, s, e['weight'], e['bias'], state_out=out), (B, W - 1, N)),
        'gated h_out': (lambda h, out, x=x0: gated_step(x, c['dt'][0], c['g'][0], c['x'][0], h, ones, ones, h_out=out)[::2], (B, N)),
    }


@pytest.mark.gpu
@pytest.mark.parametrize('B', [5, 300])
def test_states_written_over_what_a_step_reads_are_refused(dev, B):
    """Views of one buffer a row apart, and a state that the step's input lies in: an error, nothing written."""
    for name, (call, shape) in steps_of(dev, B, 64, 8, 4).items():
        ring = torch.randn(B + 1, *shape[1:], device=dev)
        kept = ring.clone()
        for h, out in ((ring[:-1], ring[1:]), (ring[1:], ring[:-1])):
            with pytest.raises(ValueError, match=name.split()[-1]):
                call(h, out)
        state = torch.randn(shape, device=dev)
        for x in (ring.reshape(-1)[:B * 64].view(B, 64), ring.reshape(-1)[-B * 64:].view(B, 64), ring.reshape(-1)[5:69].expand(B, 64)):
            with pytest.raises(ValueError, match=name.split()[-1]):
                call(state, ring[:B] if x.data_ptr() == ring.data_ptr() or x.stride(0) == 0 else ring[1:], x)
        assert torch.equal(ring, kept)


@pytest.mark.gpu
def test_states_in_memory_of_their_own_are_taken(dev):
    """The state itself, another part of a buffer of states, memory between an input's rows, the place of a
    state that is copied first."""
    B = 5
    for name, (call, shape) in steps_of(dev, B, 64, 8, 4).items():
        first = torch.randn(shape, device=dev)
        want = call(first.clone(), None)
        ring = torch.empty(3, *shape, device=dev)
        ring[1] = first
        for place in (1, 0, 2):
            got = call(ring[1].clone() if place == 1 else ring[1], ring[place])
            assert got[1].data_ptr() == ring[place].data_ptr() and all(torch.equal(a, b) for a, b in zip(got, want)), name
            ring[1] = first
        got = call(ring[1], ring[1])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
        n = first.numel()
        wide = torch.randn(B, 2 * 64 + n, device=dev)
        out, x = wide[2, 64:64 + n].view(shape), wide[:, :64]
        want = call(first, None, x)
        got = call(first, out, x)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
