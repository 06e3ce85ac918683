"""The selective block's operators at the limits of their inputs and of torch's machinery: infinite rates
and biases, values of very different sizes, tangents, opposites in memory, captured backward passes,
threads. Tolerances as in test_gpu_selective.py unless a test derives its own."""

import pytest
import torch

from oracle import selective as osel
from test_gpu_selective import (BF16, CONV_LEAVES, FP32, LEAVES, SCAN_TOL, add_case, check_scan, close, conv_case, put,  # noqa: F401
                                run_scan, scan_case)

INF, NAN = float('inf'), float('nan')


@pytest.fixture
def dev():
    return torch.device('cuda')


@pytest.mark.gpu
@pytest.mark.parametrize('S', [4, 16, 40])
@pytest.mark.parametrize('T', [5, 16, 70, 300])
def test_channels_that_stand_still(dev, T, S):
    """A step size of 0 (a bias of -inf) leaves the state as it is, whatever comes in."""
    c = scan_case(T, 3, 20, S, FP32, True)
    c['dt_bias'][3] = c['dt_bias'][11] = -INF
    got = check_scan(c, dev)
    rows = (~c['starts']).all(0) | (c['lengths'] == 0)
    for n in (3, 11):
        assert torch.equal(got['last'].cpu()[rows, n], c['h0'][rows, n])
        assert float(got['dt'][:, :, n].abs().max()) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize('S', [4, 40])
@pytest.mark.parametrize('T', [5, 70, 300])
def test_states_that_forget_at_once(dev, T, S):
    """An infinite rate keeps nothing from one step to the next, and padding keeps the state."""
    c = scan_case(T, 4, 20, S, FP32, True)
    c['A'][:, 0] = -INF
    c['A'][5] = -INF
    got = run_scan(c, dev)
    assert all(torch.isfinite(v).all() for v in got.values())
    d = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}
    y, last = osel.scan(*[d[k] for k in LEAVES], d['starts'], d['lengths'])
    close(got['y'], y, SCAN_TOL, 'y')
    close(got['last'], last, SCAN_TOL, 'last')
    # a rate of -1e30 does the same and has the formula's gradients
    c['A'] = c['A'].clamp(min=-1e30)
    for k, v in run_scan(c, dev).items():
        if k not in ('A', 'dt', 'dt_bias'):
            torch.testing.assert_close(got[k], v, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize('S', [8, 16])
def test_each_state_to_its_own_size(dev, S):
    """Without inputs a state is a product of decays. A decay's exponent is off by 2^-23 of its own and
    by the step size's 4e-7, over its steps at most 5e-7 of the whole exponent, 60 here: 3e-5."""
    T, B, N = 60, 2, 33
    c = scan_case(T, B, N, S, FP32, False)
    c['B'].zero_()
    c['dt'] = torch.rand(T, B, N) * 2 - 1
    c['dt_bias'].zero_()
    c['A'] = -torch.linspace(1e-4, 0.75, N * S).reshape(N, S)
    got = run_scan(c, dev)
    e = osel.softplus(c['dt'].double()).sum(0)[..., None] * c['A'].double()
    assert float(e.min()) > -62
    ref = c['h0'].double() * torch.exp(e)
    assert ((got['last'].double().cpu() - ref).abs() <= 3.1e-5 * ref.abs()).all()
    carry = c['dlast'].double() * torch.exp(e)
    c['dy'].zero_()
    got = run_scan(c, dev)
    assert ((got['h0'].double().cpu() - carry).abs() <= 3.1e-5 * carry.abs()).all()


def _calls(dev):
    from delrec.gated import add_norm
    from delrec.selective import causal_conv, conv_step, selective_scan, selective_step
    c, e, n = put(scan_case(6, 2, 10, 4, FP32, False), dev), put(conv_case(6, 2, 10, 4, FP32, False), dev), put(add_case((4, 2, 10), FP32, FP32), dev)
    s = [c[k] for k in LEAVES]
    return {
        'selective_scan': (selective_scan, s),
        'causal_conv': (causal_conv, [e[k] for k in CONV_LEAVES]),
        'add_norm': (add_norm, [n['x'], n['y'], n['w']]),
        'conv_step': (conv_step, [e['x'][0], e['state'], e['weight'], e['bias']]),
        'selective_step': (selective_step, [s[0][0], s[1][0], s[2], s[3][0], s[4][0], s[8], s[5], s[6][0], s[7]]),
    }


@pytest.mark.gpu
@pytest.mark.parametrize('grad', [False, True])
def test_forward_mode_tangents_are_refused(dev, grad):
    import torch.autograd.forward_ad as fw
    with torch.set_grad_enabled(grad), fw.dual_level():
        for call, args in _calls(dev).values():
            call(*args)
            for i, a in enumerate(args):
                dual = fw.make_dual(a.clone(), torch.ones_like(a))
                with pytest.raises(RuntimeError, match='forward-mode'):
                    call(*args[:i], dual, *args[i + 1:])


@pytest.mark.gpu
def test_imaginary_parts_of_conjugated_tensors(dev):
    """Real views whose memory holds the opposite of their values, as every input and gradient."""
    def opposite(t):
        view = torch.view_as_complex(torch.stack([t, -t], -1).contiguous()).conj().imag
        assert view.is_neg()
        return view
    for name, (call, args) in _calls(dev).items():
        want = call(*args)
        for a, b in zip(want, call(*[opposite(a) for a in args])):
            assert torch.equal(a, b), name
        if 'step' in name:
            continue
        g = [torch.randn_like(t) for t in want]
        grads = []
        for turn in (lambda t: t, opposite):
            leaves = [turn(a).detach().requires_grad_(True) for a in args]
            grads.append(torch.autograd.grad(call(*leaves), leaves, [turn(t) for t in g]))
        for a, b in zip(*grads):
            assert torch.equal(a, b), name


@pytest.mark.gpu
def test_captured_backward_is_refused(dev):
    """The nodes, called by themselves while the stream is capturing: an error, nothing launched, and the
    capture, the graph and the nodes stay usable."""
    calls = _calls(dev)
    outs = []
    for name in ('selective_scan', 'causal_conv', 'add_norm'):
        call, args = calls[name]
        leaves = [a.detach().requires_grad_(True) for a in args]
        outs.append((leaves, call(*leaves)))
    out = torch.ones(3, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out.mul_(2.0)
        for _, res in outs:
            with pytest.raises(RuntimeError, match='captured'):
                res[0].grad_fn(*res)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert out.tolist() == [8.0] * 3
    for leaves, res in outs:
        g = [torch.ones_like(t) for t in res]
        a = torch.autograd.grad(res, leaves, g, retain_graph=True)
        for x, y in zip(a, torch.autograd.grad(res, leaves, g)):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_backward_passes_of_two_threads_through_one_graph(dev):
    """Each either gives the graph's gradients or raises that they are gone, as torch's own nodes."""
    import threading
    from delrec.gated import add_norm
    from delrec.selective import causal_conv, selective_scan
    c = put(scan_case(30, 2, 12, 4, FP32, False), dev)
    w, nw = torch.randn(12, 4, device=dev), torch.ones(12, device=dev)
    x = c['x'].clone().requires_grad_(True)

    def forward():
        v, _ = causal_conv(x, w)
        y, _ = selective_scan(v, c['dt'], c['A'], c['B'], c['C'], c['D'], c['g'])
        return add_norm(x, y, nw)[1].sum()
    (want,) = torch.autograd.grad(forward(), x)
    for _ in range(10):
        loss = forward()
        done, start = [], threading.Barrier(4)

        def work():
            start.wait()
            try:
                done.append(torch.autograd.grad(loss, x)[0])
            except RuntimeError as e:
                assert 'second time' in str(e)
                done.append(None)
        threads = [threading.Thread(target=work) for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert len(done) == 4 and all(g is None or torch.equal(g, want) for g in done)


@pytest.mark.gpu
def test_linear8_with_what_the_norm_packed(dev):
    """The same gradients as with a pass of its own, kept on the device and on the host; under autocast."""
    from delrec.checkpoint8 import linear8
    from delrec.gated import add_norm
    n = put(add_case((6, 5, 70), BF16, FP32), dev)
    w, b = torch.randn(33, 70, device=dev, requires_grad=True), torch.randn(33, device=dev, requires_grad=True)
    _, u, p = add_norm(n['x'], n['y'], n['w'], pack=True)
    u = u.requires_grad_(True)

    def grads(packed, host=False):
        with torch.autocast('cuda', BF16):
            if host:
                with torch.autograd.graph.save_on_cpu():
                    y = linear8(u, w, b, packed=packed)
            else:
                y = linear8(u, w, b, packed=packed)
            return torch.autograd.grad(y.float().square().sum(), (u, w, b))
    want = grads(None)
    for got in (grads(p), grads(p, True)):
        assert all(torch.equal(a, c) for a, c in zip(got, want))
