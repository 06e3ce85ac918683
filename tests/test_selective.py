"""The selective block on the CPU: the 64-bit definitions against differences and each other, argument
structs, refusals, the model's parameters. No kernel is launched."""

import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from oracle import selective as osel

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, 'include', 'delrec.h')
NAMES = ('x', 'dt', 'A', 'B', 'C', 'D', 'g', 'dt_bias', 'h0')


def scan_inputs(T, R, N, S, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    c = dict(x=r(T, R, N), dt=r(T, R, N), A=-torch.rand(N, S, generator=g, dtype=torch.float64) * 3, B=r(T, R, S), C=r(T, R, S),
             D=r(N), g=r(T, R, N), dt_bias=r(N), h0=r(R, N, S))
    starts = torch.rand(T, R, generator=g) < 0.2
    lengths = torch.randint(0, T + 1, (R,), generator=g)
    lengths[0] = T
    return c, starts, lengths, r(T, R, N), r(R, N, S)


@pytest.mark.parametrize('masks', [False, True])
@pytest.mark.parametrize('gate', [False, True])
def test_scan_gradients_formula_autograd_and_differences(masks, gate):
    c, starts, lengths, dy, dlast = scan_inputs(9, 3, 4, 3)
    if not masks:
        starts = lengths = None
    if not gate:
        c['g'] = None
    leaves = {k: v.clone().requires_grad_(True) for k, v in c.items() if v is not None}
    args = [leaves.get(k) for k in NAMES]
    y, last = osel.scan(*args, starts, lengths)
    auto = dict(zip(leaves, torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast))))
    formula, mass = osel.scan_grads(*[c[k] for k in NAMES], starts, lengths, dy, dlast)
    assert set(formula) == set(auto)
    for k in auto:
        torch.testing.assert_close(formula[k], auto[k], rtol=1e-10, atol=1e-10)
    for k, m in mass.items():
        assert m >= float(formula[k].abs().max())

    def loss(d):
        yy, ll = osel.scan(*[d.get(k) for k in NAMES], starts, lengths)
        return float((yy * dy).sum() + (ll * dlast).sum())
    gen = torch.Generator().manual_seed(3)
    for k in auto:
        way = torch.randn(c[k].shape, generator=gen, dtype=torch.float64)
        e = 1e-5
        up, down = dict(c), dict(c)
        up[k], down[k] = c[k] + e * way, c[k] - e * way
        # central differences: e^2 times third derivatives, and 1e-16 / e of the loss
        assert abs((loss(up) - loss(down)) / (2 * e) - float((auto[k] * way).sum())) < 1e-6 * max(1.0, float((auto[k] * way).abs().sum())), k


def test_conv_is_a_convolution_cut_at_starts():
    g = torch.Generator().manual_seed(1)
    T, R, N, W = 11, 2, 3, 4
    x = torch.randn(T, R, N, generator=g, dtype=torch.float64)
    w = torch.randn(N, W, generator=g, dtype=torch.float64)
    y, state = osel.conv(x, w, silu=False)
    ref = torch.nn.functional.conv1d(torch.nn.functional.pad(x.permute(1, 2, 0), (W - 1, 0)), w[:, None], groups=N)
    torch.testing.assert_close(y, ref.permute(2, 0, 1))
    assert torch.equal(state, x[-(W - 1):].transpose(0, 1))
    # two parts joined by the state, and a start that makes the second one independent
    a, mid = osel.conv(x[:5], w, silu=False)
    b, _ = osel.conv(x[5:], w, None, mid, silu=False)
    torch.testing.assert_close(torch.cat([a, b]), y)
    starts = torch.zeros(T, R, dtype=torch.bool)
    starts[5] = True
    cut, _ = osel.conv(x, w, starts=starts, silu=False)
    torch.testing.assert_close(cut, torch.cat([a, osel.conv(x[5:], w, silu=False)[0]]))


_CLASSES = {'delrec_add_norm_fwd_args': 'AddNormFwdArgs', 'delrec_add_norm_bwd_args': 'AddNormBwdArgs',
            'delrec_causal_conv_fwd_args': 'CausalConvFwdArgs', 'delrec_causal_conv_bwd_args': 'CausalConvBwdArgs',
            'delrec_selective_scan_fwd_args': 'SelectiveScanFwdArgs', 'delrec_selective_scan_bwd_args': 'SelectiveScanBwdArgs',
            'delrec_selective_step_args': 'SelectiveStepArgs'}


def test_struct_layout_matches_ctypes():
    from delrec import _lib
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', 'int main(void) {']
    for st, cls in _CLASSES.items():
        lines.append(f'  printf("{st} size %zu\\n", sizeof({st}));')
        for f, _ in getattr(_lib, cls)._fields_:
            lines.append(f'  printf("{st} {f} %zu\\n", offsetof({st}, {f}));')
    lines += ['  return 0;', '}']
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, 'p.c'), os.path.join(tmp, 'p')
        open(src, 'w').write('\n'.join(lines))
        subprocess.run(['gcc', '-std=c11', src, '-o', exe], check=True)
        got = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    c = {' '.join(ln.split()[:2]): int(ln.split()[2]) for ln in got.splitlines()}
    for st, name in _CLASSES.items():
        cls = getattr(_lib, name)
        assert c[f'{st} size'] == ctypes.sizeof(cls), st
        for f, _ in cls._fields_:
            assert c[f'{st} {f}'] == getattr(cls, f).offset, f'{st}.{f}'


def test_abi_refuses_before_the_device():
    from delrec import _lib
    lib = _lib.load()
    size = ctypes.c_size_t(0)
    query = lambda kind, T, B, N, L: lib.delrec_query_workspace(kind, T, B, N, L, 0, ctypes.byref(size))  # noqa: E731
    for kind, L in ((_lib.WS_ADD_NORM_BWD, 1), (_lib.WS_CAUSAL_CONV_BWD, 4), (_lib.WS_SELECTIVE_FWD, 16), (_lib.WS_SELECTIVE_BWD, 16)):
        assert query(kind, 64, 3, 100, L) == 0
        assert query(kind, 0, 3, 100, L) == 1
    assert query(_lib.WS_SELECTIVE_BWD, 64, 3, 100, 65) == 1 and query(_lib.WS_SELECTIVE_BWD, 64, 3, 100, 0) == 1
    assert query(_lib.WS_CAUSAL_CONV_BWD, 64, 3, 100, 9) == 1 and query(_lib.WS_CAUSAL_CONV_BWD, 64, 3, 100, 1) == 1
    assert query(_lib.WS_SELECTIVE_BWD, 2 ** 31 - 1, 1, 1, 16) == 1
    for name, cls in (('delrec_add_norm_fwd', _lib.AddNormFwdArgs), ('delrec_add_norm_bwd', _lib.AddNormBwdArgs),
                      ('delrec_causal_conv_fwd', _lib.CausalConvFwdArgs), ('delrec_causal_conv_bwd', _lib.CausalConvBwdArgs),
                      ('delrec_selective_scan_fwd', _lib.SelectiveScanFwdArgs), ('delrec_selective_scan_bwd', _lib.SelectiveScanBwdArgs),
                      ('delrec_selective_step', _lib.SelectiveStepArgs)):
        fn = getattr(lib, name)
        assert fn(None, None) == 1, name
        args = cls()
        assert fn(ctypes.byref(args), None) == 1, name          # no sizes
        for f, v in (('T', 4), ('R0', 4), ('R1', 1), ('B', 2), ('N', 8), ('S', 4), ('W', 4)):
            if any(f == k for k, _ in cls._fields_):
                setattr(args, f, v)
        assert fn(ctypes.byref(args), None) == 1, name          # no tensors


def test_cpu_tensors_are_refused():
    from delrec.gated import add_norm
    from delrec.selective import causal_conv, conv_step, selective_scan, selective_step
    x, low, A = torch.zeros(3, 2, 4), torch.zeros(3, 2, 5), torch.zeros(4, 5)
    for call in (lambda: causal_conv(x, torch.zeros(4, 4)), lambda: conv_step(x[0], torch.zeros(2, 3, 4), torch.zeros(4, 4)),
                 lambda: selective_scan(x, x, A, low, low), lambda: selective_step(x[0], x[0], A, low[0], low[0], torch.zeros(2, 4, 5)),
                 lambda: add_norm(x, x, torch.ones(4))):
        with pytest.raises(RuntimeError, match='on the GPU'):
            call()


class _Config:
    input_size, hidden_layers, output_size, bias = 8, [32, 32], 4, False


def test_model_parameters_and_refusals():
    from delrec.networks import RNN_selective
    torch.manual_seed(0)
    m = RNN_selective(_Config)
    b = m.blocks[0]
    assert b.inner == 64 and b.A_log.shape == (64, 16) and b.conv_weight.shape == (64, 4) and len(m.blocks) == 2
    step = torch.nn.functional.softplus(b.dt_bias)
    assert float(step.min()) > 0.9e-3 and float(step.max()) < 1.1e-1

    class Other(_Config):
        state_size, conv_width, checkpoint8 = 8, 3, True
    m = RNN_selective(Other)
    assert m.blocks[0].A_log.shape == (64, 8) and m.blocks[0].conv_weight.shape == (64, 3) and m.blocks[0].checkpoint
    for bad in (dict(hidden_layers=[32, 64]), dict(feedforward_dropout_rate=0.1), dict(use_batch_norm=True)):
        with pytest.raises((ValueError, NotImplementedError)):
            RNN_selective(type('Bad', (_Config,), bad))
