"""CPU checks of the gated-recurrence block: refusals, argument structs and statuses of the C ABI,
the model's parameters, and the 64-bit oracle against differences. No kernel is launched."""

import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from oracle import gated as og

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include', 'delrec.h')


def test_cpu_tensors_are_refused():
    from delrec import checkpoint8, gated
    z, w = torch.zeros(4, 2, 8), torch.ones(8)
    for call in (lambda: gated.gated_scan(z, z), lambda: gated.rms_norm(z, w),
                 lambda: gated.norm_gate_residual(z, z, z, w, w), lambda: checkpoint8.pack8(z),
                 lambda: gated.gated_step(z[0], z[0], z[0], z[0], z[0], w, w)):
        with pytest.raises(RuntimeError, match='GPU'):
            call()


def test_struct_layouts_match_ctypes():
    from delrec import _lib
    classes = {'delrec_rows': _lib.Rows, 'delrec_packed8': _lib.Packed8,
               'delrec_gated_scan_fwd_args': _lib.GatedScanFwdArgs, 'delrec_gated_scan_bwd_args': _lib.GatedScanBwdArgs,
               'delrec_norm_gate_fwd_args': _lib.NormGateFwdArgs, 'delrec_norm_gate_bwd_args': _lib.NormGateBwdArgs,
               'delrec_gated_step_args': _lib.GatedStepArgs, 'delrec_pack8_args': _lib.Pack8Args}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', 'int main(void) {']
    for name, cls in classes.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, 'probe.c'), os.path.join(tmp, 'probe')
        with open(src, 'w') as f:
            f.write('\n'.join(lines + ['  return 0;', '}']))
        subprocess.run(['gcc', '-std=c11', src, '-o', exe], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    c = {' '.join(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for name, cls in classes.items():
        assert c[f'{name} size'] == ctypes.sizeof(cls), name
        for f, _ in cls._fields_:
            assert c[f'{name} {f}'] == getattr(cls, f).offset, f'{name}.{f}'


def test_abi_refuses_what_it_cannot_run():
    """Statuses that need no GPU: missing pointers, sizes, workspaces, types."""
    from delrec import _lib
    lib = _lib.load()
    one = ctypes.c_void_p(4096)          # never read: every call here is refused first
    rows = _lib.Rows(4096, 8, 8)

    def status(name, args):
        return getattr(lib, name)(ctypes.byref(args), None)
    for name in ('delrec_gated_scan_fwd', 'delrec_gated_scan_bwd', 'delrec_gated_step', 'delrec_norm_gate_fwd',
                 'delrec_norm_gate_bwd', 'delrec_pack8', 'delrec_unpack8'):
        assert getattr(lib, name)(None, None) == 1, name
    fwd = dict(T=4, B=2, N=8, z=rows, f=rows, h=rows, h_last=one)
    assert status('delrec_gated_scan_fwd', _lib.GatedScanFwdArgs(**{**fwd, 'T': 0})) == 1
    assert status('delrec_gated_scan_fwd', _lib.GatedScanFwdArgs(**{**fwd, 'f': _lib.Rows()})) == 1
    assert status('delrec_gated_scan_fwd', _lib.GatedScanFwdArgs(**{**fwd, 'z8': _lib.Packed8(4096, 4096)})) == 1
    long = dict(fwd, T=100000)           # few channels: ranges, and room for their maps
    assert status('delrec_gated_scan_fwd', _lib.GatedScanFwdArgs(**long)) == 3
    bwd = dict(T=4, B=2, N=8, z=rows, f=rows, states=one, dh=rows, dz=rows, df=rows)
    assert status('delrec_gated_scan_bwd', _lib.GatedScanBwdArgs(**bwd)) == 3
    assert status('delrec_gated_scan_bwd', _lib.GatedScanBwdArgs(**{**bwd, 'states': None})) == 1
    norm = dict(R0=3, R1=1, N=8, o=rows, g=rows, x=rows, w=one, scale=one, x_out=one, eps=1e-6)
    assert status('delrec_norm_gate_fwd', _lib.NormGateFwdArgs(**{**norm, 'x_bf16': 1})) == 2
    assert status('delrec_norm_gate_fwd', _lib.NormGateFwdArgs(**{**norm, 'w2': one})) == 1
    assert status('delrec_norm_gate_fwd', _lib.NormGateFwdArgs(**{**norm, 'N': 1})) == 1
    assert status('delrec_norm_gate_fwd', _lib.NormGateFwdArgs(**{**norm, 'R0': 1 << 30, 'R1': 1 << 30})) == 1
    assert status('delrec_pack8', _lib.Pack8Args(R0=3, R1=1, N=8, x=rows)) == 1
    size = ctypes.c_size_t(0)
    assert lib.delrec_query_workspace(_lib.WS_GATED_FWD, 100000, 2, 8, 1, 0, ctypes.byref(size)) == 0 and size.value > 0
    assert lib.delrec_query_workspace(_lib.WS_GATED_FWD, 64, 2, 8, 1, 0, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.delrec_query_workspace(_lib.WS_NORM_GATE_BWD, 100, 1, 512, 1, 0, ctypes.byref(size)) == 0
    assert size.value >= 3 * 512 * 4


def test_model_parameters_and_widths():
    from configs.perf_MEM import Config
    from delrec.networks import RNN_gated
    cfg = Config()
    cfg.hidden_layers = [32, 32]
    names = set(RNN_gated(cfg).state_dict())
    cfg.checkpoint8 = True
    assert names == set(RNN_gated(cfg).state_dict())       # the 8 bits change no parameter
    assert {'embed.weight', 'norm_weight', 'blocks.1.proj.weight', 'blocks.0.gate_bias', 'readout.weight'} <= names
    cfg.hidden_layers = [32, 48]
    with pytest.raises(ValueError):
        RNN_gated(cfg)


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    z, f, dh = (torch.randn(70, 2, 3, generator=g, dtype=torch.float64) for _ in range(3))
    h0, dlast = (torch.randn(2, 3, generator=g, dtype=torch.float64) for _ in range(2))
    bias = torch.rand(3, generator=g, dtype=torch.float64)
    starts = torch.rand(70, 2, generator=g) < 0.05
    lengths = torch.tensor([70, 31])
    got = og.scan_grads(z, f, bias, h0, starts, lengths, dh, dlast)[2:]

    def loss(*a):
        h, last, _ = og.scan(*a, starts, lengths)
        return float((h * dh).sum() + (last * dlast).sum())
    base = (z, f, bias, h0)
    for k in range(4):
        way = torch.randn(base[k].shape, generator=g, dtype=torch.float64)
        hi, lo = ([t + s * way if i == k else t for i, t in enumerate(base)] for s in (1e-5, -1e-5))
        diff = (loss(*hi) - loss(*lo)) / 2e-5
        assert abs(float((got[k] * way).sum()) - diff) < 1e-7 * (1 + float((got[k] * way).abs().sum()))


def test_oracle_8_bit_gradients_at_exact_values_are_the_gradients():
    """On values that 8 bits hold exactly, the 8-bit forms of the gradients are the ordinary ones."""
    g = torch.Generator().manual_seed(2)

    def grid(*shape):
        v = torch.randint(-127, 128, shape, generator=g).double()
        v[..., ::64] = 127
        return v / 64
    z, f = grid(70, 2, 66), grid(70, 2, 66)
    assert float((og.round8(z)[0] - z).abs().max()) < 1e-6
    dh, dlast = torch.randn(70, 2, 66, generator=g).double(), torch.randn(2, 66, generator=g).double()
    a = og.scan_grads(z, f, None, None, None, None, dh, dlast)
    b = og.scan_grads(z, f, None, None, None, None, dh, dlast, checkpoint=True)
    for x, y in zip(a, b):
        torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-5)
    o, gg, x = grid(9, 66), grid(9, 66), grid(9, 66)
    w, s, w2 = (torch.rand(66, generator=g).double() + 0.5 for _ in range(3))
    leaves = [t.clone().requires_grad_(True) for t in (o, gg, x, w, s, w2)]
    cot = (torch.randn(9, 66, generator=g).double(), torch.randn(9, 66, generator=g).double())
    want = torch.autograd.grad(og.norm_gate(*leaves, 1e-6), leaves, cot)
    for p, q in zip(og.norm_gate_grads8(o, gg, x, w, s, w2, 1e-6, *cot), want):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-5)


def test_abi_refuses_8_bits_of_only_some_inputs():
    """o, g and x of a block are kept in 8 bits together, x by itself where there is no block: any
    other mix would have a kernel go through a pointer that was not given."""
    from delrec import _lib
    lib = _lib.load()
    one, rows, packed = ctypes.c_void_p(4096), _lib.Rows(4096, 8, 8), _lib.Packed8(4096, 4096)
    fwd = dict(R0=3, R1=1, N=8, o=rows, g=rows, x=rows, w=one, scale=one, w2=one, x_out=one, u=one, stats=one, eps=1e-6)
    bwd = dict(R0=3, R1=1, N=8, w=one, scale=one, w2=one, stats=one, du=rows, d_o=rows, dg=rows, dx=rows, dw=one,
               dscale=one, dw2=one)                      # no workspace: what passes the checks stops there
    for given in range(8):
        eight = {k: packed for i, k in enumerate(('o8', 'g8', 'x8')) if given >> i & 1}
        plain = {k[0]: rows for k in ('o8', 'g8', 'x8') if k not in eight}
        if given not in (0, 7):
            assert lib.delrec_norm_gate_fwd(ctypes.byref(_lib.NormGateFwdArgs(**fwd, **eight)), None) == 1, given
        want = 3 if given in (0, 7) else 1
        for args in ({**bwd, **plain, **eight}, {**bwd, 'o': rows, 'g': rows, 'x': rows, **eight}):
            assert lib.delrec_norm_gate_bwd(ctypes.byref(_lib.NormGateBwdArgs(**args)), None) == want, (given, args)
    alone = dict(R0=3, R1=1, N=8, x=rows, w2=one, stats=one, du=rows, dx=rows, dw2=one)
    assert lib.delrec_norm_gate_bwd(ctypes.byref(_lib.NormGateBwdArgs(**alone, x8=packed)), None) == 3
    assert lib.delrec_norm_gate_bwd(ctypes.byref(_lib.NormGateBwdArgs(**alone, g8=packed)), None) == 1
    # N = 3: the kernels for rows of any width have the same contract
    assert lib.delrec_norm_gate_bwd(ctypes.byref(_lib.NormGateBwdArgs(**{**bwd, 'N': 3}, o=rows, g=rows, x8=packed)), None) == 1


def test_abi_refuses_columns_past_its_counters():
    """Column counts whose sums of three, or whose last stride, would pass the kernels' integers."""
    from delrec import _lib
    lib = _lib.load()
    one, rows = ctypes.c_void_p(4096), _lib.Rows(4096, 8, 8)
    for n in (2 ** 31 - 1, 2 ** 31 - 1023):
        assert lib.delrec_pack8(ctypes.byref(_lib.Pack8Args(R0=1, R1=1, N=n, x=rows, p=_lib.Packed8(4096, 4096))), None) == 1
        assert lib.delrec_gated_scan_fwd(ctypes.byref(_lib.GatedScanFwdArgs(T=1, B=1, N=n, z=rows, f=rows, h=rows, h_last=one)), None) == 1
    bwd = dict(R0=1, R1=1, x=rows, w2=one, stats=one, du=rows, dx=rows, dw2=one)
    assert lib.delrec_norm_gate_bwd(ctypes.byref(_lib.NormGateBwdArgs(N=2 ** 30 + 1, **bwd)), None) == 1
    assert lib.delrec_norm_gate_bwd(ctypes.byref(_lib.NormGateBwdArgs(N=2 ** 30, **bwd)), None) == 3      # no workspace


def test_abi_refuses_steps_past_its_counters():
    from delrec import _lib
    lib = _lib.load()
    one, rows = ctypes.c_void_p(4096), _lib.Rows(4096, 1, 1)
    for t in (2 ** 31 - 1, 2 ** 31 - 128 * 64):
        assert lib.delrec_gated_scan_fwd(ctypes.byref(_lib.GatedScanFwdArgs(T=t, B=1, N=1, z=rows, f=rows, h=rows, h_last=one)), None) == 1
        args = _lib.GatedScanBwdArgs(T=t, B=1, N=1, z=rows, f=rows, states=one, dh=rows, dz=rows, df=rows)
        assert lib.delrec_gated_scan_bwd(ctypes.byref(args), None) == 1
    args = _lib.GatedScanFwdArgs(T=2 ** 31 - 128 * 64 - 1, B=1, N=1, z=rows, f=rows, h=rows, h_last=one)
    assert lib.delrec_gated_scan_fwd(ctypes.byref(args), None) == 3      # no workspace
    size = ctypes.c_size_t(0)
    for kind, t, b, n in ((_lib.WS_GATED_FWD, 2 ** 31 - 1, 1, 1), (_lib.WS_GATED_BWD, 1, 1, 2 ** 31 - 1),
                          (_lib.WS_NORM_GATE_BWD, 1, 1, 2 ** 31 - 1), (_lib.WS_NORM_GATE_BWD, 4, 1, 1)):
        assert lib.delrec_query_workspace(kind, t, b, n, 1, 0, ctypes.byref(size)) == 1


@pytest.mark.parametrize('field,value', [('use_batch_norm', True), ('feedforward_dropout_rate', 0.1)])
def test_model_refuses_what_it_does_not_do(field, value):
    from configs.perf_MEM import Config
    from delrec.networks import RNN_gated
    cfg = Config()
    RNN_gated(cfg)
    setattr(cfg, field, value)
    with pytest.raises(NotImplementedError, match=field):
        RNN_gated(cfg)


def test_model_takes_a_config_of_its_own_four_fields():
    from types import SimpleNamespace
    from delrec.networks import RNN_gated
    RNN_gated(SimpleNamespace(input_size=3, hidden_layers=[32, 32], output_size=2, bias=False))
