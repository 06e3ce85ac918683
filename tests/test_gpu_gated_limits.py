"""The gated block's operators at the ends of their ranges: infinite and NaN biases, states and
residuals, gates that take everything, launches past 2^32 threads, inputs changed in place,
tangents, threads. Tolerances as in test_gpu_gated.py unless a test derives its own."""

import pytest
import torch

from oracle import gated as og
from test_gpu_gated import BF16, FP32, NAMES, check_scan, close, norm_case, rnd, run_scan, scan_case  # noqa: F401

INF, NAN = float('inf'), float('nan')


@pytest.fixture
def dev():
    return torch.device('cuda')


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [False, True])
@pytest.mark.parametrize('masks', [False, True])
@pytest.mark.parametrize('dtype', [FP32, BF16])
@pytest.mark.parametrize('T,B,N', [(5, 2, 6), (63, 3, 65), (65, 2, 1), (250, 4, 70), (3001, 2, 70)])
def test_scan_infinite_bias(dev, T, B, N, dtype, masks, checkpoint):
    """A channel that takes every input and one that takes none, at lengths that end inside a block:
    the steps past the end change no state, whatever the bias."""
    c = scan_case(T, B, N, dtype, masks, seed=21)
    c['bias'][-1] = INF
    c['bias'][0] = -INF
    check_scan(c, dev, checkpoint)


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [False, True])
def test_scan_nan_bias_leaves_empty_rows_alone(dev, checkpoint):
    c = scan_case(20, 3, 6, FP32, True, seed=22)
    assert int(c['lengths'][0]) == 0 and int(c['lengths'][1]) == 20
    c['bias'][2] = NAN
    h, last, dz, df, db, dh0 = (t.cpu() for t in run_scan(c, dev, checkpoint))
    assert torch.equal(last[0], c['h0'][0]) and torch.equal(dh0[0], c['dlast'][0])
    assert not h[:, 0].any() and not dz[:, 0].any() and not df[:, 0].any()
    assert torch.isnan(last[1]).tolist() == torch.isnan(db).tolist() == [False, False, True, False, False, False]
