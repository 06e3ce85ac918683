"""The selective block's operators where they were wrong, or untested, before: last bits of a norm's factor.
Tolerances as in test_gpu_selective.py unless a test derives its own."""

import pytest
import torch

from test_gpu_selective import BF16, FP32, add_case

INF, NAN = float('inf'), float('nan')


@pytest.fixture
def dev():
    return torch.device('cuda')


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
