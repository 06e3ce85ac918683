"""Activations kept in 8 bits between the forward and the backward pass.

``pack8`` turns a (..., N) fp32 or bf16 tensor into int8 values and one fp32 scale for each
group of 64 columns of a row (``delrec_pack8``): ``scale = max(amax / 127, 2^-126)``, ``q =
rint(x / scale)``; ``unpack8`` gives the values ``q * scale`` they stand for, at most
0.50002 scale from x (the reciprocal and the product round). That is 1.06 bytes a value. A group that holds an infinity or a NaN comes back
as NaN.

``linear8`` / ``Linear8`` are ``torch.nn.Linear`` with the saved input in that form; the
recurrence and the norms of ``delrec.gated`` keep theirs so with ``checkpoint=True``.
No counterpart in the reference.
"""

import torch
from torch.autograd.function import once_differentiable

from . import _lib

GROUP = _lib.PACK8_GROUP


class Packed8:
    """A tensor in 8 bits: ``q`` (rows, N) int8, ``scale`` (rows, ceil(N / 64)) fp32, and the
    ``shape`` and ``dtype`` it came from."""

    __slots__ = ('q', 'scale', 'shape', 'dtype')

    def __init__(self, q, scale, shape, dtype):
        self.q, self.scale, self.shape, self.dtype = q, scale, shape, dtype


def pack8(x):
    """``Packed8`` of an fp32 or bf16 GPU tensor (..., N); any strides."""
    q, scale = _lib.require_ext().pack8(x)
    return Packed8(q, scale, x.shape, x.dtype)


def unpack8(p):
    """The values that ``p`` stands for, in the shape and type it came from."""
    return _lib.require_ext().unpack8(p.q, p.scale, p.shape, p.dtype)


class Linear8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, p):
        if p is None:
            p = pack8(x)
        ctx.save_for_backward(weight, p.q, p.scale)
        ctx.meta = (p.shape, p.dtype)
        ctx.has_bias = bias is not None
        return torch.nn.functional.linear(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        weight, q, scale = ctx.saved_tensors
        g2 = g.reshape(-1, weight.shape[0])
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = (g2 @ weight).reshape(ctx.meta[0])
        if ctx.needs_input_grad[1]:
            x = unpack8(Packed8(q, scale, *ctx.meta)).reshape(-1, weight.shape[1])
            dw = g2.t() @ x
        if ctx.has_bias and ctx.needs_input_grad[2]:
            db = g2.sum(0)
        return dx, dw, db, None


def linear8(x, weight, bias=None, packed=None):
    """``torch.nn.functional.linear`` that keeps x in 8 bits for the weight's gradient.
    ``packed``: x's ``Packed8``, where what made x has packed it already (``gated.add_norm``) and x has
    not been changed in place since."""
    if not (torch.is_grad_enabled() and weight.requires_grad):
        return torch.nn.functional.linear(x, weight, bias)
    if torch.is_autocast_enabled('cuda'):
        dt = torch.get_autocast_dtype('cuda')
        x, weight, bias = x.to(dt), weight.to(dt), None if bias is None else bias.to(dt)
    if packed is not None and (packed.shape != x.shape or packed.dtype != x.dtype or packed.q.device != x.device):
        raise ValueError(f'packed is {tuple(packed.shape)} {packed.dtype} on {packed.q.device}, x is {tuple(x.shape)} {x.dtype} '
                         f'on {x.device}')
    return Linear8Fn.apply(x, weight, bias, packed)


class Linear8(torch.nn.Linear):
    """``torch.nn.Linear`` with its saved input in 8 bits (same parameters and state dict)."""

    def forward(self, x):
        return linear8(x, self.weight, self.bias)
