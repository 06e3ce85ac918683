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
from .kernels._common import require_device

GROUP = _lib.PACK8_GROUP
DTYPES = (torch.float32, torch.bfloat16)


def rows_of(t):
    """``delrec_rows`` of a (..., N) tensor whose last axis is contiguous and whose leading
    axes are at most two (``rows_form`` makes it so)."""
    if t is None:
        return _lib.Rows()
    if t.dim() == 3:
        return _lib.Rows(t.data_ptr(), t.stride(0), t.stride(1))
    return _lib.Rows(t.data_ptr(), t.stride(0), 0)


def rows_form(t):
    """``t`` as a (R0, R1, N) or (R, N) view whose last axis is contiguous; a copy only where
    the tensor has no such view."""
    if t.dim() == 1:
        t = t.unsqueeze(0)
    elif t.dim() > 3:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def row_counts(t):
    return (t.shape[0], t.shape[1]) if t.dim() == 3 else (t.shape[0], 1)


def empty8(rows, N, device):
    """Storage for ``rows`` rows of N: (int8 values, fp32 scales)."""
    return (torch.empty(rows, N, dtype=torch.int8, device=device),
            torch.empty(rows, (N + GROUP - 1) // GROUP, dtype=torch.float32, device=device))


def packed_of(q, scale):
    return _lib.Packed8() if q is None else _lib.Packed8(q.data_ptr(), scale.data_ptr())


class Packed8:
    """A tensor in 8 bits: ``q`` (rows, N) int8, ``scale`` (rows, ceil(N / 64)) fp32, and the
    ``shape`` and ``dtype`` it came from."""

    __slots__ = ('q', 'scale', 'shape', 'dtype')

    def __init__(self, q, scale, shape, dtype):
        self.q, self.scale, self.shape, self.dtype = q, scale, shape, dtype


def pack8(x):
    """``Packed8`` of an fp32 or bf16 GPU tensor (..., N); any strides."""
    require_device(x)
    if x.dtype not in DTYPES:
        raise ValueError(f'pack8 takes fp32 or bf16, got {x.dtype}')
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f'pack8 takes a (..., N) tensor with N > 0, got {tuple(x.shape)}')
    v = rows_form(x.detach())
    R0, R1 = row_counts(v)
    N = v.shape[-1]
    q, scale = empty8(R0 * R1, N, x.device)
    if R0 * R1:
        args = _lib.Pack8Args(R0=R0, R1=R1, N=N, bf16=int(v.dtype == torch.bfloat16), x=rows_of(v), p=packed_of(q, scale))
        with torch.cuda.device(x.device):
            _lib.call('delrec_pack8', args, _lib.stream_of(x))
    return Packed8(q, scale, x.shape, x.dtype)


def unpack8(p):
    """The values that ``p`` stands for, in the shape and type it came from."""
    require_device(p.q)
    out = torch.empty(p.shape, dtype=p.dtype, device=p.q.device)
    rows, N = p.q.shape
    if rows:
        v = out.view(rows, N)
        args = _lib.Pack8Args(R0=rows, R1=1, N=N, bf16=int(p.dtype == torch.bfloat16), x=rows_of(v),
                              p=packed_of(p.q, p.scale))
        with torch.cuda.device(out.device):
            _lib.call('delrec_unpack8', args, _lib.stream_of(out))
    return out


class Linear8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
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
        return dx, dw, db


def linear8(x, weight, bias=None):
    """``torch.nn.functional.linear`` that keeps x in 8 bits for the weight's gradient."""
    require_device(x)
    if not (torch.is_grad_enabled() and weight.requires_grad):
        return torch.nn.functional.linear(x, weight, bias)
    if torch.is_autocast_enabled('cuda'):
        dt = torch.get_autocast_dtype('cuda')
        x, weight, bias = x.to(dt), weight.to(dt), None if bias is None else bias.to(dt)
    return Linear8Fn.apply(x, weight, bias)


class Linear8(torch.nn.Linear):
    """``torch.nn.Linear`` with its saved input in 8 bits (same parameters and state dict)."""

    def forward(self, x):
        return linear8(x, self.weight, self.bias)
