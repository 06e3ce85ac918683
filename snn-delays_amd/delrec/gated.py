"""Gated linear recurrence, and the norms, gate and residual of the block around it, over the
same time-major (T, B, N) sequences as the delayed-LIF layers.

    gated_scan           h_t = h_{t-1} + k_t (z_t - h_{t-1}), k_t = sigmoid(-(f_t + bias))
    norm_gate_residual   x' = x + scale * rms(o) * weight * silu(g), u = rms(x') * next_weight
    rms_norm             u = rms(x) * weight
    gated_step           one time step of both, for streaming input
    GatedBlock           the residual block they make with its Linear

where ``rms(v) = v / sqrt(mean(v^2) + eps)`` over the last axis. The recurrence is the leaky
integrator of ``LIFNode(decay_input=True)`` without its threshold, with a leak that each step's
input sets. Activations are fp32 or bf16; states, gates, norms and sums are in 32 bits. With
``checkpoint=True`` an operator keeps what its backward pass reads in 8 bits
(``delrec.checkpoint8``). No counterpart in the reference.
"""

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .checkpoint8 import DTYPES, Linear8, empty8, packed_of, row_counts, rows_form, rows_of
from .kernels._common import require_device

BLOCK = _lib.GATED_BLOCK


def _bf16(t):
    return int(t.dtype == torch.bfloat16)


def _vector(v, n, what, device):
    """``v`` as a contiguous fp32 (n,) vector on ``device`` (None stays None)."""
    if v is None:
        return None
    if tuple(v.shape) != (n,):
        raise ValueError(f'{what} has shape {tuple(v.shape)}, expected {(n,)}')
    if v.device != device:
        raise ValueError(f'{what} is on {v.device}, expected {device}')
    return v.detach().to(torch.float32).contiguous()


def _same(t, like, what, dtype=None):
    if t.shape != like.shape or t.device != like.device or t.dtype != (dtype or like.dtype):
        raise ValueError(f'{what} is {tuple(t.shape)} {t.dtype} on {t.device}, expected {tuple(like.shape)} '
                         f'{dtype or like.dtype} on {like.device}')


def _check_dtype(t, what):
    require_device(t, what)
    if t.dtype not in DTYPES:
        raise ValueError(f'{what} must be fp32 or bf16, got {t.dtype}')


def _wanted(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---------------------------------------------------------------- the recurrence ------------

def _scan_forward(z, f, bias, h0, starts, lengths, save, checkpoint):
    T, B, N = z.shape
    dev = z.device
    z, f = rows_form(z.detach()), rows_form(f.detach())
    bias = _vector(bias, N, 'bias', dev)
    h = torch.empty(T, B, N, dtype=z.dtype, device=dev)
    last = torch.empty(B, N, dtype=torch.float32, device=dev)
    states = torch.empty((T + BLOCK - 1) // BLOCK, B, N, dtype=torch.float32, device=dev) if save else None
    z8 = f8 = (None, None)
    if save and checkpoint:
        z8, f8 = empty8(T * B, N, dev), empty8(T * B, N, dev)
    ws = _lib.workspace(_lib.WS_GATED_FWD, T, B, N, 1, 0, dev)
    args = _lib.GatedScanFwdArgs(T=T, B=B, N=N, bf16=_bf16(z), z=rows_of(z), f=rows_of(f), bias=_lib.ptr(bias),
                                 h0=_lib.ptr(h0), starts=_lib.ptr(starts), lengths=_lib.ptr(lengths), h=rows_of(h),
                                 h_last=_lib.ptr(last), states=_lib.ptr(states), z8=packed_of(*z8), f8=packed_of(*f8),
                                 workspace=_lib.ptr(ws), workspace_bytes=ws.numel())
    with torch.cuda.device(dev):
        _lib.call('delrec_gated_scan_fwd', args, _lib.stream_of(z))
    kept = (None, None, *z8, *f8) if z8[0] is not None else (z, f, None, None, None, None)
    return h, last, (*kept, bias, states, starts, lengths)


class GatedScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, f, bias, h0, starts, lengths, checkpoint):
        h0 = None if h0 is None else h0.detach().to(torch.float32).contiguous()
        h, last, kept = _scan_forward(z, f, bias, h0, starts, lengths, True, checkpoint)
        ctx.save_for_backward(*kept)
        ctx.shape, ctx.dtype = z.shape, z.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dlast):
        z, f, zq, zs, fq, fs, bias, states, starts, lengths = ctx.saved_tensors
        T, B, N = ctx.shape
        dev = dh.device
        dh, dlast = rows_form(dh), dlast.contiguous()
        dz, df = (torch.empty(ctx.shape, dtype=ctx.dtype, device=dev) for _ in range(2))
        db = torch.empty(N, dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        dh0 = torch.empty(B, N, dtype=torch.float32, device=dev) if ctx.needs_input_grad[3] else None
        ws = _lib.workspace(_lib.WS_GATED_BWD, T, B, N, 1, 0, dev)
        args = _lib.GatedScanBwdArgs(T=T, B=B, N=N, bf16=int(ctx.dtype == torch.bfloat16), z=rows_of(z), f=rows_of(f),
                                     z8=packed_of(zq, zs), f8=packed_of(fq, fs), bias=_lib.ptr(bias),
                                     states=_lib.ptr(states), starts=_lib.ptr(starts), lengths=_lib.ptr(lengths),
                                     dh=rows_of(dh), dlast=_lib.ptr(dlast), dz=rows_of(dz), df=rows_of(df),
                                     db=_lib.ptr(db), dh0=_lib.ptr(dh0), workspace=_lib.ptr(ws),
                                     workspace_bytes=ws.numel())
        with torch.cuda.device(dev):
            _lib.call('delrec_gated_scan_bwd', args, _lib.stream_of(dh))
        return (dz, df, None if db is None else db.to(ctx.bias_dtype), dh0, None, None, None)


def gated_scan(z, f, bias=None, h0=None, starts=None, lengths=None, checkpoint=False):
    """``h_t = h_{t-1} + k_t (z_t - h_{t-1})`` with ``k_t = sigmoid(-(f_t + bias))``: the output
    (T, B, N) in z's type and the state after the last step (B, N) in fp32.

    ``z``, ``f`` (T, B, N) fp32 or bf16, of any strides (column slices of one projection, a
    transposed batch-first tensor); ``bias`` (N,); ``h0`` (B, N) fp32, zero when absent;
    ``starts`` (T, B) bool: a sequence starts at this step, the state before it is dropped;
    ``lengths`` (B,) ints: from this step on a row is padding, its state stays, its output is 0
    and its inputs are not used. Differentiable in z, f, bias and h0; ``checkpoint=True`` keeps
    z and f in 8 bits for that."""
    _check_dtype(z, 'z')
    if z.dim() != 3 or 0 in z.shape[1:]:
        raise ValueError(f'z must be (T, B, N) with B, N > 0, got {tuple(z.shape)}')
    _same(f, z, 'f')
    T, B, N = z.shape
    if h0 is not None:
        if h0.shape != (B, N) or h0.device != z.device or h0.dtype != torch.float32:
            raise ValueError(f'h0 is {tuple(h0.shape)} {h0.dtype} on {h0.device}, expected {(B, N)} fp32 on {z.device}')
    if starts is not None:
        if starts.shape != (T, B) or starts.device != z.device:
            raise ValueError(f'starts is {tuple(starts.shape)} on {starts.device}, expected {(T, B)} on {z.device}')
        starts = starts.to(torch.bool).contiguous()
    if lengths is not None:
        if lengths.shape != (B,) or lengths.device != z.device or lengths.is_floating_point():
            raise ValueError(f'lengths is {tuple(lengths.shape)} {lengths.dtype} on {lengths.device}, expected {(B,)} '
                             f'integers on {z.device}')
        lengths = lengths.to(torch.int64).contiguous()
    if T == 0:
        return torch.zeros_like(z), (z.new_zeros(B, N, dtype=torch.float32) if h0 is None else h0.clone())
    if _wanted(z, f, bias, h0):
        return GatedScanFn.apply(z, f, bias, h0, starts, lengths, checkpoint)
    h0 = None if h0 is None else h0.contiguous()
    return _scan_forward(z, f, bias, h0, starts, lengths, False, False)[:2]


# ---------------------------------------------------------------- norms, gate, residual -----

def _norm_forward(o, g, x, w, scale, w2, eps, dtype, save, checkpoint):
    """(x', u, what the backward reads); ``o`` None: the norm of x alone."""
    N, dev = x.shape[-1], x.device
    shape = x.shape
    o, g, x = (None if t is None else rows_form(t.detach()) for t in (o, g, x))
    R0, R1 = row_counts(x)
    w, scale, w2 = (_vector(v, N, what, dev) for v, what in ((w, 'weight'), (scale, 'scale'), (w2, 'next_weight')))
    xo = torch.empty(shape, dtype=x.dtype, device=dev) if o is not None else None
    u = torch.empty(shape, dtype=dtype, device=dev) if w2 is not None else None
    stats = torch.empty(R0 * R1, 2, dtype=torch.float32, device=dev) if save else None
    o8 = g8 = x8 = (None, None)
    if save and checkpoint:
        x8 = empty8(R0 * R1, N, dev)
        if o is not None:
            o8, g8 = empty8(R0 * R1, N, dev), empty8(R0 * R1, N, dev)
    args = _lib.NormGateFwdArgs(R0=R0, R1=R1, N=N, bf16=int(dtype == torch.bfloat16), x_bf16=_bf16(x), o=rows_of(o),
                                g=rows_of(g), x=rows_of(x), w=_lib.ptr(w), scale=_lib.ptr(scale), w2=_lib.ptr(w2),
                                eps=float(eps), x_out=_lib.ptr(xo), u=_lib.ptr(u), stats=_lib.ptr(stats),
                                o8=packed_of(*o8), g8=packed_of(*g8), x8=packed_of(*x8))
    with torch.cuda.device(dev):
        _lib.call('delrec_norm_gate_fwd', args, _lib.stream_of(x))
    if x8[0] is not None:
        kept = (None, None, None, *o8, *g8, *x8)
    else:
        kept = (o, g, x, None, None, None, None, None, None)
    return xo, u, (*kept, w, scale, w2, stats)


class NormGateFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, o, g, x, w, scale, w2, eps, checkpoint):
        dtype = x.dtype if o is None else o.dtype
        xo, u, kept = _norm_forward(o, g, x, w, scale, w2, eps, dtype, True, checkpoint)
        ctx.save_for_backward(*kept)
        ctx.set_materialize_grads(False)
        ctx.shape, ctx.dtype, ctx.x_dtype, ctx.block = x.shape, dtype, x.dtype, o is not None
        ctx.rows = row_counts(rows_form(x))
        ctx.w_dtypes = tuple(None if v is None else v.dtype for v in (w, scale, w2))
        return (xo, u) if o is not None else u

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        o, g, x, oq, os_, gq, gs, xq, xs, w, scale, w2, stats = ctx.saved_tensors
        dxo, du = grads if ctx.block else (None, grads[0])
        if dxo is None and du is None:
            return (None,) * 8
        dev, N = stats.device, ctx.shape[-1]
        R0, R1 = ctx.rows
        dxo, du = (None if t is None else rows_form(t) for t in (dxo, du))
        dx = torch.empty(ctx.shape, dtype=ctx.x_dtype, device=dev)
        do = dg = dw = dscale = dw2 = None
        if ctx.block:
            do, dg = (torch.empty(ctx.shape, dtype=ctx.dtype, device=dev) for _ in range(2))
            dw, dscale = (torch.empty(N, dtype=torch.float32, device=dev) for _ in range(2))
        if w2 is not None:
            dw2 = torch.empty(N, dtype=torch.float32, device=dev)
        ws = _lib.workspace(_lib.WS_NORM_GATE_BWD, R0, R1, N, 1, 0, dev)
        flat = [None if t is None else rows_form(t) for t in (do, dg, dx)]
        args = _lib.NormGateBwdArgs(R0=R0, R1=R1, N=N, bf16=int(ctx.dtype == torch.bfloat16),
                                    x_bf16=int(ctx.x_dtype == torch.bfloat16), o=rows_of(o), g=rows_of(g), x=rows_of(x),
                                    o8=packed_of(oq, os_), g8=packed_of(gq, gs), x8=packed_of(xq, xs), w=_lib.ptr(w),
                                    scale=_lib.ptr(scale), w2=_lib.ptr(w2), stats=_lib.ptr(stats), dx_out=rows_of(dxo),
                                    du=rows_of(du), d_o=rows_of(flat[0]), dg=rows_of(flat[1]), dx=rows_of(flat[2]),
                                    dw=_lib.ptr(dw), dscale=_lib.ptr(dscale), dw2=_lib.ptr(dw2), workspace=_lib.ptr(ws),
                                    workspace_bytes=ws.numel())
        with torch.cuda.device(dev):
            _lib.call('delrec_norm_gate_bwd', args, _lib.stream_of(stats))
        dw, dscale, dw2 = (None if v is None else v.to(dt) for v, dt in zip((dw, dscale, dw2), ctx.w_dtypes))
        return do, dg, dx, dw, dscale, dw2, None, None


def _check_width(x):
    # over one column v - e <v e> cancels to eps / x^2 of v, which 32-bit norms do not resolve
    if x.dim() == 0 or x.shape[-1] < 2:
        raise ValueError(f'a norm needs (..., N) tensors with N >= 2, got {tuple(x.shape)}')


def _check_rows(o, g, x):
    _check_dtype(o, 'o')
    _same(g, o, 'g')
    if x.dtype not in (o.dtype, torch.float32):
        raise ValueError(f'x must be {o.dtype} or fp32, got {x.dtype}')
    _same(x, o, 'x', x.dtype)
    _check_width(o)


def norm_gate_residual(o, g, x, weight, scale, next_weight=None, eps=1e-6, checkpoint=False):
    """``x' = x + scale * rms(o) * weight * silu(g)`` and, with ``next_weight``, the next block's
    input ``u = rms(x') * next_weight`` (``None`` without): ``(x', u)``.

    ``o`` (the block's output) and ``g`` (its gate) are (..., N) fp32 or bf16, the residual
    stream ``x`` is of their type or fp32; ``weight``, ``scale``, ``next_weight`` (N,). x' has
    x's type, u has o's; u's norm is taken before x' is rounded. Differentiable in all six;
    ``checkpoint=True`` keeps o, g and x in 8 bits for that, the norms in 32."""
    _check_rows(o, g, x)
    if weight is None or scale is None:
        raise ValueError('norm_gate_residual needs weight and scale')
    if o.numel() == 0:
        y = x + (o * weight * scale * g).to(x.dtype)
        return y, None if next_weight is None else (y * next_weight).to(o.dtype)
    if _wanted(o, g, x, weight, scale, next_weight):
        return NormGateFn.apply(o, g, x, weight, scale, next_weight, eps, checkpoint)
    return _norm_forward(o, g, x, weight, scale, next_weight, eps, o.dtype, False, False)[:2]


def rms_norm(x, weight, eps=1e-6, checkpoint=False):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last axis of an fp32 or bf16 (..., N)
    tensor; ``checkpoint=True`` keeps x in 8 bits for the backward pass."""
    _check_dtype(x, 'x')
    _check_width(x)
    if weight is None:
        raise ValueError('rms_norm needs weight')
    if x.numel() == 0:
        return (x * weight).to(x.dtype)
    if _wanted(x, weight):
        return NormGateFn.apply(None, None, x, None, None, weight, eps, checkpoint)
    return _norm_forward(None, None, x, None, None, weight, eps, x.dtype, False, False)[1]


def gated_step(z, f, g, x, h, weight, scale, next_weight=None, bias=None, eps=1e-6, h_out=None):
    """One time step of the block for B rows, in one launch: ``h' = h + k (z - h)`` with ``k =
    sigmoid(-(f + bias))``, then ``norm_gate_residual`` of ``o = h'`` (kept in 32 bits, where the
    scan rounds its output to z's type): ``(x', u, h')``.

    ``z``, ``f``, ``g``, ``x`` (B, N) as there, the state ``h`` (B, N) fp32. ``h_out``: where h'
    goes, ``h`` itself to update in place. Not differentiable."""
    _check_rows(z, g, x)
    _same(f, z, 'f')
    if z.dim() != 2 or z.shape[0] == 0:
        raise ValueError(f'gated_step takes (B, N) tensors with B > 0, got {tuple(z.shape)}')
    _same(h, z, 'h', torch.float32)
    if weight is None or scale is None:
        raise ValueError('gated_step needs weight and scale')
    if _wanted(z, f, g, x, h, weight, scale, next_weight, bias):
        raise RuntimeError('gated_step has no backward pass: call it under torch.no_grad(), or gated_scan and '
                           'norm_gate_residual')
    B, N = z.shape
    dev = z.device
    if h_out is None:
        h_out = torch.empty(B, N, dtype=torch.float32, device=dev)
    else:
        _same(h_out, h, 'h_out')
        if not h_out.is_contiguous():
            raise ValueError('h_out must be contiguous')
    z, f, g, x = (rows_form(t) for t in (z, f, g, x))
    h = h.contiguous()
    bias, weight, scale, next_weight = (_vector(v, N, what, dev) for v, what in (
        (bias, 'bias'), (weight, 'weight'), (scale, 'scale'), (next_weight, 'next_weight')))
    xo = torch.empty(B, N, dtype=x.dtype, device=dev)
    u = torch.empty(B, N, dtype=z.dtype, device=dev) if next_weight is not None else None

    def step_rows(t):
        return _lib.Rows(t.data_ptr(), 0, t.stride(0))
    args = _lib.GatedStepArgs(B=B, N=N, bf16=_bf16(z), x_bf16=_bf16(x), z=step_rows(z), f=step_rows(f), g=step_rows(g),
                              x=step_rows(x), h=_lib.ptr(h), bias=_lib.ptr(bias), w=_lib.ptr(weight),
                              scale=_lib.ptr(scale), w2=_lib.ptr(next_weight), eps=float(eps), h_out=_lib.ptr(h_out),
                              x_out=_lib.ptr(xo), u=_lib.ptr(u))
    with torch.cuda.device(dev):
        _lib.call('delrec_gated_step', args, _lib.stream_of(z))
    return xo, u, h_out


# ---------------------------------------------------------------- the block -----------------

class GatedBlock(torch.nn.Module):
    """A residual block over (T, B, N): ``z, f, g = Linear(u)``, ``h = gated_scan(z, f)``, ``x', u'
    = norm_gate_residual(h, g, x)``, where u' is the next block's input. ``bias`` starts with
    leaks from two steps to some hundred, ``scale`` at ``scale_init``. With ``checkpoint=True``
    all that the block keeps for its backward pass is in 8 bits."""

    def __init__(self, N, bias=False, scale_init=0.5, eps=1e-6, checkpoint=False):
        super().__init__()
        self.N, self.eps, self.checkpoint = int(N), float(eps), bool(checkpoint)
        self.proj = (Linear8 if checkpoint else torch.nn.Linear)(N, 3 * N, bias=bias)
        self.gate_bias = torch.nn.Parameter(torch.linspace(0.0, 6.0, N))
        self.weight = torch.nn.Parameter(torch.ones(N))
        self.scale = torch.nn.Parameter(torch.full((N,), float(scale_init)))
        self.next_weight = torch.nn.Parameter(torch.ones(N))

    def forward(self, x, u, h0=None, starts=None, lengths=None):
        """(x', u', the state after the last step)."""
        z, f, g = self.proj(u).chunk(3, -1)
        h, last = gated_scan(z, f, self.gate_bias, h0, starts, lengths, checkpoint=self.checkpoint)
        x, u = norm_gate_residual(h, g, x, self.weight, self.scale, self.next_weight, self.eps,
                                  checkpoint=self.checkpoint)
        return x, u, last

    def step(self, x, u, h, h_out=None):
        """One time step, (B, N) tensors: (x', u', h')."""
        z, f, g = torch.nn.functional.linear(u, self.proj.weight, self.proj.bias).chunk(3, -1)
        return gated_step(z, f, g, x, h, self.weight, self.scale, self.next_weight, self.gate_bias, self.eps, h_out)
