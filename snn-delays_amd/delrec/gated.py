"""Gated linear recurrence, and the norms, gate and residual of the block around it, over the
same time-major (T, B, N) sequences as the delayed-LIF layers.

    gated_scan           h_t = h_{t-1} + k_t (z_t - h_{t-1}), k_t = sigmoid(-(f_t + bias))
    norm_gate_residual   x' = x + scale * rms(o) * weight * silu(g), u = rms(x') * next_weight
    rms_norm             u = rms(x) * weight
    add_norm             x' = x + y, u = rms(x') * weight, u also in 8 bits
    gated_step           one time step of both, for streaming input
    GatedBlock           the residual block they make with its Linear

where ``rms(v) = v / sqrt(mean(v^2) + eps)`` over the last axis. The recurrence is the leaky
integrator of ``LIFNode(decay_input=True)`` without its threshold, with a leak that each step's
input sets. Activations are fp32 or bf16; states, gates, norms and sums are in 32 bits. With
``checkpoint=True`` an operator keeps what its backward pass reads in 8 bits
(``delrec.checkpoint8``). Gradients are first-order and reverse-mode; forward calls can be
captured in a graph, backward passes cannot. No counterpart in the reference.
"""

import torch

from . import _lib
from .checkpoint8 import Linear8, Packed8


def gated_scan(z, f, bias=None, h0=None, starts=None, lengths=None, checkpoint=False):
    """``h_t = h_{t-1} + k_t (z_t - h_{t-1})`` with ``k_t = sigmoid(-(f_t + bias))``: the output
    (T, B, N) in z's type and the state after the last step (B, N) in fp32.

    ``z``, ``f`` (T, B, N) fp32 or bf16, of any strides (column slices of one projection, a
    transposed batch-first tensor); ``bias`` (N,); ``h0`` (B, N) fp32, zero when absent;
    ``starts`` (T, B) bool: a sequence starts at this step, the state before it is dropped;
    ``lengths`` (B,) ints: from this step on a row is padding, its state stays, its output is 0
    and its inputs are not used. Differentiable in z, f, bias and h0; ``checkpoint=True`` keeps
    z and f in 8 bits for that."""
    return _lib.require_ext().gated_scan(z, f, bias, h0, starts, lengths, checkpoint)


def norm_gate_residual(o, g, x, weight, scale, next_weight=None, eps=1e-6, checkpoint=False):
    """``x' = x + scale * rms(o) * weight * silu(g)`` and, with ``next_weight``, the next block's
    input ``u = rms(x') * next_weight`` (``None`` without): ``(x', u)``.

    ``o`` (the block's output) and ``g`` (its gate) are (..., N) fp32 or bf16, the residual
    stream ``x`` is of their type or fp32; ``weight``, ``scale``, ``next_weight`` (N,). x' has
    x's type, u has o's; u's norm is taken before x' is rounded. Differentiable in all six;
    ``checkpoint=True`` keeps o, g and x in 8 bits for that, the norms in 32."""
    return _lib.require_ext().norm_gate_residual(o, g, x, weight, scale, next_weight, eps, checkpoint)


def rms_norm(x, weight, eps=1e-6, checkpoint=False):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last axis of an fp32 or bf16 (..., N)
    tensor; ``checkpoint=True`` keeps x in 8 bits for the backward pass."""
    return _lib.require_ext().rms_norm(x, weight, eps, checkpoint)


def add_norm(x, y, weight, eps=1e-6, pack=False):
    """The residual stream and the next block's input: ``x' = x + y``, ``u = rms(x') * weight``:
    ``(x', u)``, or with ``pack`` ``(x', u, packed)``, u's ``checkpoint8.Packed8`` as ``pack8(u)`` makes
    it, in the same pass (not differentiable; for ``linear8``).

    ``y`` (..., N) fp32 or bf16, ``x`` of its type or fp32; ``weight`` (N,). x' has x's type, u has
    y's; u's norm is taken before x' is rounded. Differentiable in all three."""
    x, u, q, scale = _lib.require_ext().add_norm(x, y, weight, eps, pack)
    return (x, u, Packed8(q, scale, u.shape, u.dtype)) if pack else (x, u)


def gated_step(z, f, g, x, h, weight, scale, next_weight=None, bias=None, eps=1e-6, h_out=None):
    """One time step of the block for B rows, in one launch: ``h' = h + k (z - h)`` with ``k =
    sigmoid(-(f + bias))``, then ``norm_gate_residual`` of ``o = h'`` (kept in 32 bits, where the
    scan rounds its output to z's type): ``(x', u, h')``.

    ``z``, ``f``, ``g``, ``x`` (B, N) as there, the state ``h`` (B, N) fp32. ``h_out``: where h'
    goes, ``h`` itself to update in place, or memory that no input shares (anything else raises
    ``ValueError``). Not differentiable."""
    return _lib.require_ext().gated_step(z, f, g, x, h, weight, scale, next_weight, bias, eps, h_out)


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
