"""Selective state-space recurrence and the short causal convolution before it, over the same
time-major (T, B, N) sequences as the delayed-LIF layers.

    causal_conv       y_t = silu(bias + sum_i weight_i x_{t-W+1+i})
    selective_scan    d_t = softplus(dt_t + dt_bias), h_t = exp(d_t A) h_{t-1} + d_t x_t B_t,
                      y_t = (<C_t, h_t> + D x_t) silu(g_t)
    conv_step, selective_step   one time step of each, for streaming input
    SelectiveBlock    the residual block they make with its Linears and ``gated.add_norm``

A channel has S states, each with its own decay ``A``; the input sets the step size ``dt`` and the
maps ``B`` (into the states) and ``C`` (out of them), which all channels share. Activations are fp32
or bf16; states, decays and sums are in 32 bits. Gradients are first-order and reverse-mode; forward
calls can be captured in a graph, backward passes cannot. No counterpart in the reference.
"""

import math

import torch

from . import _lib
from .checkpoint8 import Linear8, linear8
from .gated import add_norm


def causal_conv(x, weight, bias=None, state=None, starts=None, lengths=None, silu=True):
    """``y_t = act(bias + sum_i weight[:, i] x_{t-W+1+i})`` for each channel, ``act`` being
    ``silu`` or nothing: the output (T, B, N) in x's type, and the inputs of the last W - 1 steps
    (B, W - 1, N), which the next call on the same sequences takes as its ``state``.

    ``x`` (T, B, N) fp32 or bf16, of any strides; ``weight`` (N, W) with 2 <= W <= 8, ``bias`` (N,);
    ``state`` (B, W - 1, N) in x's type: the inputs before the first step, zero when absent;
    ``starts`` (T, B) bool: a sequence starts at this step, the inputs before it count as zeros;
    ``lengths`` (B,) ints: from this step on a row is padding, its output is 0 and its inputs are not
    used. Differentiable in x, weight, bias and state."""
    return _lib.require_ext().causal_conv(x, weight, bias, state, starts, lengths, silu)


def conv_step(x, state, weight, bias=None, silu=True, state_out=None):
    """One time step of ``causal_conv``: x (B, N), the state (B, W - 1, N); ``(y, state')``.
    ``state_out``: where the state goes, ``state`` itself to update in place, or memory that no
    input shares (anything else raises ``ValueError``). Not differentiable."""
    return _lib.require_ext().conv_step(x, state, weight, bias, silu, state_out)


def selective_scan(x, dt, A, B, C, D=None, g=None, dt_bias=None, h0=None, starts=None, lengths=None):
    """``d_t = softplus(dt_t + dt_bias)``, ``h_t = exp(d_t A) h_{t-1} + d_t x_t B_t``, ``y_t =
    (<C_t, h_t> + D x_t) silu(g_t)`` (without the last factor where there is no ``g``): the output
    (T, B, N) in x's type and the state after the last step (B, N, S) in fp32.

    ``x``, ``dt``, ``g`` (T, B, N) and ``B``, ``C`` (T, B, S) fp32 or bf16, of any strides (column
    slices of one projection, a transposed batch-first tensor); ``A`` (N, S) with S <= 64 states a
    channel, ``D``, ``dt_bias`` (N,); ``h0`` (B, N, S) fp32, zero when absent; ``starts`` (T, B) bool:
    a sequence starts at this step, the state before it is dropped; ``lengths`` (B,) ints: from this
    step on a row is padding, its state stays, its output is 0 and its inputs are not used.
    Differentiable in all but the masks; the backward pass keeps the state before every 8th step."""
    return _lib.require_ext().selective_scan(x, dt, A, B, C, D, g, dt_bias, h0, starts, lengths)


def selective_step(x, dt, A, B, C, h, D=None, g=None, dt_bias=None, h_out=None):
    """One time step of ``selective_scan`` in one launch: x, dt, g (B, N), B, C (B, S), the state h
    (B, N, S) fp32; ``(y, h')``. ``h_out``: where h' goes, ``h`` itself to update in place, or memory
    that no input shares (anything else raises ``ValueError``). Not differentiable."""
    return _lib.require_ext().selective_step(x, dt, A, B, C, h, D, g, dt_bias, h_out)


class SelectiveBlock(torch.nn.Module):
    """A residual block over (T, B, N): ``x_in, g = Linear(u)``, ``c = causal_conv(x_in)``, ``low, B, C
    = Linear(c)``, ``dt = Linear(low)``, ``y = Linear(selective_scan(c, dt, ..., g))``, ``x', u' =
    add_norm(x, y)``, where u' is the next block's input. The inner width is ``expand * N``, ``S`` the
    states of an inner channel, ``W`` the convolution's steps, ``rank`` the width of ``low`` (N / 16
    by default). ``A`` starts at -1 .. -S, step sizes (by ``dt_bias``) between 1e-3 and 1e-1. With
    ``checkpoint=True`` the first Linear's input is kept in 8 bits, as ``add_norm`` packs it.
    ``undecayed``: parameters that are no weights, for an optimiser that decays weights."""

    undecayed = ('A_log', 'D', 'dt_bias')

    def __init__(self, N, S=16, W=4, expand=2, rank=None, bias=False, eps=1e-6, checkpoint=False):
        super().__init__()
        self.N, self.S, self.W, self.eps, self.checkpoint = int(N), int(S), int(W), float(eps), bool(checkpoint)
        self.inner, self.rank = int(expand * N), int(rank or max(1, N // 16))
        E = self.inner
        self.proj = (Linear8 if checkpoint else torch.nn.Linear)(N, 2 * E, bias=bias)
        self.conv_weight = torch.nn.Parameter(torch.empty(E, W).uniform_(-W ** -0.5, W ** -0.5))
        self.conv_bias = torch.nn.Parameter(torch.zeros(E))
        self.low = torch.nn.Linear(E, self.rank + 2 * S, bias=False)
        self.dt = torch.nn.Linear(self.rank, E, bias=False)
        step = torch.exp(torch.empty(E).uniform_(math.log(1e-3), math.log(1e-1)))
        self.dt_bias = torch.nn.Parameter(torch.log(torch.expm1(step)))
        self.A_log = torch.nn.Parameter(torch.log(torch.arange(1, S + 1, dtype=torch.float32)).repeat(E, 1))
        self.D = torch.nn.Parameter(torch.ones(E))
        self.out = torch.nn.Linear(E, N, bias=bias)
        self.next_weight = torch.nn.Parameter(torch.ones(N))

    def _maps(self, c):
        """(dt, B, C) of the convolution's output"""
        low, B, C = self.low(c).split([self.rank, self.S, self.S], -1)
        return self.dt(low), B, C

    def _join(self, x, y):
        if self.checkpoint and torch.is_grad_enabled():
            return add_norm(x, y, self.next_weight, self.eps, pack=True)
        return (*add_norm(x, y, self.next_weight, self.eps), None)

    def forward(self, x, u, packed=None, state=None, starts=None, lengths=None):
        """(x', u', u' in 8 bits or None, the state after the last step). ``packed``: u in 8 bits, as
        the block before gave it; ``state``: (convolution's, recurrence's)."""
        conv, h = (None, None) if state is None else state
        a = linear8(u, self.proj.weight, self.proj.bias, packed=packed) if self.checkpoint else self.proj(u)
        c, g = a.chunk(2, -1)
        c, conv = causal_conv(c, self.conv_weight, self.conv_bias, conv, starts, lengths)
        dt, B, C = self._maps(c)
        y, h = selective_scan(c, dt, -torch.exp(self.A_log), B, C, self.D, g, self.dt_bias, h, starts, lengths)
        return (*self._join(x, self.out(y)), (conv, h))

    def step(self, x, u, state):
        """One time step, (B, N) tensors: (x', u'); the state is updated in place."""
        conv, h = state
        c, g = torch.nn.functional.linear(u, self.proj.weight, self.proj.bias).chunk(2, -1)
        c, _ = conv_step(c, conv, self.conv_weight, self.conv_bias, state_out=conv)
        dt, B, C = self._maps(c)
        y, _ = selective_step(c, dt, -torch.exp(self.A_log), B, C, h, self.D, g, self.dt_bias, h_out=h)
        return add_norm(x, self.out(y), self.next_weight, self.eps)

    def zero_state(self, B, dtype=torch.float32):
        """The state before the first step of B rows; ``dtype``: the activations'."""
        dev = self.A_log.device
        return (torch.zeros(B, self.W - 1, self.inner, dtype=dtype, device=dev), torch.zeros(B, self.inner, self.S, device=dev))
