"""Gated linear recurrence over whole sequences and single steps, on the HIP kernels of ``csrc/glr_scan.h``.

The recurrent cell of the reference (``model/MegaCRN.py:38-48``) blends its state with a candidate,
``h = r * state + (1 - r) * hc``, where gate and candidate read the state: T steps are T launches in a row.  With gate and
candidate that come from the input alone the same blend is a first-order linear recurrence, and a sequence of any length
is one scan:

    a_t = sigmoid(gate_t)        h_t = a_t h_{t-1} + (1 - a_t) phi(cand_t)        phi = tanh or the identity

``gated_linear_recurrence`` runs it over (B, T, N, H) with its gradients, ``gated_linear_recurrence_step`` advances the state
of a server by one step in place (both in ``csrc/host_nodes.cpp``), ``AGLRCell`` is the module: the reference's graph convolution produces gate and
candidate of all steps at once.  States are fp32 whatever the inputs' type.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from ._lib import host
from .modules import AGCN


def gated_linear_recurrence(gate, cand, state=None, mask=None, activation="tanh"):
    """h_t = a_t h_{t-1} + (1 - a_t) phi(cand_t), a_t = sigmoid(gate_t), over the T steps of a sequence -> (out, last).

    gate (B, T, N, G), cand (B, T, N, H) of one type (float32, bfloat16, float16); G divides H and gate j holds for the
    channels j H/G .. (j+1) H/G - 1 (G = H: a gate for each channel, G = 1: one for each node).  state (B, N, H) float32 is
    h before the first step, None = zeros.  mask (B, T, N) or (B, T) bool: a step that is False keeps the state, whatever its
    gate and cand hold, and gives them a gradient of 0; a row that is False throughout returns its state.  `out` (B, T, N, H)
    has the inputs' type, `last` (B, N, H) is the float32 state behind the last step (T = 0: the state itself).

    Strided inputs (slices of one product, expanded masks) are read in place as long as the last dimension is contiguous.
    Differentiable in gate, cand and state, once and in reverse mode (dual tensors and traces are refused).  A backward pass inside
    a graph capture wants leaves that no eager graph holds."""
    return host.glr(gate, cand, state, mask, activation)


def gated_linear_recurrence_step(gate, cand, state, mask=None, activation="tanh"):
    """One step of the recurrence for serving: gate (B, N, G), cand (B, N, H), mask (B, N) or (B,).  `state` (B, N, H) float32,
    contiguous, is advanced in place (inputs may lie in its memory); returns it in the inputs' type as a new tensor.  Not differentiable."""
    return host.glr_step(gate, cand, state, mask, activation)


class AGLRCell(nn.Module):
    """Recurrent cell beside ``AGCRNCell`` (``model/MegaCRN.py:30-51``) for long sequences: the adaptive-graph convolution
    (``AGCN``, ``:16-28``) of the inputs gives gate and candidate of every step in one product, the recurrence runs over them."""

    def __init__(self, node_num, dim_in, dim_out, cheb_k):
        super().__init__()
        self.node_num = node_num
        self.hidden_dim = dim_out
        self.gate_cand = AGCN(dim_in, 2 * dim_out, cheb_k)

    def _products(self, x, supports):
        if x.shape[0] == 0:                       # no batch, or no step
            y = x.new_empty(0, x.shape[1], 2 * self.hidden_dim)
        else:
            y = self.gate_cand(x, supports)
        return y[..., :self.hidden_dim], y[..., self.hidden_dim:]

    def forward(self, x, state, supports, mask=None):
        """x (B, T, num_nodes, dim_in), state (B, num_nodes, hidden_dim) or None -> (states (B, T, num_nodes, hidden_dim), last state)."""
        B, T = x.shape[:2]
        gate, cand = self._products(x.reshape(B * T, *x.shape[2:]), supports)
        gate, cand = (t.unflatten(0, (B, T)) for t in (gate, cand))
        return gated_linear_recurrence(gate, cand, None if state is None else state.to(x.device), mask)

    @torch.no_grad()
    def step(self, x, state, supports, mask=None):
        """One step in place, for serving: x (B, num_nodes, dim_in) -> the new state."""
        return gated_linear_recurrence_step(*self._products(x, supports), state, mask)

    def init_hidden_state(self, batch_size):
        return torch.zeros(batch_size, self.node_num, self.hidden_dim)
