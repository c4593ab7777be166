"""Gated linear recurrence over whole sequences and single steps, on the HIP kernels of ``csrc/glr_scan.h``.

The recurrent cell of the reference (``model/MegaCRN.py:38-48``) blends its state with a candidate,
``h = r * state + (1 - r) * hc``, where gate and candidate read the state: T steps are T launches in a row.  With gate and
candidate that come from the input alone the same blend is a first-order linear recurrence, and a sequence of any length
is one scan:

    a_t = sigmoid(gate_t)        h_t = a_t h_{t-1} + (1 - a_t) phi(cand_t)        phi = tanh or the identity

``gated_linear_recurrence`` runs it over (B, T, N, H) with its gradients, ``gated_linear_recurrence_step`` advances the state
of a server by one step in place, ``AGLRCell`` is the module: the reference's graph convolution produces gate and
candidate of all steps at once.  States are fp32 whatever the inputs' type.
"""
from __future__ import annotations

import ctypes as C

import torch
import torch.nn as nn

from ._lib import lib, check, Glr, DTYPES, ACTIVATIONS
from .modules import AGCN, _need_gpu, _stream


def _kept(t, last_contiguous):
    """`t` with strides the kernels take: none negative (torch has none) and, if asked, a last dimension without gaps."""
    return t if not last_contiguous or t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _strides3(t):
    return (C.c_longlong * 3)(*[0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride())])


def _check(gate, cand, state, mask, activation, who, lead):
    """Everything that the C entry point cannot see in raw pointers."""
    for name, t in (("gate", gate), ("cand", cand)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{who}: {name} must be a tensor")
        if t.dtype not in DTYPES:
            raise TypeError(f"{who}: {name} must be float32, bfloat16 or float16; got {t.dtype}")
    if cand.dim() != lead + 1 or gate.dim() != lead + 1 or gate.shape[:lead] != cand.shape[:lead]:
        raise ValueError(f"{who}: gate {tuple(gate.shape)} and cand {tuple(cand.shape)} must agree in all but their last of {lead + 1} dimensions")
    if gate.dtype != cand.dtype or gate.device != cand.device:
        raise ValueError(f"{who}: gate and cand must have one type and one device")
    H, G = cand.shape[-1], gate.shape[-1]
    if H < 1 or G < 1 or H % G:
        raise ValueError(f"{who}: the gates' number {G} must divide the channels' {H}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{who}: activation must be one of {sorted(ACTIVATIONS)}; got {activation!r}")
    want = (cand.shape[0], cand.shape[-2], H)
    if state is not None and (not isinstance(state, torch.Tensor) or state.dtype != torch.float32 or state.device != cand.device or tuple(state.shape) != want):
        raise ValueError(f"{who}: state must be a float32 tensor of shape {want} on {cand.device}")
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.bool or mask.device != cand.device:
            raise ValueError(f"{who}: mask must be a bool tensor on {cand.device}")
        rows = tuple(cand.shape[:lead])
        if mask.dim() == lead - 1:                       # (B, T) or (B,): the same for every node
            mask = mask.unsqueeze(-1)
        if mask.dim() != lead or any(m not in (1, r) for m, r in zip(mask.shape, rows)):
            raise ValueError(f"{who}: mask must be {rows}, with 1 where all share an entry, or lack its last dimension; got {tuple(mask.shape)}")
        mask = mask.expand(rows)
    _need_gpu(cand, who)
    return mask


def _dims(gate, cand, mask, activation, dout=None):
    B, T, N, H = cand.shape
    d = Glr(B, T, N, H, gate.shape[-1], DTYPES[cand.dtype], ACTIVATIONS[activation], 0)
    d.gate_s, d.cand_s = _strides3(gate), _strides3(cand)
    if mask is not None:
        d.mask_s = _strides3(mask)
    if dout is not None:
        d.dout_s = _strides3(dout)
    return d


def _p(t):
    return None if t is None else t.data_ptr()


def _workspace(d, backward, device):
    """From torch's allocator, call by call: it knows streams and graph captures, and the block is free again when the kernels are queued."""
    nb = lib.mcrn_glr_workspace_bytes(C.byref(d), backward)
    return (torch.empty(nb, dtype=torch.uint8, device=device), nb) if nb else (None, 0)


def _forward(gate, cand, state, mask, activation, keep):
    B, T, N, H = cand.shape
    dev = cand.device
    with torch.cuda.device(dev):
        d = _dims(gate, cand, mask, activation)
        out = torch.empty(B, T, N, H, dtype=cand.dtype, device=dev)
        last = torch.empty(B, N, H, device=dev)
        nck = lib.mcrn_glr_checkpoint_floats(C.byref(d)) if keep else 0
        ckpt = torch.empty(nck, device=dev) if nck else None
        ws, nb = _workspace(d, 0, dev)
        check(lib.mcrn_glr_forward(C.byref(d), gate.data_ptr(), cand.data_ptr(), _p(mask), _p(state), _p(ws), nb,
                                   out.data_ptr(), last.data_ptr(), _p(ckpt), _stream()), "mcrn_glr_forward")
    return out, last, ckpt


class _RecurrenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, cand, state, mask, activation):
        gate, cand = _kept(gate, True), _kept(cand, True)
        state = None if state is None else state.contiguous()
        out, last, ckpt = _forward(gate, cand, state, mask, activation, any(ctx.needs_input_grad))
        # fp32: the backward reads the states before every 8th step from `out` itself; 16-bit types keep those in fp32
        ctx.save_for_backward(gate, cand, state, mask, out if cand.dtype == torch.float32 else ckpt)
        ctx.activation = activation
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlast):
        gate, cand, state, mask, kept = ctx.saved_tensors
        dev = cand.device
        if dout is None and dlast is None:
            return None, None, None, None, None
        dout = None if dout is None else _kept(dout, True)
        dlast = None if dlast is None else dlast.contiguous()
        with torch.cuda.device(dev):
            d = _dims(gate, cand, mask, ctx.activation, dout)
            dgate = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
            dcand = torch.empty(cand.shape, dtype=cand.dtype, device=dev)
            dstate = torch.empty_like(state) if ctx.needs_input_grad[2] else None
            ws, nb = _workspace(d, 1, dev)
            check(lib.mcrn_glr_backward(C.byref(d), gate.data_ptr(), cand.data_ptr(), _p(mask), _p(state), _p(kept), _p(dout),
                                        _p(dlast), _p(ws), nb, dgate.data_ptr(), dcand.data_ptr(), _p(dstate), _stream()),
                  "mcrn_glr_backward")
        return dgate, dcand, dstate, None, None


def gated_linear_recurrence(gate, cand, state=None, mask=None, activation="tanh"):
    """h_t = a_t h_{t-1} + (1 - a_t) phi(cand_t), a_t = sigmoid(gate_t), over the T steps of a sequence -> (out, last).

    gate (B, T, N, G), cand (B, T, N, H) of one type (float32, bfloat16, float16); G divides H and gate j holds for the
    channels j H/G .. (j+1) H/G - 1 (G = H: a gate for each channel, G = 1: one for each node).  state (B, N, H) float32 is
    h before the first step, None = zeros.  mask (B, T, N) or (B, T) bool: a step that is False keeps the state, whatever its
    gate and cand hold, and gives them a gradient of 0; a row that is False throughout returns its state.  `out` (B, T, N, H)
    has the inputs' type, `last` (B, N, H) is the float32 state behind the last step (T = 0: the state itself).

    Strided inputs (slices of one product, expanded masks) are read in place as long as the last dimension is contiguous.
    Differentiable in gate, cand and state, once.  A backward pass inside a graph capture wants leaves that no eager graph holds."""
    mask = _check(gate, cand, state, mask, activation, "gated_linear_recurrence", 3)
    if cand.numel() == 0:                                # nothing to read or no step to take
        last = torch.zeros(cand.shape[0], cand.shape[2], cand.shape[3], device=cand.device) if state is None else state.clone()
        return torch.empty_like(cand), last
    return _RecurrenceFn.apply(gate, cand, state, mask, activation)


def gated_linear_recurrence_step(gate, cand, state, mask=None, activation="tanh"):
    """One step of the recurrence for serving: gate (B, N, G), cand (B, N, H), mask (B, N) or (B,).  `state` (B, N, H) float32,
    contiguous, is advanced in place; returns it in the inputs' type as a new tensor.  Not differentiable."""
    if state is None or not state.is_contiguous():
        raise ValueError("gated_linear_recurrence_step: state must be a contiguous tensor; it is advanced in place")
    mask = _check(gate, cand, state, mask, activation, "gated_linear_recurrence_step", 2)
    if torch.is_grad_enabled() and (gate.requires_grad or cand.requires_grad or state.requires_grad):
        raise RuntimeError("gated_linear_recurrence_step is not differentiable: call it under torch.no_grad()")
    gate, cand = _kept(gate, True), _kept(cand, True)
    dev = cand.device
    out = torch.empty(cand.shape, dtype=cand.dtype, device=dev)
    if out.numel() == 0:
        return out
    with torch.cuda.device(dev):
        d = _dims(gate.unsqueeze(1), cand.unsqueeze(1), None if mask is None else mask.unsqueeze(1), activation)
        check(lib.mcrn_glr_forward(C.byref(d), gate.data_ptr(), cand.data_ptr(), _p(mask), state.data_ptr(), None, 0,
                                   out.data_ptr(), state.data_ptr(), None, _stream()), "mcrn_glr_forward")
    return out


class AGLRCell(nn.Module):
    """Recurrent cell beside ``AGCRNCell`` (``model/MegaCRN.py:30-51``) for long sequences: the adaptive-graph convolution
    (``AGCN``, ``:16-28``) of the inputs gives gate and candidate of every step in one product, the recurrence runs over them."""

    def __init__(self, node_num, dim_in, dim_out, cheb_k):
        super().__init__()
        self.node_num = node_num
        self.hidden_dim = dim_out
        self.gate_cand = AGCN(dim_in, 2 * dim_out, cheb_k)

    def _products(self, x, supports):
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
