"""AdamW over many tensors in one pass (``csrc/adamw_multi.h``), moments in 32 or in 8 bits.

The reference trains with clip_grad_norm_ + Adam (``model/traintest_MegaCRN.py:104,129-130``), which the trainer keeps as one
kernel pair on its flat bucket.  ``AdamW`` adds decoupled weight decay, parameters that are separate tensors, bf16 parameters
with fp32 masters and 8-bit moments: 16 bytes a parameter and step instead of 28.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import lib, host, Adamw, T_F32, T_BF16
from .modules import _need_gpu

BLOCK = 64          # elements that share a scale of the 8-bit moments


class AdamW:
    """AdamW(params, lr, betas, eps, weight_decay, max_grad_norm, state_bits, seed, capturable)

    params: tensors, or dicts {"params": [...], "lr": ..., "weight_decay": ...} as for torch's optimizers; float32, or bfloat16
    (fp32 masters carry the update then), all of one type and device, contiguous.  `max_grad_norm` > 0 clips by the norm over ALL
    tensors, as clip_grad_norm_ before the step would, without writing the gradients; `total_norm` (device) is that norm.
    `state_bits`: 32, or 8 for moments in one byte with a scale for each 64 elements, rounded at random but reproducibly by `seed`.

    `step()` takes `.grad` of each parameter, `step(grads=[...])` the given tensors; None leaves a tensor and its moments alone.
    Learning rates and decays are read from `param_groups` at each step, `max_grad_norm` too; betas and eps are fixed.  (Not a torch.optim.Optimizer, which
    torch's schedulers ask for: set `param_groups[i]["lr"]`, as the trainer does.)  `capturable=True` keeps step counts and learning rates on the
    device, so that a step captured into a HIP graph can be replayed; there a changed learning rate takes effect by `sync_lr()`
    outside the capture.  One optimizer belongs to one sequence of steps on one stream at a time."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_grad_norm=0.0, state_bits=32,
                 seed=0, capturable=False):
        params = list(params)
        if params and not isinstance(params[0], dict):
            params = [{"params": params}]
        for g in params:
            if set(g) - {"params", "lr", "weight_decay"}:
                raise ValueError(f"AdamW: a group has params, lr and weight_decay; got {sorted(g)}")
        self.param_groups = [{"params": list(g["params"]), "lr": float(g.get("lr", lr)),
                              "weight_decay": float(g.get("weight_decay", weight_decay))} for g in params]
        self.params = [p for g in self.param_groups for p in g["params"]]
        if not self.params:
            raise ValueError("AdamW: no parameters")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("AdamW: a parameter is given twice")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32; got {state_bits}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1) or not 1.2e-38 <= eps < 3e38:
            raise ValueError(f"AdamW: betas must lie in [0, 1) and eps be a normal float32 above 0; got {betas}, {eps}")
        for g in self.param_groups:
            if not (g["lr"] >= 0 and g["weight_decay"] >= 0):
                raise ValueError("AdamW: lr and weight_decay must not be negative")
        if max_grad_norm != max_grad_norm:
            raise ValueError("AdamW: max_grad_norm is NaN")
        first = self.params[0]
        for p in self.params:
            if not isinstance(p, torch.Tensor) or p.dtype not in (torch.float32, torch.bfloat16) or p.dtype != first.dtype:
                raise TypeError("AdamW: parameters must be float32 or bfloat16 tensors, all of one type")
            if p.device != first.device or not p.is_contiguous():
                raise ValueError("AdamW: parameters must be contiguous tensors on one device")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("AdamW: two parameters share memory")
        host.adamw_step                        # raises where the host nodes are not built
        _need_gpu(first, "AdamW")
        self.device, self.dtype = first.device, first.dtype
        self._betas, self._eps, self.max_grad_norm = tuple(betas), float(eps), float(max_grad_norm or 0.0)
        self.state_bits, self.seed, self.capturable = state_bits, int(seed), bool(capturable)
        k = len(self.params)
        self._numel = (C.c_longlong * k)(*[p.numel() for p in self.params])
        self._cfg = Adamw(k, T_F32 if self.dtype == torch.float32 else T_BF16, state_bits, self.seed & 0xFFFFFFFF, int(self.capturable), 0, self.betas[0],
                          self.betas[1], self.eps, self.max_grad_norm, 1.0)
        n = lib.mcrn_adamw_arena_elements(C.byref(self._cfg), self._numel)
        if n < 0:
            raise ValueError("AdamW: a parameter has more than 2^34 - 1024 elements, or there are more than 2^20")
        dev = self.device
        if state_bits == 32:
            self._m, self._v = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
            self._ms = self._vs = None
        else:
            self._m, self._v = (torch.zeros(n, dtype=torch.uint8, device=dev) for _ in range(2))
            self._ms, self._vs = (torch.ones(n // BLOCK, dtype=torch.uint8, device=dev) for _ in range(2))
        self.offsets, at = [], 0
        for p in self.params:
            self.offsets.append(at)
            at += (p.numel() + BLOCK - 1) // BLOCK * BLOCK
        self.master = None
        if self.dtype == torch.bfloat16:
            self.master = torch.zeros(n, device=dev)
            self.sync_masters()
        nb = lib.mcrn_adamw_workspace_bytes(C.byref(self._cfg), self._numel)
        self._ws = torch.empty(nb, dtype=torch.uint8, device=dev)
        self.total_norm = torch.zeros((), device=dev)
        self._lr, self._wd, self._steps = (C.c_double * k)(), (C.c_double * k)(), (C.c_int * k)()
        self._dev = self._seen = None
        if self.capturable:
            self._dev = (torch.zeros(k, dtype=torch.float64, device=dev), torch.zeros(k, dtype=torch.float64, device=dev),
                         torch.zeros(k, dtype=torch.int32, device=dev))
            self.sync_lr()
        self._addresses()

    betas = property(lambda self: self._betas, doc="of the constructor; step counts and moments belong to them")
    eps = property(lambda self: self._eps, doc="of the constructor")

    def _addresses(self):
        self._numel_at = C.addressof(self._numel)
        self._hyper = tuple(C.addressof(a) for a in (self._lr, self._wd, self._steps)) if self._dev is None else tuple(t.data_ptr() for t in self._dev)

    def __setstate__(self, d):                 # a copy (copy.deepcopy, pickle) has arrays of its own
        self.__dict__.update(d)
        self._addresses()

    # -- learning rates
    def _read_groups(self):
        now = [(float(g["lr"]), float(g["weight_decay"])) for g in self.param_groups]      # (a tensor may change in place)
        if now == self._seen:
            return
        if any(not (lr >= 0 and wd >= 0) for lr, wd in now):
            raise ValueError(f"AdamW: lr and weight_decay must not be negative; the groups have {now}")
        self._seen, i = now, 0
        for g, (lr, wd) in zip(self.param_groups, now):
            for _ in g["params"]:
                self._lr[i], self._wd[i] = lr, wd
                i += 1

    def sync_lr(self):
        """capturable: brings the groups' learning rates and decays to the device (the next step, or replay, uses them)."""
        if self._dev is None:
            return
        self._read_groups()
        self._dev[0].copy_(torch.tensor(list(self._lr), dtype=torch.float64))
        self._dev[1].copy_(torch.tensor(list(self._wd), dtype=torch.float64))

    def sync_masters(self):
        """bf16 parameters: takes their values into the fp32 masters - after they were written by anything but `step` (a loaded model)."""
        if self.master is not None:
            for p, o in zip(self.params, self.offsets):
                self.master[o:o + p.numel()].copy_(p.detach().reshape(-1))

    # -- the step
    @torch.no_grad()
    def step(self, grads=None, grad_scale=1.0):
        """One update; grad_scale (> 0) multiplies the gradients before norm and clipping (1 / world_size after a summed all-reduce)."""
        params = self.params
        if grads is None:
            grads = [p.grad for p in params]
        if not self.capturable:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW.step inside a graph capture needs capturable=True: its step counts would be replayed unchanged")
            self._read_groups()
        cfg = self._cfg
        cfg.max_norm, cfg.grad_scale = self.max_grad_norm, float(grad_scale)
        host.adamw_step(C.addressof(cfg), params, grads, self._numel_at, *self._hyper, self._m, self._v, self._ms, self._vs,
                        self.master, self._ws, self.total_norm if self.max_grad_norm > 0 else None)

    def zero_grad(self, set_to_none=True):
        for p in self.params:
            if p.grad is not None:
                if set_to_none:
                    p.grad = None
                else:
                    p.grad.zero_()

    # -- state
    def moments(self):
        """(m, v) as float32 arenas: the tensors behind one another, each filled up with zeros to whole blocks of 64 (`offsets`).
        32 bits: the optimizer's own; 8 bits: what the codes stand for."""
        if self.state_bits == 32:
            return self._m, self._v
        return host.adamw_unpack(self._m, self._ms, self._v, self._vs)

    def steps(self):
        """Updates of each tensor so far."""
        return list(self._steps) if self._dev is None else self._dev[2].tolist()

    def state_dict(self):
        d = {"state_bits": self.state_bits, "seed": self.seed, "steps": self.steps(), "m": self._m.clone(), "v": self._v.clone(),
             "groups": [{"lr": g["lr"], "weight_decay": g["weight_decay"]} for g in self.param_groups]}
        if self._ms is not None:
            d["m_scale"], d["v_scale"] = self._ms.clone(), self._vs.clone()
        if self.master is not None:
            d["master"] = self.master.clone()
        return d

    def load_state_dict(self, d):
        """Takes what state_dict() of an optimizer of the same parameters and state_bits gave: moments, masters, step counts, seed and the
        groups' rates."""
        if d["state_bits"] != self.state_bits:
            raise ValueError(f"AdamW: the state holds {d['state_bits']}-bit moments, this optimizer {self.state_bits}-bit ones")
        mine = {"m": self._m, "v": self._v}
        if self._ms is not None:
            mine.update(m_scale=self._ms, v_scale=self._vs)
        if self.master is not None:
            mine["master"] = self.master
        for k, t in mine.items():
            if k not in d or d[k].shape != t.shape or d[k].dtype != t.dtype:
                raise ValueError(f"AdamW: the state's {k!r} is missing or not of shape {tuple(t.shape)} and type {t.dtype}")
        if len(d["steps"]) != len(self.params) or any(int(s) < 0 for s in d["steps"]):
            raise ValueError(f"AdamW: the state must hold a step count for each of the {len(self.params)} parameters")
        if "groups" in d and len(d["groups"]) != len(self.param_groups):
            raise ValueError(f"AdamW: the state has {len(d['groups'])} parameter groups, this optimizer {len(self.param_groups)}")
        for k, t in mine.items():
            t.copy_(d[k])
        for i, s in enumerate(d["steps"]):
            self._steps[i] = int(s)
        self.seed = int(d.get("seed", self.seed))
        self._cfg.seed = self.seed & 0xFFFFFFFF
        for g, h in zip(self.param_groups, d.get("groups", ())):
            g.update(lr=float(h["lr"]), weight_decay=float(h["weight_decay"]))
        if self._dev is not None:
            self._dev[2].copy_(torch.tensor(list(self._steps), dtype=torch.int32))
            self.sync_lr()
