"""Adam and AdamW on the HIP library: one launch over a model's tensors, states
in fp32 or in 8 bits.

Drop-in for ``torch.optim.Adam(model.parameters(), lr=0.001,
weight_decay=5e-4)`` of the reference's training loop (train.py:353, stepped at
train.py:143): the same constructor arguments and update, over
``gfd_adam_step``.  ``amsgrad``, ``maximize`` and ``differentiable`` can only be
false; ``foreach``, ``capturable`` and ``fused``, which choose among torch's own
implementations, change nothing.

* ``state_bits=32``: the two moments in fp32.  ``state_bits=8``: the first
  moment and the root of the second as e4m3 codes over a power-of-two scale per
  256 elements, rounded stochastically from ``seed`` (include/gfd.h): 2 bytes an
  element instead of 8.
* Parameters in fp32, bf16 or fp16, gradients in the same type; the arithmetic
  is fp32 and a parameter is rounded once.  There is no fp32 master copy of a
  16-bit parameter.
* A group's states are flat device buffers (``flat_state``); ``state[p]`` holds
  views of them, so ``state_dict`` / ``load_state_dict`` work as in torch, also
  with the state dict of a ``torch.optim.Adam`` / ``AdamW``.
* The step count is on the device, so ``step()`` can be captured into a graph
  (after one call outside of it, which makes the states) and every replay is a
  step; ``mark_stepped()`` after replays lets what watches the parameters'
  versions know.  ``lr`` may be a 0-dim fp32 device tensor, which replays then follow.
"""
from __future__ import annotations

from collections import defaultdict
from operator import attrgetter
from typing import Dict, Tuple

import numpy as np
import torch

from . import _lib

STATE_BLOCK = 256
_CODES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16,
          torch.float16: _lib.DTYPE_F16}


_grad, _dtype, _layout = attrgetter("grad"), attrgetter("dtype"), attrgetter("layout")
_data_ptr, _numel, _device, _contiguous = (torch.Tensor.data_ptr, torch.Tensor.numel,
                                           torch.Tensor.get_device, torch.Tensor.is_contiguous)
_NONE = type(None)


def _dense(p: torch.Tensor) -> bool:
    """No gaps and no overlaps: its elements are its storage's, in some order."""
    return p.is_contiguous() or torch.empty_like(p, device="meta").stride() == p.stride()


def _strides(p: torch.Tensor):
    """Of a parameter; None: contiguous."""
    return None if p.is_contiguous() else p.stride()


def _refuse(options: dict) -> None:
    for name in ("amsgrad", "maximize", "differentiable"):
        if options.get(name):
            raise NotImplementedError(f"gfd Adam: {name} is not supported")


class Adam(torch.optim.Optimizer):
    """``torch.optim.Adam`` (weight decay added to the gradient)."""

    _decoupled = False

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.0, amsgrad: bool = False, *, foreach=None,
                 maximize: bool = False, capturable: bool = False, differentiable: bool = False,
                 fused=None, state_bits: int = 32, seed: int = 0):
        _refuse(dict(amsgrad=amsgrad, maximize=maximize, differentiable=differentiable))
        self._flat: Dict[int, dict] = {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay, state_bits=state_bits, seed=seed,
                                      decoupled_weight_decay=self._decoupled))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    def _check_group(self, group: dict) -> None:
        lr, (b1, b2) = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor):
            if lr.dim() != 0 or lr.dtype != torch.float32:
                raise ValueError("gfd Adam: a tensor lr is a 0-dim float32 tensor")
        elif not lr >= 0:
            raise ValueError(f"gfd Adam: lr must be >= 0 (got {lr})")
        if not (0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError(f"gfd Adam: betas must be in [0, 1) (got {group['betas']})")
        if not group["eps"] >= 0:
            raise ValueError(f"gfd Adam: eps must be >= 0 (got {group['eps']})")
        if not group["weight_decay"] >= 0:
            raise ValueError(f"gfd Adam: weight_decay must be >= 0 (got {group['weight_decay']})")
        if group["state_bits"] not in (32, 8):
            raise ValueError(f"gfd Adam: state_bits is 32 or 8 (got {group['state_bits']})")
        if not 0 <= int(group["seed"]) < 2 ** 32:
            raise ValueError(f"gfd Adam: seed must be in [0, 2**32) (got {group['seed']})")
        _refuse(group)
        if group["decoupled_weight_decay"] != self._decoupled:
            raise ValueError("gfd Adam: Adam adds the weight decay to the gradient, AdamW applies it to "
                             "the parameter; a group is of the other kind")
        for p in group["params"]:
            if p.dtype not in _CODES:
                raise TypeError("gfd Adam: parameters must be float32, bfloat16 or float16 "
                                f"(got {p.dtype})")
            if not _dense(p):
                raise ValueError("gfd Adam: a parameter's elements must be dense in memory "
                                 f"(strides {p.stride()} of shape {tuple(p.shape)})")

    # -- the states ---------------------------------------------------------

    def flat_state(self, group: int = 0) -> Dict[str, torch.Tensor]:
        """The states of a parameter group, made on first use: ``step`` (int32, an
        entry per parameter) and flat ``exp_avg`` / ``exp_avg_sq`` in which every
        parameter starts at a multiple of 256.  With 8-bit states these are float8_e4m3fn
        codes, ``exp_avg_sq`` the root of the second moment, to be multiplied by
        ``exp_avg_scale`` / ``exp_avg_sq_scale`` (fp32, an entry per 256 elements)."""
        return {k: t for k, t in self._group_state(group).items() if isinstance(t, torch.Tensor)
                and k != "ticket"}

    def _group_state(self, gi: int) -> dict:
        params = self.param_groups[gi]["params"]
        f = self._flat.get(gi)
        if f is not None:
            if len(f["first"]) != len(params) or f["bits"] != self.param_groups[gi]["state_bits"]:
                raise RuntimeError("gfd Adam: a group's parameters and state_bits stay as they were at "
                                   "its first step")
            return f
        self._check_group(self.param_groups[gi])
        dev = params[0].device
        for p in params:
            if not p.is_cuda or p.device != dev:
                raise RuntimeError("gfd Adam: a group's parameters must be on one HIP device "
                                   f"(got {p.device} and {dev})")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("gfd Adam: call step() once before capturing it (the states are "
                               "made by the first call)")
        f = self._flat[gi] = self._buffers(params, self.param_groups[gi]["state_bits"], dev)
        for i, p in enumerate(params):
            self.state[p] = self._views(f, i, p)
        return f

    @staticmethod
    def _buffers(params: list, bits: int, dev) -> dict:
        first, total = [], 0
        for p in params:
            first.append(total)
            total += -(-p.numel() // STATE_BLOCK) * STATE_BLOCK
        total = max(total, STATE_BLOCK)          # of parameters without elements too there is a buffer
        f = {"first": first, "numel": [p.numel() for p in params], "bits": bits, "device": dev,
             "strides": [_strides(p) for p in params],      # the states have them too
             "step": torch.zeros(len(params), dtype=torch.int32, device=dev),
             "ticket": torch.zeros(1056, dtype=torch.int32, device=dev)}
        if f["bits"] == 32:
            f["exp_avg"] = torch.zeros(total, dtype=torch.float32, device=dev)
            f["exp_avg_sq"] = torch.zeros(total, dtype=torch.float32, device=dev)
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                f[k] = torch.zeros(total, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
                f[k + "_scale"] = torch.zeros(total // STATE_BLOCK, dtype=torch.float32, device=dev)
        f["plain"] = f["strides"].count(None) == len(params)
        f["states"] = [t for k, t in f.items() if isinstance(t, torch.Tensor) and k != "ticket"]
        # gfd_adam_tensor of every parameter; the two pointers are filled in at each step
        f["table"] = np.array([(0, 0, p.numel(), at, i) for i, (p, at) in enumerate(zip(params, first))],
                              dtype=np.int64)
        return f

    @staticmethod
    def _views(f: dict, i: int, p: torch.Tensor) -> Dict[str, torch.Tensor]:
        at, n = f["first"][i], p.numel()
        s = {"step": f["step"][i]}
        for k in ("exp_avg", "exp_avg_sq"):
            # in the parameter's own element order
            s[k] = f[k].as_strided(p.shape, p.stride(), at)
            if f["bits"] == 8:
                s[k + "_scale"] = f[k + "_scale"][at // STATE_BLOCK:-(-(at + n) // STATE_BLOCK)]
        return s

    def state_dict(self) -> dict:
        """As torch's; a state is a copy of its own, not a view of the flat buffers."""
        sd = super().state_dict()
        sd["state"] = {k: {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in s.items()}
                       for k, s in sd["state"].items()}
        return sd

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        """Of this class, or of torch.optim.Adam / AdamW (fp32 states).  One that is refused leaves
        the optimizer as it was.  States of the same ``state_bits`` are filled where they are, and
        so is an lr that is a tensor: a captured ``step()`` goes on from what was loaded (but for
        the numbers among the options, which it holds).  With other ``state_bits`` the states are
        made anew, and a captured step has to be captured again."""
        groups = []
        for g, mine in zip(state_dict["param_groups"], self.param_groups):
            groups.append({**{k: mine[k] for k in ("state_bits", "seed", "decoupled_weight_decay")}, **g})
        if len(groups) != len(state_dict["param_groups"]):
            raise ValueError("loaded state dict has a different number of parameter groups")
        before = self._flat, self.state, self.param_groups
        copies = []                     # (to, from) of everything that is kept, once nothing is refused
        try:
            super().load_state_dict({"state": {}, "param_groups": groups})
            self._flat, self.state = {}, defaultdict(dict)
            for gi, saved in enumerate(groups):
                self._load_group(gi, saved["params"], state_dict["state"], before, copies)
        except Exception:
            self._flat, self.state, self.param_groups = before
            raise
        for to, t in copies:
            to.copy_(t) if t is not None else to.zero_()

    def _load_group(self, gi: int, keys: list, states: dict, before: tuple, copies: list) -> None:
        flat, _, old_groups = before
        group, old, f = self.param_groups[gi], old_groups[gi], flat.get(gi)
        self._check_group(group)
        known = any(k in states for k in keys)
        # one that cannot be gone on with (other bits, parameters added, moved or laid out anew) is
        # made anew
        if (f is not None and f["bits"] == group["state_bits"] and
                f["numel"] == [p.numel() for p in group["params"]] and
                f["strides"] == [_strides(p) for p in group["params"]] and
                all(p.get_device() == f["device"].index for p in group["params"])):
            self._flat[gi] = f
            for i, p in enumerate(group["params"]):
                self.state[p] = self._views(f, i, p)
        elif known:
            self._group_state(gi)
        if gi in self._flat:
            for p, k in zip(group["params"], keys):
                copies += (self._loaded(group, p, states[k]) if k in states else
                           [(to, None) for to in self.state[p].values()])
        lr = old["lr"]
        if isinstance(lr, torch.Tensor):
            copies.append((lr, torch.as_tensor(group["lr"])))
            group["lr"] = lr

    def _loaded(self, group: dict, p: torch.Tensor, old: dict) -> list:
        """(to, from) of a parameter's states; says which one does not fit."""
        copies = []
        for name, to in self.state[p].items():
            if name not in old:
                raise ValueError(f"gfd Adam: the loaded state has no {name!r} (its states are not "
                                 f"those of state_bits={group['state_bits']})")
            t = torch.as_tensor(old[name])
            if t.shape != to.shape or (t.dtype.itemsize == 1 or to.dtype.itemsize == 1) and t.dtype != to.dtype:
                raise ValueError(f"gfd Adam: the loaded {name!r} is {t.dtype} {tuple(t.shape)}, "
                                 f"expected {to.dtype} {tuple(to.shape)}")
            copies.append((to, t))
        return copies

    @torch.no_grad()
    def __setstate__(self, state: dict) -> None:
        """A copy or an unpickled optimizer: its states, which came one by one, go back into
        flat buffers."""
        super().__setstate__(state)
        self._flat = {}
        for gi, group in enumerate(self.param_groups):
            old = {p: self.state[p] for p in group["params"] if self.state.get(p)}
            if old:
                self._group_state(gi)
                for p, s in old.items():
                    for to, t in self._loaded(group, p, s):
                        to.copy_(t)

    # -- the step -----------------------------------------------------------

    @torch.no_grad()
    def step(self, closure=None):
        """One step over every parameter that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            if group["params"]:
                self._step_group(group, self._group_state(gi))
        return loss

    def mark_stepped(self) -> None:
        """To be called after replays of a captured ``step()``: a replay writes the parameters
        and states, but raises no version counter of theirs, by which autograd and what is
        derived from parameters (the packed weights of an inference layer) notice a change."""
        for gi, group in enumerate(self.param_groups):
            self._raise_versions(self._flat.get(gi), group["params"])

    @staticmethod
    def _raise_versions(f, params: list) -> None:
        # (the flat buffers share theirs with the views of them)
        torch.autograd.graph.increment_version(params + f["states"] if f is not None else params)

    def _step_group(self, group: dict, f: dict) -> None:
        params = group["params"]
        grads = list(map(_grad, params))
        index, numel = f["device"].index, f["numel"]
        dtype, n = params[0].dtype, len(params)
        # the ordinary step, looked over a property at a time: every gradient there, dense and
        # contiguous like its parameter, one type, the device and sizes that the states were made for
        if (_NONE not in map(type, grads) and
                list(map(_dtype, params)).count(dtype) == n == list(map(_dtype, grads)).count(dtype) and
                list(map(_layout, grads)).count(torch.strided) == n and
                list(map(_device, params)).count(index) == n == list(map(_device, grads)).count(index) and
                list(map(_numel, params)) == numel == list(map(_numel, grads)) and
                all(map(_contiguous, params)) and all(map(_contiguous, grads)) and
                f["plain"] and dtype in _CODES):
            table = f["table"]
            table[:, 0] = list(map(_data_ptr, params))
            table[:, 1] = list(map(_data_ptr, grads))
            self._launch(group, f, dtype, table, params)
            return
        self._step_mixed(group, f)

    def _step_mixed(self, group: dict, f: dict) -> None:
        """A step whose gradients are missing in part, of several types or in other orders
        than their parameters'; says what is wrong with one that cannot be taken."""
        dev, numel = f["device"], f["numel"]
        index = dev.index
        tables: Dict[torch.dtype, Tuple[list, list, list]] = {}
        kept = []                       # copies of gradients, alive until the launch is queued
        dtype = params = grads = places = None
        for i, p in enumerate(group["params"]):
            g = p.grad
            if g is None:
                continue
            if p.dtype is not dtype:
                dtype = p.dtype
                params, grads, places = tables.setdefault(dtype, ([], [], []))
                if dtype not in _CODES:
                    raise RuntimeError(f"gfd Adam: a parameter changed its type to {dtype}")
            if (g.dtype is not dtype or g.is_sparse or g.get_device() != index or
                    p.get_device() != index):
                raise RuntimeError(f"gfd Adam: a gradient must be dense, {dtype} and on {dev} like its "
                                   f"parameter (got {g.layout}, {g.dtype}, {g.device})")
            n = numel[i]
            if p.numel() != n or g.numel() != n:
                raise RuntimeError(f"gfd Adam: a parameter changed its size from {n} to {p.numel()}")
            if _strides(p) != f["strides"][i]:
                raise RuntimeError("gfd Adam: a parameter changed its strides to "
                                   f"{p.stride()} after its states were made")
            if not (p.is_contiguous() and g.is_contiguous()) and g.stride() != p.stride():
                g = torch.empty_like(p).copy_(g)
                kept.append(g)
            params.append(p.data_ptr())
            grads.append(g.data_ptr())
            places.append(i)
        for dtype, (params, grads, places) in tables.items():
            table = f["table"][places]
            table[:, 0] = params
            table[:, 1] = grads
            self._launch(group, f, dtype, table, [group["params"][i] for i in places])

    def _launch(self, group: dict, f: dict, dtype: torch.dtype, table: np.ndarray, params: list) -> None:
        dev, lr, lr_ptr = f["device"], group["lr"], None
        if isinstance(lr, torch.Tensor):
            if lr.device != dev:
                raise RuntimeError(f"gfd Adam: lr is on {lr.device}, expected {dev}")
            lr, lr_ptr = 0.0, lr.data_ptr()
        b1, b2 = group["betas"]
        _check_apart(table, dtype.itemsize)
        _lib.call_on(dev, "gfd_adam_step", table.ctypes.data, len(table), _CODES[dtype], f["bits"],
                     f["exp_avg"].data_ptr(), f["exp_avg_sq"].data_ptr(),
                     _lib.ptr(f.get("exp_avg_scale")), _lib.ptr(f.get("exp_avg_sq_scale")),
                     f["step"].data_ptr(), float(lr), lr_ptr, float(b1), float(b2),
                     float(group["eps"]), float(group["weight_decay"]), 1 if self._decoupled else 0,
                     int(group["seed"]), f["ticket"].data_ptr(), _lib.stream_handle(dev))
        self._raise_versions(f, params)


def _check_apart(table: np.ndarray, itemsize: int) -> None:
    """Refuse parameters that share memory: one launch updates all of them."""
    begin, size = table[:, 0], table[:, 2] * itemsize
    if size.size > 1 and ((begin[1:] < begin[:-1] + size[:-1]) | (size[1:] == 0)).any():
        # not in the order of their addresses
        order = np.argsort(begin[size > 0], kind="stable")
        begin, size = begin[size > 0][order], size[size > 0][order]
        if (begin[1:] < begin[:-1] + size[:-1]).any():
            raise ValueError("gfd Adam: two parameters share memory")


class AdamW(Adam):
    """``torch.optim.AdamW`` (weight decay applied to the parameter)."""

    _decoupled = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, amsgrad: bool = False, **options):
        super().__init__(params, lr, betas, eps, weight_decay, amsgrad, **options)
