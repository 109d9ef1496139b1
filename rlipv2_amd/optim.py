"""Fused optimiser step of the bf16 train step: gradient-norm clipping (max-norm 0.1, reference
engine.py:170-172) + AdamW with the reference's three parameter groups (main.py:523-541) on float32 master
weights, writing the bf16 parameters back -- two HIP launches (csrc/fused_adamw.hip, C ABI
include/rlipv2_optim.h) instead of ~90 PyTorch launches.

For any other optimiser: the global norm over a list of gradients and clipping to it as operators of their own (`clip_grad_norm_`,
`grad_norm`, `GradientClipper`; csrc/grad_norm.hip, C ABI include/rlipv2_gradnorm.h)."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _lib, roofline


def _same_layout(a, b):
    """same element order in memory (strides of size-1 dimensions are arbitrary and ignored)"""
    return a.shape == b.shape and all(sa == sb for n, sa, sb in zip(a.shape, a.stride(), b.stride()) if n > 1)


class _Group(ctypes.Structure):
    _fields_ = [(n, ctypes.c_float) for n in ("beta1", "beta2", "one_minus_beta1", "one_minus_beta2", "eps", "decay",
                                              "step_size", "bias_correction2_sqrt")]


class FusedMasterAdamW:
    """AdamW over float32 master copies of bf16 parameters; same update rule as torch.optim.AdamW and the
    same clipping as torch.nn.utils.clip_grad_norm_ (tests/test_optim_gpu.py compares them step by step)."""

    def __init__(self, model, lr=1.41e-4, lr_backbone=1.41e-5, text_encoder_lr=1.41e-5, weight_decay=1e-4,
                 betas=(0.9, 0.999), eps=1e-8):
        named = [(n, p) for n, p in model.named_parameters() if p.requires_grad]
        if not named:
            raise ValueError("no trainable parameters")
        for n, p in named:
            if not p.is_cuda:
                raise RuntimeError("Not implemented on the CPU")
            if p.dtype != torch.bfloat16:
                raise RuntimeError(f"FusedMasterAdamW expects bfloat16 parameters ({n} is {p.dtype})")
        self.names = [n for n, _ in named]
        self.params = [p for _, p in named]
        self.master = [p.detach().float().clone() for p in self.params]
        self.exp_avg = [torch.zeros_like(m) for m in self.master]
        self.exp_avg_sq = [torch.zeros_like(m) for m in self.master]
        group_of = [1 if "backbone" in n else 2 if "text_encoder" in n else 0 for n in self.names]
        lrs = [lr, lr_backbone, text_encoder_lr]
        used = sorted(set(group_of))
        self.group_index = [used.index(g) for g in group_of]
        self.param_groups = [{"lr": lrs[g], "betas": tuple(betas), "eps": eps, "weight_decay": weight_decay,
                              "params": [p for p, gi in zip(self.params, group_of) if gi == g]} for g in used]
        self.t = 0
        self.steps = [0] * len(self.params)     # per-parameter step count, as torch.optim keeps it
        self.device = self.params[0].device
        self.sqnorm = torch.zeros(1, dtype=torch.float32, device=self.device)
        self._last_grad_scale = 1.0
        sizes = [ctypes.c_int() for _ in range(4)]
        _lib.lib().adamw_abi_sizes(*[ctypes.byref(s) for s in sizes])
        assert (sizes[0].value, sizes[1].value, sizes[2].value) == (56, 8, ctypes.sizeof(_Group)), "ABI mismatch"
        self.chunk = sizes[3].value
        self._tables = {}        # tuple of gradient pointers -> (tensor table, chunk table, n_chunks)
        self._relayout = {}
        self._checked = [None] * len(self.params)    # per parameter: the gradient OBJECT whose dtype / layout passed last

    def zero_grad(self, set_to_none=True):
        for p in self.params:
            p.grad = None

    def _grads(self):
        """(indices, gradients) of the parameters that have one.  The graphed step hands over the SAME gradient tensors every
        step (static buffers): a gradient object that passed the dtype / layout check once is not checked again -- the
        per-parameter shape / stride comparison was ~1 ms of Python per step for ~750 parameters, between the end of the
        backward graph and the optimiser's two launches."""
        idx, grads = [], []
        checked = self._checked
        for i, p in enumerate(self.params):
            g = p.grad
            if g is None:
                continue                                   # torch.optim skips parameters without gradient
            if g is checked[i]:
                idx.append(i)
                grads.append(g)
                continue
            if g.dtype != torch.bfloat16 or not _same_layout(g, p):
                # e.g. a convolution weight kept channels-last whose gradient arrives contiguous: re-lay it
                # out into a persistent buffer (stable address -> the pointer table stays cached)
                buf = self._relayout.get(i)
                if buf is None:
                    buf = self._relayout[i] = torch.empty_like(p)
                g = buf.copy_(g)
                self.grad_copies = getattr(self, "grad_copies", 0) + 1
            else:
                checked[i] = g
            idx.append(i)
            grads.append(g)
        return idx, grads

    def _table(self, idx, grads, eff_group):
        # (parameter addresses are part of the key: modules may re-lay their parameters out, deform_attn.adjacent_cat)
        key = (tuple(idx), tuple(g.data_ptr() for g in grads), tuple(eff_group), tuple(self.params[i].data_ptr() for i in idx))
        hit = self._tables.get(key)
        if hit is not None:
            return hit
        rows = np.empty((len(idx), 7), dtype=np.int64)
        chunks = []
        for r, (i, g) in enumerate(zip(idx, grads)):
            n = self.params[i].numel()
            rows[r] = (g.data_ptr(), self.master[i].data_ptr(), self.exp_avg[i].data_ptr(),
                       self.exp_avg_sq[i].data_ptr(), self.params[i].data_ptr(), n, eff_group[r])
            chunks += [(r, c) for c in range((n + self.chunk - 1) // self.chunk)]
        t_dev = torch.from_numpy(rows).to(self.device)
        c_dev = torch.from_numpy(np.asarray(chunks, dtype=np.int32).reshape(-1, 2)).to(self.device)
        self.table_builds = getattr(self, "table_builds", 0) + 1
        if len(self._tables) > 8:
            self._tables.clear()
        self._tables[key] = (t_dev, c_dev, len(chunks))
        return self._tables[key]

    @torch.no_grad()
    def step(self, max_norm=0.1, grad_scale=1.0):
        """`grad_scale`: factor on every gradient, applied inside the kernels (norm and update): the data-parallel step
        hands over the all-reduced SUM with grad_scale = 1 / world instead of scaling its 425 MB buffer first."""
        idx, grads = self._grads()
        if not idx:
            return
        self._last_grad_scale = float(grad_scale)
        self.t += 1
        # bias corrections depend on how many updates a parameter has had; a parameter that skipped a step
        # (no gradient) lags behind, so the kernel's "group" is (parameter group, update count)
        for i in idx:
            self.steps[i] += 1
        pairs = sorted({(self.group_index[i], self.steps[i]) for i in idx})
        if len(pairs) > 8:
            raise RuntimeError("FusedMasterAdamW: more than 8 distinct (group, step-count) combinations")
        eff_group = [pairs.index((self.group_index[i], self.steps[i])) for i in idx]
        t_dev, c_dev, n_chunks = self._table(idx, grads, eff_group)
        groups = (_Group * len(pairs))()
        for gi, (pg, t) in enumerate(pairs):
            g = self.param_groups[pg]
            b1, b2 = g["betas"]
            groups[gi] = _Group(b1, b2, 1.0 - b1, 1.0 - b2, g["eps"], 1.0 - g["lr"] * g["weight_decay"],
                                g["lr"] / (1.0 - b1 ** t), math.sqrt(1.0 - b2 ** t))
        L = _lib.lib()
        stream = torch.cuda.current_stream(self.device).cuda_stream
        clip = max_norm is not None and max_norm > 0
        if clip:
            st = L.adamw_grad_sqnorm_bf16(t_dev.data_ptr(), c_dev.data_ptr(), n_chunks, self.sqnorm.data_ptr(), stream)
            if st:
                raise RuntimeError("adamw_grad_sqnorm: " + _lib.strerror(st))
        st = L.adamw_step_scaled_bf16(t_dev.data_ptr(), c_dev.data_ptr(), n_chunks, self.sqnorm.data_ptr(),
                                      float(max_norm) if clip else 0.0, float(grad_scale), groups, len(pairs), stream)
        if st:
            raise RuntimeError("adamw_step: " + _lib.strerror(st))
        # gradient (bf16) read twice (norm + update), master / two moments read + written (f32), bf16 parameter written
        n = sum(self.params[i].numel() for i in idx)
        roofline.add(n * (2 * (2 if clip else 1) + 3 * 8 + 2))

    def grad_norm(self):
        """norm of the last step's gradients as the update saw them, i.e. with that step's `grad_scale` applied -- the
        value the reference logs from clip_grad_norm_ (engine.py:170); a device tensor, no sync."""
        return self.sqnorm.sqrt() * self._last_grad_scale

    def state_dict(self):
        return {"t": self.t, "steps": list(self.steps), "names": list(self.names), "master": self.master, "exp_avg": self.exp_avg,
                "exp_avg_sq": self.exp_avg_sq, "param_groups": [{k: v for k, v in g.items() if k != "params"}
                                                                for g in self.param_groups]}

    def load_state_dict(self, state):
        if list(state["names"]) != self.names:
            raise ValueError("optimizer state belongs to a different parameter set")
        self.t = int(state["t"])
        self.steps = list(state.get("steps", [self.t] * len(self.params)))
        with torch.no_grad():
            for dst, src in ((self.master, state["master"]), (self.exp_avg, state["exp_avg"]),
                             (self.exp_avg_sq, state["exp_avg_sq"])):
                for d, s in zip(dst, src):
                    d.copy_(s)
            for p, m in zip(self.params, self.master):
                p.copy_(m)
        for g, s in zip(self.param_groups, state["param_groups"]):
            g.update(s)


# ---- the global gradient norm as an operator of its own ------------------------------------------------------------------
_ORDERS = {1.0: 1, 2.0: 2, math.inf: 3}
_GRAD_TYPES = {torch.float32: _lib.MSDA_F32, torch.bfloat16: _lib.MSDA_BF16}


def _dense(t):
    """every element of the tensor's memory span belongs to it, once"""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _spans(tensors):
    """[begin, end) byte ranges of the tensors that have elements, by address"""
    return sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), i) for i, t in enumerate(tensors) if t.numel())


class GradientClipper:
    """Global norm over many tensors, and clipping to it, for tensors that stay where they are (a graphed step's static
    gradient buffers, the views of a flat gradient buffer): the lists are laid out once, a call is its launches.

    `tensors`: gradients on one GPU, bfloat16 or float32 (also mixed), each dense in memory (contiguous or permuted, at any
    offset).  `out`: where `clip` writes, tensors of the same shapes and element order, bfloat16 or float32 (e.g. the float32
    gradients of master weights: conversion and clipping in one pass); None: in place.  The memory the tensors
    have when the object is made is what it works on, and it is kept alive: after `.data =` or `zero_grad(set_to_none=True)` make a
    new one.

    Results as of torch.nn.utils.clip_grad_norm_ on gradients multiplied by `grad_scale` (reference engine.py:170-172), with
    float64 sums: no square overflows, and calls are repeatable bit for bit.  Capturable in a HIP graph; every call has its own
    workspace."""

    def __init__(self, tensors, out=None):
        self.tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        self.out = None if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
        if self.out is not None and len(self.out) != len(self.tensors):
            raise ValueError(f"GradientClipper: {len(self.tensors)} tensors but {len(self.out)} outputs")
        for what, group in (("gradient", self.tensors), ("output", self.out or ())):
            for t in group:
                if not isinstance(t, torch.Tensor) or t.is_sparse or t.dtype not in _GRAD_TYPES:
                    raise TypeError(f"GradientClipper: every {what} must be a dense bfloat16 or float32 tensor "
                                    f"(got {t.dtype if isinstance(t, torch.Tensor) else type(t).__name__})")
                if not _dense(t):
                    raise ValueError(f"GradientClipper: a {what} of shape {tuple(t.shape)} and strides {t.stride()} leaves gaps in "
                                     "memory or repeats elements")
        if self.out is not None:
            for g, o in zip(self.tensors, self.out):
                if not _same_layout(g, o):
                    raise ValueError(f"GradientClipper: an output has another shape or element order than its gradient "
                                     f"({tuple(o.shape)}, {o.stride()} for {tuple(g.shape)}, {g.stride()})")
        every = self.tensors + (self.out or [])
        self.device = every[0].device if every else None
        if any(t.device != self.device for t in every):
            raise RuntimeError("GradientClipper: all tensors must be on the same device")
        if every and not every[0].is_cuda:
            raise RuntimeError("Not implemented on the CPU")
        self._shared = self._find_shared()
        # (the kernels work on the memory the tensors have NOW; these aliases keep it alive whatever becomes of the tensors)
        self._memory = [t.detach() for t in every]
        self._arrays = [(ctypes.c_int64 * len(self.tensors))(*[t.numel() for t in self.tensors])]
        self._numel = ctypes.addressof(self._arrays[0])
        self._src = self._lay_out(self.tensors)
        self._dst = self._src if self.out is None else self._lay_out(self.out)

    def _lay_out(self, group):
        """addresses of the host arrays (pointers, types) of a list of tensors"""
        arrays = ((ctypes.c_void_p * len(group))(*[t.data_ptr() for t in group]),
                  (ctypes.c_uint8 * len(group))(*[_GRAD_TYPES[t.dtype] for t in group]))
        self._arrays += arrays
        return tuple(ctypes.addressof(x) for x in arrays)

    def _find_shared(self):
        """a message if `clip` would write memory that it reads for another element, else None (the norm may count twice)"""
        written = self.tensors if self.out is None else self.out
        spans = [(*s, True) for s in _spans(written)]
        if self.out is not None:
            # (an output that IS its gradient, of the same type, is in place; any other overlap is not)
            spans += [(*s, False) for s in _spans(self.tensors)
                      if not (self.out[s[2]].data_ptr() == s[0] and self.out[s[2]].dtype == self.tensors[s[2]].dtype)]
            spans.sort()
        end, wrote = 0, False
        for begin, stop, _, writes in spans:
            if begin < end and (writes or wrote):
                return "GradientClipper: two of the tensors share memory, clip() would scale it twice or read what it has written"
            if stop > end:
                end, wrote = stop, writes if begin >= end else writes or wrote
            else:
                wrote = wrote or writes
        return None

    def _check(self, grad_scale, norm_type):
        if float(norm_type) not in _ORDERS:
            raise ValueError(f"norm_type must be 1, 2 or infinity (got {norm_type})")
        if not 0.0 < grad_scale < math.inf:
            raise ValueError(f"grad_scale must be positive and finite (got {grad_scale})")

    def _norm(self, norm_type, grad_scale):
        if roofline.active:
            roofline.add(roofline.tensor_bytes(*self.tensors))
        return _lib.operators().grad_norm(*self._src, self._numel, len(self.tensors), _ORDERS[float(norm_type)], grad_scale, self.device.index)

    def norm(self, norm_type=2.0, grad_scale=1.0):
        """the global norm, a float32 scalar on the device (no synchronisation)"""
        self._check(grad_scale, norm_type)
        if not self.tensors:
            return torch.tensor(0.0)
        return self._norm(norm_type, grad_scale)[0]

    def clip(self, max_norm, norm_type=2.0, grad_scale=1.0, error_if_nonfinite=False):
        """out = grad_scale * min(1, max_norm / (norm + 1e-6)) * gradient for every tensor; -> the norm (float32, on the device).
        error_if_nonfinite: raises for a norm that is infinite or NaN, before anything is written (waits for the device)."""
        max_norm = float(max_norm)
        if not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative (got {max_norm})")
        self._check(grad_scale, norm_type)
        if self._shared:
            raise ValueError(self._shared)
        if not self.tensors:
            return torch.tensor(0.0)
        norm, work = self._norm(norm_type, grad_scale)
        if error_if_nonfinite and not bool(torch.isfinite(norm)):
            raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients is non-finite, so it cannot be clipped.")
        _lib.operators().grad_clip(*self._src, *self._dst, self._numel, len(self.tensors), max_norm, grad_scale, work)
        if roofline.active:
            roofline.add(roofline.tensor_bytes(*self.tensors, *(self.tensors if self.out is None else self.out)))
        torch.autograd.graph.increment_version(self.tensors if self.out is None else self.out)
        return norm


def _gradients(parameters):
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    return [p.grad for p in parameters if p.grad is not None]


def grad_norm(tensors, norm_type=2.0, grad_scale=1.0):
    """global norm over a tensor or a list of tensors (see GradientClipper), a float32 scalar on the device"""
    return GradientClipper(tensors).norm(norm_type, grad_scale)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, grad_scale=1.0):
    """clips the gradients of the parameters to a global norm in place, as torch.nn.utils.clip_grad_norm_; -> the norm.  Parameters
    without a gradient are skipped.  The lists are laid out in every call (754 gradients: 0.8 ms of host time, the kernels 0.37 ms); a loop
    whose gradients stay in place keeps a GradientClipper instead (0.07 ms)."""
    return GradientClipper(_gradients(parameters)).clip(max_norm, norm_type, grad_scale, error_if_nonfinite)
