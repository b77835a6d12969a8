"""Clip + AdamW on the model's flat buffers (``FlatAdamW``, two kernel launches per step) and over any number of separate
tensors (``MultiAdamW``, ``clip_grad_norm_``, ``grad_norm``).

Same update rule and defaults as the reference's optimizer
(torch.optim.AdamW(model.parameters(), lr), vae/training/train.py:310: betas (0.9, 0.999),
eps 1e-8, weight_decay 0.01) preceded by clip_grad_norm_(max_norm) (train.py:336)."""
from __future__ import annotations

import copy
import ctypes
import threading

import numpy as np
import torch
from torch.autograd.graph import increment_version
from torch.optim.optimizer import _global_optimizer_post_hooks as _global_post_hooks
from torch.optim.optimizer import _global_optimizer_pre_hooks as _global_pre_hooks

from . import _lib


class FlatAdamW:
    def __init__(self, model, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01):
        if model.flat_params is None:
            raise RuntimeError("move the model to the GPU before creating the optimizer")
        self.model = model
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), betas, float(eps), float(weight_decay)
        self.exp_avg = torch.zeros_like(model.flat_params)
        self.exp_avg_sq = torch.zeros_like(model.flat_params)
        self.step_count = 0
        n = model.flat_params.numel()
        self._partial = torch.empty(_lib.call("vae_adamw_grid", n), device=model.flat_params.device)
        self.grad_norm = torch.zeros(1, device=model.flat_params.device)   # pre-clip norm of the last step
        self.grad_mul = 1.0          # gradients are multiplied by this first (1/world_size after a SUM all-reduce)

    def zero_grad(self, set_to_none=True):
        for p in self.model.parameters():
            p.grad = None

    def step_flat(self, model=None, max_norm=1.0, elbo=None):
        """clip_grad_norm_(max_norm) + AdamW step on model.flat_grads, then refresh the bf16 weights.
        elbo: the arguments of vae_elbo_combine (recon partials, count, KL partials, count, kl_weight, 1/batch, out3);
        the step's loss sums are then finished inside the first launch here instead of in a launch of their own."""
        m = self.model
        _lib.check_device(m.flat_params)
        self.step_count += 1
        e = elbo if elbo is not None else (None, 0, None, 0, 0.0, 0.0, None)
        _lib.call("vae_adamw_clip_step_elbo", m.flat_params.data_ptr(), m.flat_grads.data_ptr(), self.exp_avg.data_ptr(),
                  self.exp_avg_sq.data_ptr(), m.flat_params.numel(), self._partial.data_ptr(), float(self.grad_mul),
                  float(max_norm if max_norm is not None else 0.0), self.lr, self.betas[0], self.betas[1], self.eps,
                  self.weight_decay, self.step_count, self.grad_norm.data_ptr(), e[0], int(e[1]), e[2], int(e[3]),
                  float(e[4]), float(e[5]), e[6], _lib.current_stream())
        m.repack_weights()

    def step(self):
        """optimizer.step() on parameters' .grad (no clipping): gathers .grad into flat_grads first."""
        m = self.model
        for p, view in zip(m._ordered_params(), m.grad_views()):
            if p.grad is None:
                view.zero_()
            elif p.grad.data_ptr() != view.data_ptr():
                view.copy_(p.grad)
        self.step_flat(m, max_norm=None)


# ------------------------------------------------------------------------------------ many separate tensors
_TYPES = {torch.float32: 0, torch.bfloat16: 1}
_JOB = np.dtype([("param", np.uint64), ("grad", np.uint64), ("n", np.int64), ("block", np.uint32), ("slot", np.uint32),
                 ("flags", np.uint32), ("reserved", np.uint32)])       # struct vae_mt_tensor


def _dense(t):
    """whether t's elements fill one run of memory without gaps or overlaps, in whatever order of the dims"""
    if t.is_contiguous():
        return True
    step = 1
    for st, size in sorted((st, size) for st, size in zip(t.stride(), t.shape) if size != 1):
        if st != step:
            return False
        step *= size
    return True


class _Tables(threading.local):
    """Each thread's table for the calls that keep none: the library has read it when a call returns."""
    jobs, addr = np.empty(0, _JOB), 0

    def room(self, n):
        if len(self.jobs) < n:
            self.jobs = np.empty(max(64, 2 * n), _JOB)
            self.addr = self.jobs.ctypes.data
        return self.jobs


_tables = _Tables()


def _grad_jobs(parameters, who, write):
    """(address of the table of the parameters' gradients, their number, what has to live until the launch).  ``write``: they are
    written in place"""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    first = None
    for p in params:
        first = p.grad
        if first is not None:
            break
    if first is None:
        return 0, 0, None
    _lib.check_device(first)
    jobs = _tables.room(len(params))
    n = _lib.host().collect_grads(params, jobs, first.get_device(), write)
    return (_tables.addr, n, first) if n >= 0 else _grad_jobs_general(params, first, who, write)


@torch.no_grad()
def _grad_jobs_general(params, first, who, write):
    grads = [p.grad for p in params if p.grad is not None]
    for g in grads:
        if g.layout is not torch.strided or g.dtype not in _TYPES:
            raise TypeError(f"{who}: a gradient is {g.layout} {g.dtype}; dense fp32 and bf16 gradients are supported")
        if g.device != first.device:
            raise RuntimeError(f"{who}: the gradients live on {first.device} and {g.device}")
    if write:
        for g in grads:
            if not _dense(g):
                raise ValueError(f"{who}: a gradient of shape {tuple(g.shape)} with strides {g.stride()} has gaps or overlaps and cannot be written "
                                 "in place")
        spans = sorted((g.data_ptr(), g.data_ptr() + g.nbytes) for g in grads if g.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError(f"{who}: two of the gradients are the same memory, wholly or in part")
        increment_version(grads)
    else:
        grads = [g if _dense(g) else g.contiguous() for g in grads]
    jobs = np.zeros(len(grads), _JOB)
    jobs["grad"] = [g.data_ptr() for g in grads]
    jobs["n"] = [g.numel() for g in grads]
    jobs["flags"] = [_lib.MT_GRAD_BF16 if g.dtype is torch.bfloat16 else 0 for g in grads]
    return jobs.ctypes.data, len(grads), (jobs, grads)


def grad_norm(parameters):
    """Global L2 norm of the parameters' gradients as a 0-dim fp32 tensor: one launch per 256 tensors and one that finishes the
    sum.  Squares and sums in 64 bits, in a fixed order."""
    jobs, n, keep = _grad_jobs(parameters, "grad_norm", False)
    if n == 0:
        return torch.zeros(())
    partial = torch.empty(_lib.call("vae_multi_partials", n), dtype=torch.float64, device="cuda")
    out = torch.empty((), device="cuda")
    _lib.call("vae_multi_grad_norm", jobs, n, partial.data_ptr(), 1.0, out.data_ptr(), _lib.current_stream())
    return out


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ (vae/training/train.py:336) for fp32 and bf16 gradients of any number of tensors: scales
    them in place by ``min(1, max_norm / (norm + 1e-6))`` and returns the norm before that as a 0-dim fp32 tensor.  Two launches per
    256 tensors, no host synchronisation unless ``error_if_nonfinite``."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm={max_norm} must not be negative or NaN")
    if norm_type != 2.0 and float(norm_type) != 2.0:
        raise ValueError(f"clip_grad_norm_: norm_type={norm_type}; only the L2 norm is computed")
    if error_if_nonfinite:
        parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
        norm = grad_norm(parameters)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"clip_grad_norm_: the gradients' norm is {norm.item()}, so it cannot be clipped")
    jobs, n, keep = _grad_jobs(parameters, "clip_grad_norm_", True)
    if n == 0:
        return torch.zeros(())
    partial = torch.empty(_lib.call("vae_multi_partials", n), dtype=torch.float64, device="cuda")
    out = torch.empty((), device="cuda")
    _lib.call("vae_multi_clip", jobs, n, partial.data_ptr(), 1.0, max_norm, out.data_ptr(), _lib.current_stream())
    return out


class _GroupState:
    """One param group's tensors and state: where each tensor's blocks start, the flat state buffers, and the tables handed to
    the library."""

    def __init__(self, params, state_bits):
        self.params = list(params)
        self.device = params[0].device
        self.home = _lib.current_stream()
        self.bits = state_bits
        self.shapes = [tuple(p.shape) for p in params]
        self.strides = [p.stride() for p in params]
        self.contiguous = [p.is_contiguous() for p in params]
        self.dtypes = [p.dtype for p in params]
        self.nbytes = [p.nbytes for p in params]
        self.n = [p.numel() for p in params]
        self.start, at = [], 0
        for n in self.n:
            self.start.append(at)
            at += -(-n // _lib.MT_BLOCK)
        self.nblocks = at
        elems = max(at, 1) * _lib.MT_BLOCK
        z = lambda *shape, dtype=torch.float32: torch.zeros(*shape, dtype=dtype, device=self.device)  # noqa: E731
        kind = torch.float32 if state_bits == 32 else torch.uint8
        self.exp_avg, self.exp_avg_sq = z(elems, dtype=kind), z(elems, dtype=kind)
        self.bases = z(max(at, 1), 2, dtype=torch.int16) if state_bits == 8 else None
        self.remainder = z(elems, dtype=torch.int16) if torch.bfloat16 in self.dtypes else None
        self.steps = z(len(params), dtype=torch.int64)
        self.scalars = z(len(params), 8)
        self.jobs = np.zeros(len(params), _JOB)
        self.jobs_addr = self.jobs.ctypes.data
        self.index = self.device.index
        self.param_flags = [_lib.MT_PARAM_BF16 if d is torch.bfloat16 else 0 for d in self.dtypes]
        self.layout = np.stack([self.n, self.start, np.arange(len(params)), self.param_flags], 1).astype(np.int64)
        self.layout[:, 3] |= [0 if c else _lib.MT_STRIDED for c in self.contiguous]
        self.c = _lib.MtGroup(state_bits=state_bits, nslots=len(params), exp_avg=self.exp_avg.data_ptr(),
                              exp_avg_sq=self.exp_avg_sq.data_ptr(), bases=_lib.ptr(self.bases), remainder=_lib.ptr(self.remainder),
                              nblocks=self.nblocks, steps=self.steps.data_ptr(), scalars=self.scalars.data_ptr())

    def used_on(self, stream):
        """the allocator may not hand the state on before this stream's work on it is done"""
        if stream != self.home:
            cur = torch.cuda.current_stream()
            for b in (self.exp_avg, self.exp_avg_sq, self.bases, self.remainder, self.steps, self.scalars):
                if b is not None:
                    b.record_stream(cur)

    def check_param(self, k):
        """a parameter is read and written through its address: it still has to be what the state was laid out for"""
        p = self.params[k]
        if (p.nbytes != self.nbytes[k] or p.dtype is not self.dtypes[k] or p.device != self.device
                or not (p.is_contiguous() if self.contiguous[k] else p.stride() == self.strides[k])):
            raise RuntimeError(f"MultiAdamW: parameter {k} was {self.shapes[k]} {self.dtypes[k]} on {self.device} and is now {tuple(p.shape)} "
                               f"{p.dtype} on {p.device} (or its strides changed): make a new optimizer after moving or casting the model")
        return p

    def collect(self):
        """fills the table of the tensors that have a gradient; returns their number and what has to live until the launch"""
        n = _lib.host().collect_step(self.params, self.jobs, self.layout, self.index)
        if n >= 0:
            self.c.tensors, self.c.count = self.jobs_addr, n
            return n, None
        ptrs, gptrs, flags, keep, live, at = [], [], [], [], [], []
        for k, p in enumerate(self.params):
            g = p.grad
            if g is None:
                continue
            self.check_param(k)
            if g.layout is not torch.strided or g.dtype not in _TYPES:
                raise TypeError(f"MultiAdamW: the gradient of parameter {k} is {g.layout} {g.dtype}; dense fp32 and bf16 gradients are supported")
            if g.device != self.device or g.shape != p.shape:
                raise RuntimeError(f"MultiAdamW: the gradient of parameter {k} is {tuple(g.shape)} on {g.device}, the parameter "
                                   f"{self.shapes[k]} on {self.device}")
            if not (g.is_contiguous() if self.contiguous[k] else g.stride() == self.strides[k]):
                with torch.no_grad():
                    g = torch.empty_like(p, dtype=g.dtype).copy_(g)       # into the parameter's order of elements
                keep.append(g)
            ptrs.append(p.data_ptr())
            gptrs.append(g.data_ptr())
            flags.append(self.param_flags[k] | (_lib.MT_GRAD_BF16 if g.dtype is torch.bfloat16 else 0))
            live.append(p)
            at.append(k)
        n = len(live)
        jobs = np.zeros(max(n, 1), _JOB)
        jobs["param"][:n], jobs["grad"][:n], jobs["flags"][:n] = ptrs, gptrs, flags
        jobs["n"][:n], jobs["block"][:n], jobs["slot"][:n] = self.layout[at, 0], self.layout[at, 1], self.layout[at, 2]
        keep.append(jobs)
        self.c.tensors, self.c.count = jobs.ctypes.data, n
        increment_version(live)      # written through their addresses: whoever watches the version counters has to see it
        return n, keep

    def view(self, flat, k):
        """element run k of a buffer in the state's layout, in the parameter's shape"""
        run = flat[self.start[k] * _lib.MT_BLOCK:self.start[k] * _lib.MT_BLOCK + self.n[k]]
        return run.view(self.shapes[k]) if self.contiguous[k] else torch.as_strided(run, self.shapes[k], self.strides[k], run.storage_offset())

    def run(self, flat, k):
        return flat[self.start[k] * _lib.MT_BLOCK:self.start[k] * _lib.MT_BLOCK + self.n[k]]

    def rows(self, k):
        return slice(self.start[k], self.start[k] + -(-self.n[k] // _lib.MT_BLOCK))


# keys of a saved param group that stay as they are here: the tensors, the moments' width, and torch's choices among its own forms
_NOT_LOADED = {"params", "state_bits", "amsgrad", "maximize", "foreach", "fused", "capturable", "differentiable", "decoupled_weight_decay"}


class MultiAdamW(torch.optim.Optimizer):
    """AdamW over any number of separate fp32 or bf16 tensors, with the gradient clip of the loop in the same pass.

    torch.optim.AdamW's rule and defaults (vae/training/train.py:310) and its interface: param groups with their own ``lr``, ``betas``,
    ``eps``, ``weight_decay``, learning-rate schedulers, ``state_dict``s that interchange with torch's in both directions (32-bit
    moments), parameters without a gradient left alone.  All arithmetic is in 32 bits; step counts live on the device.

    ``state_bits=8`` (also per group) holds both moments in 8 bits, 2 bytes a parameter instead of 8: blocks of 256 elements, 8 levels per
    octave, rounded with a dither over the steps (see csrc/multi_optim.hip).  A bf16 parameter keeps a 16-bit remainder with which it is a
    32-bit master; writing the parameter from outside needs nothing.

    ``step(max_norm=1.0)`` is ``clip_grad_norm_(params, 1.0); step()`` without the pass that rewrites the gradients: two launches
    per group and 256 tensors (a small step without a clip: one); the norm before the clip is in ``grad_norm``.  Gradients are multiplied by ``grad_mul`` first
    (1/world_size after a SUM all-reduce).

    A step can be captured into a graph: step counts advance when it is replayed.  A float ``lr`` is recorded as it is; give an fp32
    device tensor as ``lr`` to change it between replays."""

    def __init__(self, params, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32):
        self._groups, self._spans = [], []
        self.grad_mul = 1.0
        self.grad_norm = None
        self._partial, self._old_partials = None, []
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    @staticmethod
    def _check_group(g):
        lr, (b1, b2) = g["lr"], g["betas"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype is not torch.float32 or not lr.is_cuda:
                raise ValueError("MultiAdamW: a tensor lr must be one fp32 element on the GPU")
        elif not float(lr) >= 0.0:
            raise ValueError(f"MultiAdamW: lr={lr} must not be negative")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"MultiAdamW: betas={g['betas']} must be in [0, 1)")
        if not float(g["eps"]) >= 0.0 or not float(g["weight_decay"]) >= 0.0:
            raise ValueError(f"MultiAdamW: eps={g['eps']} and weight_decay={g['weight_decay']} must not be negative")
        if g["state_bits"] not in (8, 32):
            raise ValueError(f"MultiAdamW: state_bits={g['state_bits']} must be 8 or 32")
        if g["state_bits"] == 8 and float(g["eps"]) < _lib.MT_MIN_EPS8:
            raise ValueError(f"MultiAdamW: eps={g['eps']}: 8-bit moments need at least {_lib.MT_MIN_EPS8}")

    def add_param_group(self, param_group):
        if len(self._groups) >= _lib.MT_MAX_GROUPS:
            raise ValueError(f"MultiAdamW: more than {_lib.MT_MAX_GROUPS} param groups")
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
            params = group["params"]
            if not params:
                raise ValueError("MultiAdamW: a param group is empty")
            if len(params) > _lib.MT_MAX_TENSORS:
                raise ValueError(f"MultiAdamW: more than {_lib.MT_MAX_TENSORS} tensors in a param group")
            spans = list(self._spans)
            for k, p in enumerate(params):
                if p.dtype not in _TYPES or p.layout is not torch.strided:
                    raise TypeError(f"MultiAdamW: parameter {k} is {p.layout} {p.dtype}; dense fp32 and bf16 parameters are supported")
                if not p.is_cuda:
                    raise RuntimeError("MultiAdamW runs on an MI355X only: move the model to 'cuda' before creating the optimizer")
                first = self._groups[0].device if self._groups else params[0].device
                if p.device != first:
                    raise RuntimeError(f"MultiAdamW: parameters live on {first} and {p.device}: one optimizer per GPU")
                if not _dense(p):
                    raise ValueError(f"MultiAdamW: parameter {k} of shape {tuple(p.shape)} with strides {p.stride()} has gaps or overlaps")
                if p.numel():
                    spans.append((p.data_ptr(), p.data_ptr() + p.nbytes))
            spans.sort()
            if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
                raise ValueError("MultiAdamW: two parameters share memory")
            _lib.check_device(params[0])
            self._groups.append(_GroupState(params, int(group["state_bits"])))
            self._spans = spans
        except Exception:
            self.param_groups.pop()
            raise
        n = _lib.call("vae_multi_partials", sum(len(g.params) for g in self._groups))
        self._old_partials.append(self._partial)       # a graph that captured a step goes on using the one it captured
        self._partial = torch.empty(n, dtype=torch.float64, device=params[0].device)
        if self.grad_norm is None:
            self.grad_norm = torch.zeros(1, device=params[0].device)
        self._c = (_lib.MtGroup * len(self._groups))()
        self._home = _lib.current_stream()

    def holds(self, parameters):
        """whether these are exactly the tensors it steps"""
        return {id(p) for p in parameters} == {id(p) for st in self._groups for p in st.params}

    def holds_gradients(self, parameters):
        """whether those of these parameters that have a gradient are exactly those that a step takes now (frozen ones do not matter)"""
        return {id(p) for p in parameters if p.grad is not None} == {id(p) for st in self._groups for p in st.params if p.grad is not None}

    def __getstate__(self):
        raise TypeError("MultiAdamW holds device buffers and is not copied or pickled: save state_dict() and load it into a new one")

    def step(self, closure=None, max_norm=None):
        """One step; with ``max_norm`` the gradients' global norm (over all groups) is clipped to it first.  ``closure``, as in torch,
        recomputes the loss and its gradients; its value is returned."""
        args, kwargs = (self, closure), {"max_norm": max_norm}
        if _global_pre_hooks or self._optimizer_step_pre_hooks:
            for hook in (*_global_pre_hooks.values(), *self._optimizer_step_pre_hooks.values()):
                args, kwargs = hook(self, args, kwargs) or (args, kwargs)
            closure, max_norm = args[1] if len(args) > 1 else kwargs.get("closure"), kwargs.get("max_norm")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._step(max_norm)
        if _global_post_hooks or self._optimizer_step_post_hooks:
            for hook in (*self._optimizer_step_post_hooks.values(), *_global_post_hooks.values()):
                hook(self, args, kwargs)
        return loss

    step.hooked = True      # torch would wrap it into a profiler range, 14 us of host time a step

    def _step(self, max_norm):
        clip = -1.0 if max_norm is None else float(max_norm)
        if max_norm is not None and not clip >= 0.0:
            raise ValueError(f"MultiAdamW: max_norm={max_norm} must not be negative or NaN")
        _lib.check_device(self.grad_norm)
        keep, total, same = [], 0, _lib.host().same_tensors
        for g, st in zip(self.param_groups, self._groups):
            if not same(g["params"], st.params):
                raise RuntimeError("MultiAdamW: a param group's list of tensors was changed")
            self._check_group(g)
            if g["state_bits"] != st.bits:
                raise RuntimeError(f"MultiAdamW: state_bits of a group was changed from {st.bits} to {g['state_bits']}")
            if isinstance(g["lr"], torch.Tensor) and g["lr"].device != st.device:
                raise RuntimeError(f"MultiAdamW: lr lives on {g['lr'].device}, the parameters on {st.device}")
        for k, (g, st) in enumerate(zip(self.param_groups, self._groups)):
            n, kept = st.collect()
            total += n
            keep.append(kept)
            c, lr = st.c, g["lr"]
            c.lr, c.lr_dev = (0.0, lr.data_ptr()) if isinstance(lr, torch.Tensor) else (float(lr), None)
            (c.beta1, c.beta2), c.eps, c.weight_decay = g["betas"], g["eps"], g["weight_decay"]
            self._c[k] = c
        if total == 0:
            if clip >= 0.0:
                self.grad_norm.zero_()
            return
        stream = _lib.current_stream()
        if stream != self._home or len(self._groups) > 1:
            for st in self._groups:
                st.used_on(stream)
        if stream != self._home:
            self._partial.record_stream(torch.cuda.current_stream())
            self.grad_norm.record_stream(torch.cuda.current_stream())
        _lib.call("vae_multi_adamw_step", ctypes.byref(self._c), len(self._groups), self._partial.data_ptr(), float(self.grad_mul), clip,
                  self.grad_norm.data_ptr() if clip >= 0.0 else None, stream)

    # -------------------------------------------------------------------------------- state
    def flat_moments(self, group=0):
        """(exp_avg, exp_avg_sq) of a group in the state's layout: every tensor starts on a multiple of 256 elements, the
        padding is zero.  32-bit moments: the state itself; 8-bit ones: their values in bf16, which holds them exactly."""
        st = self._groups[group]
        if st.bits == 32:
            return st.exp_avg, st.exp_avg_sq
        _lib.check_device(st.exp_avg)
        st.used_on(_lib.current_stream())
        m, v = (torch.empty(st.exp_avg.numel(), dtype=torch.bfloat16, device=st.device) for _ in range(2))
        self._unpack(st, st.exp_avg, st.exp_avg_sq, st.bases, m, v)
        return m, v

    @staticmethod
    def _unpack(st, qm, qv, bases, m, v):
        _lib.call("vae_moments8_unpack", qm.data_ptr(), qv.data_ptr(), bases.data_ptr(), m.data_ptr(), v.data_ptr(), bases.shape[0],
                  _lib.M8_INF | (_lib.M8_BF16 if m.dtype is torch.bfloat16 else 0), _lib.current_stream())

    def flat_master(self, group=0):
        """32-bit values of a group's parameters in the state's layout: a bf16 parameter's master, an fp32 parameter itself"""
        st = self._groups[group]
        _lib.check_device(st.exp_avg)
        st.used_on(_lib.current_stream())
        # every block is some tensor's and is written whole
        out = (torch.empty if st.nblocks else torch.zeros)(max(st.nblocks, 1) * _lib.MT_BLOCK, device=st.device)
        jobs = _tables.room(len(st.params))
        addr = _tables.addr
        if _lib.host().collect_params(st.params, jobs, st.layout, st.index) < 0:
            jobs = np.zeros(len(st.params), _JOB)
            addr = jobs.ctypes.data
            for k in range(len(st.params)):
                st.check_param(k)
            jobs["n"], jobs["block"], jobs["slot"] = st.layout[:, 0], st.layout[:, 1], st.layout[:, 2]
            jobs["param"] = [p.data_ptr() for p in st.params]
            jobs["grad"] = jobs["param"]       # not read
            jobs["flags"] = [f * (_lib.MT_PARAM_BF16 | _lib.MT_GRAD_BF16) for f in st.param_flags]
        _lib.call("vae_multi_master", addr, len(st.params), _lib.ptr(st.remainder), out.data_ptr(), st.nblocks, _lib.current_stream())
        return out

    @torch.no_grad()
    def state_dict(self):
        """torch's layout: ``state[i]`` of the i-th parameter with ``step``, ``exp_avg``, ``exp_avg_sq`` in the parameter's shape (views
        of the live state, as in torch; ``step`` is a copy).  8-bit moments: the codes ``exp_avg_q``, ``exp_avg_sq_q`` in the order of the
        parameter's memory and the blocks' ``exp_avg_base``, ``exp_avg_sq_base`` (int16).  bf16 parameters: ``remainder`` too."""
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        state, groups, at = {}, [], 0
        for g, st in zip(self.param_groups, self._groups):
            steps = st.steps.tolist()
            for k in range(len(st.params)):
                e = {"step": torch.tensor(float(steps[k]), dtype=torch.float32 if steps[k] < 1 << 24 else torch.float64)}
                if st.bits == 32:
                    e["exp_avg"], e["exp_avg_sq"] = st.view(st.exp_avg, k), st.view(st.exp_avg_sq, k)
                else:
                    e["exp_avg_q"], e["exp_avg_sq_q"] = st.run(st.exp_avg, k), st.run(st.exp_avg_sq, k)
                    e["exp_avg_base"], e["exp_avg_sq_base"] = (st.bases[st.rows(k), j] for j in (0, 1))
                    e["stride"] = st.strides[k]
                if st.dtypes[k] is torch.bfloat16:
                    e["remainder"] = st.view(st.remainder, k)
                state[at + k] = e
            groups.append({**{key: x for key, x in g.items() if key != "params"}, "params": list(range(at, at + len(st.params)))})
            at += len(st.params)
        state_dict = {"state": state, "param_groups": groups}
        for hook in self._optimizer_state_dict_post_hooks.values():
            new = hook(self, state_dict)
            state_dict = state_dict if new is None else new
        return state_dict

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Takes what ``state_dict`` gives, of this class or of torch.optim.AdamW, and converts between moments in 32 and in 8 bits
        (to nearest) where the two differ.  A parameter without an entry starts from zero.  The groups' other keys (a scheduler's, the user's)
        are taken over too, the moments' width is not.  Nothing is written if an entry does not fit."""
        state_dict = dict(state_dict)       # a hook may exchange its parts
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            new = hook(self, state_dict)
            state_dict = state_dict if new is None else new
        groups, state = state_dict["param_groups"], state_dict["state"]
        if [len(g["params"]) for g in groups] != [len(st.params) for st in self._groups]:
            raise ValueError("MultiAdamW: the state_dict's param groups have other lengths")
        owned = {b.untyped_storage().data_ptr() for st in self._groups for b in (st.exp_avg, st.exp_avg_sq, st.bases, st.remainder) if b is not None}
        entries = []
        for saved, st in zip(groups, self._groups):
            # what state_dict() gave are views of the buffers written below: copied, because an entry may go to another tensor's place
            row = [{key: x.clone() if isinstance(x, torch.Tensor) and x.is_cuda and x.untyped_storage().data_ptr() in owned else x
                    for key, x in state.get(i, {}).items()} for i in saved["params"]]
            for k, e in enumerate(row):
                self._check_entry(st, k, e)
            for key, limit in (("exp_avg_base", 0x7F7 - 127), ("exp_avg_sq_base", 0x7F7 - 254)):       # + the largest code: fp32's last level
                bases = [e[key].reshape(-1) for e in row if "exp_avg_q" in e]
                if sum(b.numel() for b in bases):
                    low, high = torch.stack(torch.cat(bases).aminmax()).tolist()
                    if low < 0 or high > limit:
                        raise ValueError(f"MultiAdamW: {key} from {low} to {high}: above {limit} they are no levels of finite numbers")
            entries.append(row)
        merged = []
        for saved, g in zip(groups, self.param_groups):
            if saved.get("amsgrad") or saved.get("maximize"):
                raise ValueError("MultiAdamW: the state_dict is of an AdamW with amsgrad or maximize, which is another rule")
            new = {key: copy.deepcopy(x) for key, x in saved.items() if key not in _NOT_LOADED}
            if "lr" in new:
                new["lr"] = float(new["lr"])
            if "betas" in new:
                new["betas"] = tuple(float(b) for b in new["betas"])
            self._check_group({**g, **new})
            merged.append(new)
        for new, g, st, row in zip(merged, self.param_groups, self._groups, entries):
            st.used_on(_lib.current_stream())
            for key, x in new.items():
                if key in ("lr", "initial_lr") and isinstance(g.get(key), torch.Tensor):
                    g[key].fill_(x)       # a captured step reads this tensor
                else:
                    g[key] = x
            st.steps.copy_(torch.tensor([int(e.get("step", 0)) for e in row], dtype=torch.int64))       # checked above
            if st.remainder is not None:
                st.remainder.zero_()
                have = [k for k, e in enumerate(row) if "remainder" in e and st.dtypes[k] is torch.bfloat16]
                if have:
                    src = [row[k]["remainder"] for k in have]
                    torch._foreach_copy_([st.view(st.remainder, k) for k in have],
                                         [x if tuple(x.shape) == st.shapes[k] else x.reshape(st.shapes[k]) for k, x in zip(have, src)])
            self._load_moments(st, row)
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    @staticmethod
    def _check_entry(st, k, e):
        def fits(key, numel):
            if key in e and e[key].numel() != numel:
                raise ValueError(f"MultiAdamW: {key} of parameter {k} has {e[key].numel()} elements where {numel} are wanted")
        step = float(e.get("step", 0))
        if not 0.0 <= step < 2.0 ** 62 or step != int(step):
            raise ValueError(f"MultiAdamW: the step count of parameter {k} is {step}")
        if ("exp_avg" in e) != ("exp_avg_sq" in e) or ("exp_avg" in e and "exp_avg_q" in e):
            raise ValueError(f"MultiAdamW: the entry of parameter {k} has {sorted(e)}")
        for key in e:
            if key in ("exp_avg", "exp_avg_sq", "exp_avg_q", "exp_avg_sq_q", "remainder"):
                fits(key, st.n[k])
        if "remainder" in e and st.dtypes[k] is torch.bfloat16 and e["remainder"].dtype is not torch.int16:
            raise TypeError(f"MultiAdamW: the remainder of parameter {k} is {e['remainder'].dtype}, not int16")
        if "exp_avg_q" in e:
            for key in ("exp_avg_sq_q", "exp_avg_base", "exp_avg_sq_base"):
                if key not in e:
                    raise ValueError(f"MultiAdamW: the entry of parameter {k} has no {key}")
            rows = st.rows(k)
            for key in ("exp_avg_base", "exp_avg_sq_base"):
                fits(key, rows.stop - rows.start)
                if e[key].dtype.is_floating_point:
                    raise TypeError(f"MultiAdamW: {key} of parameter {k} is {e[key].dtype}, not of whole numbers")
            if e["exp_avg_q"].dtype is not torch.uint8 or e["exp_avg_sq_q"].dtype is not torch.uint8:
                raise TypeError(f"MultiAdamW: the codes of parameter {k} are not uint8")
            if "stride" in e and st.n[k] > 1 and (len(e["stride"]) != len(st.shapes[k]) or any(
                    a != b and size != 1 for a, b, size in zip(e["stride"], st.strides[k], st.shapes[k]))):
                raise ValueError(f"MultiAdamW: the codes of parameter {k} are in the order of strides {tuple(e['stride'])}, the parameter has {st.strides[k]}")
        elif "exp_avg" in e:
            for key in ("exp_avg", "exp_avg_sq"):
                if tuple(e[key].shape) != st.shapes[k]:
                    raise ValueError(f"MultiAdamW: {key} of parameter {k} has shape {tuple(e[key].shape)}, the parameter {st.shapes[k]}")

    def _load_moments(self, st, row):
        _lib.check_device(st.exp_avg)
        eight, full = [k for k, e in enumerate(row) if "exp_avg_q" in e], [k for k, e in enumerate(row) if "exp_avg" in e]
        scratch = lambda dtype: (torch.zeros_like(st.exp_avg, dtype=dtype), torch.zeros_like(st.exp_avg, dtype=dtype))  # noqa: E731

        def fill(dst, view, which, keys):
            if which:
                for buf, key in zip(dst, keys):
                    to, src = [view(buf, k) for k in which], [row[k][key] for k in which]
                    torch._foreach_copy_(to, [x if x.shape == t.shape else x.reshape(t.shape) for x, t in zip(src, to)])
        if st.bits == 8:
            q, bases = (st.exp_avg, st.exp_avg_sq), st.bases
            if full:
                f32 = scratch(torch.float32)
                fill(f32, st.view, full, ("exp_avg", "exp_avg_sq"))
                f32[0].masked_fill_(f32[1].isnan(), float("nan"))       # alone in exp_avg_sq it would be taken for infinity
                _lib.call("vae_moments8_pack", f32[0].data_ptr(), f32[1].data_ptr(), q[0].data_ptr(), q[1].data_ptr(), bases.data_ptr(),
                          bases.shape[0], _lib.current_stream())
            else:
                q[0].zero_(), q[1].zero_(), bases.zero_()
        elif eight:
            q, bases = scratch(torch.uint8), torch.zeros(max(st.nblocks, 1), 2, dtype=torch.int16, device=st.device)
        if eight:
            fill(q, st.run, eight, ("exp_avg_q", "exp_avg_sq_q"))
            rows = slice(0, st.nblocks)
            if len(eight) < len(row):
                rows = torch.cat([torch.arange(st.rows(k).start, st.rows(k).stop) for k in eight]).to(st.device)
            for j, key in enumerate(("exp_avg_base", "exp_avg_sq_base")):
                bases[rows, j] = torch.cat([row[k][key].reshape(-1) for k in eight]).to(device=st.device, dtype=torch.int16)
        if st.bits == 32:
            m = (st.exp_avg, st.exp_avg_sq)
            if eight:
                self._unpack(st, q[0], q[1], bases, *m)
            else:
                m[0].zero_(), m[1].zero_()
            fill(m, st.view, full, ("exp_avg", "exp_avg_sq"))
