"""torch.optim.Adam as the reference configures it (src/SpectralTrainer.py:188: defaults apart from the learning rate)
with the update of all parameter tensors in one launch of libsparc_hip.so (sparc_adam_step), the global gradient norm
over many tensors, and clipping by it, in place (clip_grad_norm_) or on the way into the update (max_grad_norm).  Adam is a
torch Optimizer: param_groups, state_dict and learning-rate schedulers (src/SpectralTrainer.py:189-192) work as with
torch's own."""
from __future__ import annotations

import ctypes
import operator
from array import array

import torch
from torch.autograd.graph import increment_version

from ._lib import AdamTensor, check, lib
from .embedding import DTYPES, refuse_forward_mode
from .graph import launch, require_gpu

MAX_TENSORS = 32


def _dense(t: torch.Tensor) -> bool:
    """Every element once in numel() consecutive places, in any order of the dimensions."""
    at = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != at:
            return False
        at *= size
    return True


_type_of = operator.attrgetter("dtype")
_device_of, _address_of, _size_of = torch.Tensor.get_device, torch.Tensor.data_ptr, torch.Tensor.numel
_is_contiguous = torch.Tensor.is_contiguous


def _dense_on(tensors, device, dense=None) -> bool:
    """All on the device, and contiguous or, with dense, at least passing it."""
    try:
        ok = set(map(_device_of, tensors)) == {device.index}
        return ok and (all(map(_is_contiguous, tensors)) or (dense is not None and all(map(dense, tensors))))
    except RuntimeError:   # a sparse tensor has no strides to ask for
        return False


def _grad_records(grads, device):
    """(the list as the C calls take it, an array of {address, elements, type}: keep it while they run; how many records)."""
    types = list(map(_type_of, grads))
    if not _dense_on(grads, device, _dense) or not DTYPES.keys() >= set(types):
        raise ValueError("the gradients of one norm are dense float32, bfloat16 or float16 tensors on one device")
    codes = [DTYPES[types[0]]] * len(types) if types.count(types[0]) == len(types) else [DTYPES[t] for t in types]
    at, sizes = list(map(_address_of, grads)), list(map(_size_of, grads))
    if len(set(at)) < len(at):
        at, sizes, codes = _each_once(at, sizes, codes)
    return _records(at, sizes, codes), len(at)


def _each_once(at, sizes, codes):
    """The three columns without the empty tensors and those whose memory an earlier one has: two workgroups that scale the
    same elements would race."""
    seen = {}
    for a, n, code in zip(at, sizes, codes):
        if n and seen.setdefault(a, (a, n, code)) != (a, n, code):
            raise ValueError("gradients that overlap in part")
    return [[r[i] for r in seen.values()] for i in range(3)]


def _records(*columns):
    """One int64 array of the columns' entries, record by record."""
    out = [0] * (len(columns) * len(columns[0]))
    for i, column in enumerate(columns):
        out[i::len(columns)] = column
    return array("q", out)


def _norm_of(records, n, device):
    """(partial sums of the squares on the device, how many) of n records."""
    nbytes = lib.sparc_grad_norm_workspace_bytes(n)
    parts = torch.empty(nbytes >> 3, dtype=torch.float64, device=device)
    count = ctypes.c_int64()
    launch("sparc_grad_norm", lib.sparc_grad_norm, device, n, _address(records), parts.data_ptr(), nbytes, ctypes.byref(count))
    return parts, count.value


def _address(records) -> int:
    return records.buffer_info()[0]


def _limit(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must be a number >= 0")
    return max_norm


def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """Scales the gradients of `parameters` (one tensor or several; those without a gradient are passed over, a gradient met
    twice, the same memory, counts once) in place by min(1, max_norm / (norm + 1e-6)), norm being the 2-norm of all of them
    together, and returns the norm before (float32, on their device; nothing synchronises).  float32, bfloat16 and float16
    gradients may be mixed, each dense in memory (any order of the dimensions, views into a bucket too); gradients that overlap
    in part raise.  Sums in float64.  A norm that is not finite leaves what the formula gives; an infinite max_norm never
    clips."""
    max_norm = _limit(max_norm)
    if torch.is_tensor(parameters):
        parameters = (parameters,)
    parameters = list(parameters)
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return torch.zeros((), device=parameters[0].device if parameters else None)
    refuse_forward_mode("clip_grad_norm_", grads)
    device = grads[0].device
    if not grads[0].is_cuda:
        require_gpu(device)
    records, n = _grad_records(grads, device)
    nbytes = lib.sparc_grad_norm_workspace_bytes(n)
    parts = torch.empty(nbytes >> 3, dtype=torch.float64, device=device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    launch("sparc_clip_grad_norm", lib.sparc_clip_grad_norm, device, n, _address(records), max_norm, parts.data_ptr(), nbytes,
           norm.data_ptr())
    increment_version(grads)   # whatever graph has saved one of them refuses to go back through it
    return norm


def _adam_records(params, grads, exp_avgs, exp_avg_sqs, device):
    """(records of the update as the C calls take them; None, or, where parameters share gradients, these once)."""
    n = len(params)
    every = [*params, *grads, *exp_avgs, *exp_avg_sqs]
    refuse_forward_mode("an Adam step", every)
    sizes = list(map(_size_of, every))
    if set(map(_type_of, every)) != {torch.float32} or not _dense_on(every, device) or sizes != sizes[:n] * 4:
        raise ValueError("an Adam step takes contiguous float32 tensors of one device, four of a size")
    at = list(map(_address_of, every))
    once = None
    if len(set(at[n:2 * n])) < n:   # (memory that is written and shared: the library refuses it)
        once = _each_once(at[n:2 * n], sizes[:n], [0] * n)
    return _records(at[:n], at[n:2 * n], at[2 * n:3 * n], at[3 * n:], sizes[:n]), once


def adam_step_(params, grads, exp_avgs, exp_avg_sqs, step: int, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.0, max_grad_norm=None):
    """Update number `step` (from 1) of torch.optim.Adam on lists of tensors, in place: params, exp_avgs and exp_avg_sqs.
    With max_grad_norm the gradients enter as clip_grad_norm_(..., max_grad_norm) would leave them, but are only read
    (once for the norm, once by the update); returns their norm then, None otherwise.  Gradients may be shared, what is written
    may not: it raises where it has memory in common with any other tensor."""
    params = list(params)
    if not (len(params) == len(grads) == len(exp_avgs) == len(exp_avg_sqs)):
        raise ValueError("as many gradients and moments as parameters")
    if not params:
        return None if max_grad_norm is None else torch.zeros(())
    device = params[0].device
    if not params[0].is_cuda:
        require_gpu(device)
    records, once = _adam_records(params, grads, exp_avgs, exp_avg_sqs, device)
    rates = (float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay), int(step))
    norm = None
    if max_grad_norm is None:
        _adam_launches(records, len(params), rates, device)
    else:
        norm = _clipped_step(records, once, len(params), rates, _limit(max_grad_norm), device)
    increment_version([*params, *exp_avgs, *exp_avg_sqs])
    return norm


def _clipped_step(records, once, n, rates, max_norm, device):
    """The update of n records by their own gradients' norm, which is returned."""
    norm = torch.empty((), dtype=torch.float32, device=device)
    if once is not None:
        parts, count = _norm_of(_records(*once), len(once[0]), device)
        launch("sparc_adam_step_clipped", lib.sparc_adam_step_clipped, device, n, _address(records), *rates, parts.data_ptr(), count,
               max_norm, norm.data_ptr())
        return norm
    nbytes = lib.sparc_grad_norm_workspace_bytes(n)
    parts = torch.empty(nbytes >> 3, dtype=torch.float64, device=device)
    launch("sparc_clip_adam_step", lib.sparc_clip_adam_step, device, n, _address(records), *rates, max_norm, parts.data_ptr(), nbytes,
           norm.data_ptr())
    return norm


def _adam_launches(records, n, rates, device):
    size = ctypes.sizeof(AdamTensor)
    if n > MAX_TENSORS:   # nothing moves where a later launch would be refused
        check(lib.sparc_adam_check(n, _address(records)), "sparc_adam_check")
    for a in range(0, n, MAX_TENSORS):
        launch("sparc_adam_step", lib.sparc_adam_step, device, min(MAX_TENSORS, n - a), _address(records) + a * size, *rates)


class Adam(torch.optim.Optimizer):
    """max_grad_norm: clip the gradients of all groups together on their way into the update (they themselves stay as
    they are); grad_norm is then their norm in the latest step, a float32 scalar on the device."""

    grad_norm = None

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.0,
                 max_grad_norm=None):
        if lr < 0 or eps < 0 or not 0 <= betas[0] < 1 or not 0 <= betas[1] < 1 or weight_decay < 0:
            raise ValueError("invalid Adam hyper-parameter")
        if max_grad_norm is not None:
            max_grad_norm = _limit(max_grad_norm)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_grad_norm=max_grad_norm))

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:   # a state written before there was a max_grad_norm
            group.setdefault("max_grad_norm", self.defaults.get("max_grad_norm"))

    def _clip_at(self):
        limits = {group.get("max_grad_norm") for group in self.param_groups}
        if len(limits) > 1:
            raise ValueError("one max_grad_norm for all parameter groups: the norm is taken over all of them")
        limit = limits.pop()
        return None if limit is None else _limit(limit)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        max_norm = self._clip_at()
        work = []
        laid_out = {}   # copies of gradients that are not laid out as their parameters: one of each, or the norm would count them again
        for group in self.param_groups:
            live = [p for p in group["params"] if p.grad is not None]
            if not live:
                continue
            grads, ms, vs = [], [], []
            for p in live:
                if p.dtype != torch.float32 or p.grad.dtype != torch.float32 or not p.is_cuda or p.grad.is_sparse:
                    raise RuntimeError("sparc_amd.optim.Adam updates dense float32 parameters on an MI355X")
                if not p.is_contiguous():
                    raise RuntimeError("sparc_amd.optim.Adam needs contiguous parameters")
                st = self.state[p]
                if not st:
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                g = p.grad
                if not g.is_contiguous():
                    key = g.data_ptr(), g.shape, g.stride()
                    g = laid_out[key] if key in laid_out else laid_out.setdefault(key, g.contiguous())
                grads.append(g)
                ms.append(st["exp_avg"])
                vs.append(st["exp_avg_sq"])
            dev = live[0].device
            records, once = _adam_records(live, grads, ms, vs, dev)
            rates = (float(group["lr"]), float(group["betas"][0]), float(group["betas"][1]), float(group["eps"]),
                     float(group["weight_decay"]), int(group.get("step", 0)) + 1)
            work.append((group, live, grads, ms, vs, dev, records, once, rates))
        if not work:
            return loss
        if len(work) > 1:   # nothing moves where a later group would be refused
            every = array("q")
            for w in work:
                every.extend(w[6])
            check(lib.sparc_adam_check(sum(len(w[1]) for w in work), _address(every)), "sparc_adam_check")
        if max_norm is not None and len(work) > 1:   # the norm over all groups
            device = work[0][5]
            require_gpu(device)
            parts, count = _norm_of(*_grad_records([g for w in work for g in w[2]], device), device)
            self.grad_norm = torch.empty((), dtype=torch.float32, device=device)
        for group, live, _, ms, vs, dev, records, once, rates in work:   # all that can be refused but a rate has been
            if max_norm is None:
                _adam_launches(records, len(live), rates, dev)
            elif len(work) == 1:
                self.grad_norm = _clipped_step(records, once, len(live), rates, max_norm, dev)
            else:
                launch("sparc_adam_step_clipped", lib.sparc_adam_step_clipped, dev, len(live), _address(records), *rates,
                       parts.data_ptr(), count, max_norm, self.grad_norm.data_ptr())
            group["step"] = rates[-1]
            increment_version([*live, *ms, *vs])
        return loss
