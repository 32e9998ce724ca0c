"""The global gradient norm over many tensors, clipping by it, and an Adam step on the clipped gradient (csrc/grad_clip.hip).

The reference's loop steps ``torch.optim.Adam`` as it is (vddp.py:1481, 1629-1633); these are what it takes to train a recurrent encoder with it:
``clip_grad_norm_`` in front of an optimizer of the caller's own, ``ClippedAdam`` -- the same update with the clipping inside, so that it costs no pass
over the gradients -- or ``DataParallelTrainer(max_grad_norm=...)``.
"""
from __future__ import annotations

from operator import attrgetter
from typing import Iterable, List, Optional, Sequence

import numpy as np
import torch

from . import _native as N

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_dtype = attrgetter("dtype")


def on_device(index: int):
    """The device of a call's tensors made current for its launches, where another one is."""
    return torch.cuda.device(index if index != torch.cuda.current_device() else -1)


def stream_of(index: int) -> int:
    """Handle of the current stream of a device."""
    return torch._C._cuda_getCurrentRawStream(index)


def _same_device(tensors: Sequence[torch.Tensor], what: str) -> int:
    places = set(map(torch.Tensor.get_device, tensors))
    if len(places) != 1:
        raise ValueError(f"{what}: the tensors are on several devices")
    (index,) = places
    if index < 0 or not tensors[0].is_cuda:
        raise N.NativeError(f"{what}: tensors must live on the GPU (there is no CPU path)")
    return index


def _check_grads(tensors: Sequence[torch.Tensor], what: str) -> int:
    bad = set(map(_dtype, tensors)) - set(TYPES)
    if bad:
        raise TypeError(f"{what}: float32, bfloat16 or float16 tensors, got {sorted(map(str, bad))}")
    if not all(map(torch.Tensor.is_contiguous, tensors)):
        raise ValueError(f"{what}: tensors must be contiguous")
    return _same_device(tensors, what)


def _as_list(tensors, what: str) -> List[torch.Tensor]:
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    for kind in set(map(type, tensors)):
        if not issubclass(kind, torch.Tensor):
            raise TypeError(f"{what}: expected tensors, got {kind.__name__}")
    return tensors


# the job structs of include/vmm_sequence.h as rows of an array: hundreds of tensors are filled in column by column
GRAD_JOB = np.dtype([("g", np.uint64), ("n", np.int64), ("type", np.int32), ("reserved", np.int32)])
ADAM_JOB = np.dtype([("p", np.uint64), ("g", np.uint64), ("m", np.uint64), ("v", np.uint64), ("n", np.int64), ("type", np.int32), ("reserved", np.int32)])


def _grad_jobs(tensors: Sequence[torch.Tensor]) -> np.ndarray:
    jobs = np.zeros(len(tensors), GRAD_JOB)
    jobs["g"] = list(map(torch.Tensor.data_ptr, tensors))
    jobs["n"] = list(map(torch.Tensor.numel, tensors))
    kinds = list(map(_dtype, tensors))
    first = kinds[0]
    jobs["type"] = TYPES[first] if kinds.count(first) == len(kinds) else [TYPES[k] for k in kinds]
    return jobs


def _norm(jobs, n: int, max_norm: float, index: int, scale: float = 1.0) -> torch.Tensor:
    """(norm, factor) on the device; max_norm <= 0: the factor is one."""
    lib = N.lib()
    size = lib.vmm_grad_norm_workspace(jobs.ctypes.data, n)
    if size < 0:
        raise ValueError("gradient norm: a tensor that is not aligned to its type")
    work = torch.empty(size // 8 + 1, dtype=torch.float64, device=index)  # (the last one holds the two results)
    out = work[size // 8:].view(torch.float32)
    N.check(lib.vmm_grad_norm(jobs.ctypes.data, n, scale, max_norm, None, work.data_ptr(), out.data_ptr(), stream_of(index)),
            "vmm_grad_norm")
    return out


@torch.no_grad()
def grad_norm(grads: Iterable[torch.Tensor]) -> torch.Tensor:
    """sqrt of the sum of all squares of `grads` (any mixture of float32, bfloat16, float16), as a float32 scalar on their device; sums are held in 64 bits
    and have the same bits every time.  No tensors: a zero on the CPU."""
    grads = _as_list(grads, "grad_norm")
    if not grads:
        return torch.zeros(())
    index = _check_grads(grads, "grad_norm")
    with on_device(index):
        return _norm(_grad_jobs(grads), len(grads), 0.0, index)[0]


@torch.no_grad()
def clip_grad_norm_(grads: Iterable[torch.Tensor], max_norm: float) -> torch.Tensor:
    """Scales `grads` (the gradient tensors themselves) in place by min(1, max_norm / (norm + 1e-6)) and returns the norm they had, as a float32 scalar on
    their device -- torch.nn.utils.clip_grad_norm_ without its host work; nothing is read or written a second time where the norm is within the bound.
    A NaN norm makes every gradient NaN, an infinite one makes the finite ones zero, as there.  Tensors must not overlap."""
    grads = _as_list(grads, "clip_grad_norm_")
    max_norm = float(max_norm)
    if not max_norm > 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm must be positive, got {max_norm}")
    if not grads:
        return torch.zeros(())
    index = _check_grads(grads, "clip_grad_norm_")
    with on_device(index):
        jobs = _grad_jobs(grads)
        out = _norm(jobs, len(grads), max_norm, index)
        code = N.lib().vmm_grad_clip(jobs.ctypes.data, len(grads), out.data_ptr(), stream_of(index))
        if code == -2:
            raise ValueError("clip_grad_norm_: tensors overlap in memory")
        N.check(code, "vmm_grad_clip")
        torch.autograd.graph.increment_version(grads)  # written through raw pointers
    return out[0]


class ClippedAdam:
    """Adam (the update of torch.optim.Adam without weight decay or amsgrad) on gradients clipped by their global norm.

    params: float32 tensors, kept contiguous; exp_avgs / exp_avg_sqs: their moments (zeros where not given), step: the updates they have had.
    max_norm None: no clipping.  The optimizer keeps one table of its tensors; ``step`` re-reads the parameters' addresses, so they may be re-homed
    (``p.data = ...``) but not resized; the moments stay where they are: to load others, ``copy_`` into them."""

    def __init__(self, params: Iterable[torch.Tensor], lr: float = 1e-4, betas=(0.9, 0.999), eps: float = 1e-8, max_norm: Optional[float] = None, *,
                 exp_avgs: Optional[Iterable[torch.Tensor]] = None, exp_avg_sqs: Optional[Iterable[torch.Tensor]] = None, step: int = 0):
        self.params = _as_list(params, "ClippedAdam")
        if not self.params:
            raise ValueError("ClippedAdam: no parameters")
        if max_norm is not None and not max_norm > 0.0:
            raise ValueError(f"ClippedAdam: max_norm must be positive or None, got {max_norm}")
        if not (lr >= 0.0 and eps >= 0.0 and all(0.0 <= b < 1.0 for b in betas) and len(betas) == 2 and step >= 0):
            raise ValueError(f"ClippedAdam: lr {lr}, betas {betas}, eps {eps}, step {step}")
        self.lr, self.betas, self.eps, self.max_norm, self.steps_taken = lr, tuple(betas), eps, max_norm, int(step)
        self.exp_avgs = [torch.zeros_like(p, memory_format=torch.contiguous_format) for p in self.params] if exp_avgs is None else _as_list(exp_avgs, "ClippedAdam")
        self.exp_avg_sqs = [torch.zeros_like(p, memory_format=torch.contiguous_format) for p in self.params] if exp_avg_sqs is None \
            else _as_list(exp_avg_sqs, "ClippedAdam")
        self.exp_avgs, self.exp_avg_sqs = tuple(m.detach() for m in self.exp_avgs), tuple(v.detach() for v in self.exp_avg_sqs)
        self._moments = (self.exp_avgs, self.exp_avg_sqs)  # the table below holds their addresses
        self._sizes = list(map(torch.Tensor.numel, self.params))
        for name, ts in (("params", self.params), ("exp_avgs", self.exp_avgs), ("exp_avg_sqs", self.exp_avg_sqs)):
            if len(ts) != len(self.params) or list(map(torch.Tensor.numel, ts)) != self._sizes:
                raise ValueError(f"ClippedAdam: {name} do not fit the parameters")
        self._device = self._check_own()
        self._jobs = np.zeros(len(self.params), ADAM_JOB)
        self._jobs["m"] = list(map(torch.Tensor.data_ptr, self.exp_avgs))
        self._jobs["v"] = list(map(torch.Tensor.data_ptr, self.exp_avg_sqs))
        self._jobs["n"] = self._sizes
        self._at: List[int] = []

    def _check_own(self) -> int:
        every = [*self.params, *self._moments[0], *self._moments[1]]
        if set(map(_dtype, every)) != {torch.float32}:
            raise TypeError("ClippedAdam: parameters and moments must be float32")
        if not all(map(torch.Tensor.is_contiguous, every)):
            raise ValueError("ClippedAdam: parameters and moments must be contiguous")
        return _same_device(every, "ClippedAdam")

    @torch.no_grad()
    def step(self, grads: Optional[Iterable[Optional[torch.Tensor]]] = None) -> torch.Tensor:
        """One update from `grads` (one per parameter; default: every ``p.grad``; None: that parameter stays as it is, and its moments too).
        Returns the gradients' global norm before clipping, a float32 scalar on the device."""
        if torch.cuda.is_current_stream_capturing():  # (its replays would all be the same step)
            raise RuntimeError("ClippedAdam.step: cannot be captured into a graph, the count of steps is the host's")
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"ClippedAdam.step: {len(grads)} gradients for {len(self.params)} parameters")
        here = [i for i, g in enumerate(grads) if g is not None]
        if len(here) < len(grads):
            grads = [grads[i] for i in here]
            if not grads:
                return torch.zeros((), device=self._device)
        sizes = self._sizes if len(here) == len(self._sizes) else [self._sizes[i] for i in here]
        if list(map(torch.Tensor.numel, grads)) != sizes:
            raise ValueError("ClippedAdam.step: gradients do not fit the parameters")
        if _check_grads(grads, "ClippedAdam.step") != self._device:
            raise ValueError("ClippedAdam.step: gradients and parameters are on different devices")
        at = list(map(torch.Tensor.data_ptr, self.params))
        if at != self._at:  # first step, or parameters were re-homed
            if self._check_own() != self._device or list(map(torch.Tensor.numel, self.params)) != self._sizes:
                raise ValueError("ClippedAdam.step: parameters were moved to another device or resized")
            self._jobs["p"] = at
            self._at = at
        with on_device(self._device):
            jobs = self._jobs if len(here) == len(self.params) else self._jobs[here]
            norm_jobs = _grad_jobs(grads)
            jobs["g"], jobs["type"] = norm_jobs["g"], norm_jobs["type"]
            out = _norm(norm_jobs, len(grads), self.max_norm or 0.0, self._device)
            code = N.lib().vmm_adam_step_clipped(jobs.ctypes.data, len(here), self.lr, self.betas[0], self.betas[1], self.eps, self.steps_taken + 1, 1.0, out.data_ptr(),
                                                 None, stream_of(self._device))
            if code == -2:
                raise ValueError("ClippedAdam.step: parameters, moments or gradients overlap in memory")
            N.check(code, "vmm_adam_step_clipped")
        self.steps_taken += 1
        written = self.params if len(here) == len(self.params) else [self.params[i] for i in here]
        torch.autograd.graph.increment_version(written)  # written through raw pointers
        return out[0]
