"""The global gradient norm over many tensors, clipping by it, and an Adam step on the clipped gradient (csrc/grad_clip.hip).

The reference's loop steps ``torch.optim.Adam`` as it is (vddp.py:1481, 1629-1633); these are what it takes to train a recurrent encoder with it:
``clip_grad_norm_`` in front of an optimizer of the caller's own, ``ClippedAdam`` -- the same update with the clipping inside, so that it costs no pass
over the gradients -- or ``DataParallelTrainer(max_grad_norm=...)``.
"""
from __future__ import annotations

import ctypes as C
from typing import Iterable, Optional

import torch

from . import _native as N


def positive_bound(max_norm: float, what: str) -> float:
    """`max_norm`, if it is positive as the float32 that it becomes: below half of the smallest one it would turn into zero, which means no clipping."""
    max_norm = float(max_norm)
    if not C.c_float(max_norm).value > 0.0:
        raise ValueError(f"{what} must be positive (in float32), got {max_norm}")
    return max_norm


def _as_list(tensors, what: str) -> list:
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    for kind in set(map(type, tensors)):
        if not issubclass(kind, torch.Tensor):
            raise TypeError(f"{what}: expected tensors, got {kind.__name__}")
    return tensors


def grad_norm(grads: Iterable[torch.Tensor]) -> torch.Tensor:
    """sqrt of the sum of all squares of `grads` (any mixture of float32, bfloat16, float16), as a float32 scalar on their device; sums are held in 64 bits
    and have the same bits every time.  Tensors must be contiguous.  No tensors: a zero on the CPU."""
    return N.binding().grad_norm([grads] if isinstance(grads, torch.Tensor) else grads)


def clip_grad_norm_(grads: Iterable[torch.Tensor], max_norm: float) -> torch.Tensor:
    """Scales `grads` (the gradient tensors themselves) in place by min(1, max_norm / (norm + 1e-6)) and returns the norm they had, as a float32 scalar on
    their device -- torch.nn.utils.clip_grad_norm_ without its host work; nothing is read or written a second time where the norm is within the bound.
    A NaN norm makes every gradient NaN, an infinite one makes the finite ones zero, as there.  Tensors must be contiguous and not overlap."""
    max_norm = positive_bound(max_norm, "clip_grad_norm_: max_norm")
    return N.binding().clip_grad_norm([grads] if isinstance(grads, torch.Tensor) else grads, max_norm)


class ClippedAdam:
    """Adam (the update of torch.optim.Adam without weight decay or amsgrad) on gradients clipped by their global norm.

    params: float32 tensors, kept contiguous; exp_avgs / exp_avg_sqs: their moments (zeros where not given), step: the updates they have had.
    max_norm None: no clipping.  Parameters may be re-homed (``p.data = ...``) but not resized."""

    def __init__(self, params: Iterable[torch.Tensor], lr: float = 1e-4, betas=(0.9, 0.999), eps: float = 1e-8, max_norm: Optional[float] = None, *,
                 exp_avgs: Optional[Iterable[torch.Tensor]] = None, exp_avg_sqs: Optional[Iterable[torch.Tensor]] = None, step: int = 0):
        self.params = _as_list(params, "ClippedAdam")
        if not self.params:
            raise ValueError("ClippedAdam: no parameters")
        if max_norm is not None:
            max_norm = positive_bound(max_norm, "ClippedAdam: max_norm")
        if not (lr >= 0.0 and eps >= 0.0 and all(0.0 <= b < 1.0 for b in betas) and len(betas) == 2 and step >= 0):
            raise ValueError(f"ClippedAdam: lr {lr}, betas {betas}, eps {eps}, step {step}")
        self.lr, self.betas, self.eps, self.max_norm, self.steps_taken = lr, tuple(betas), eps, max_norm, int(step)
        self.exp_avgs = [torch.zeros_like(p, memory_format=torch.contiguous_format) for p in self.params] if exp_avgs is None else _as_list(exp_avgs, "ClippedAdam")
        self.exp_avg_sqs = [torch.zeros_like(p, memory_format=torch.contiguous_format) for p in self.params] if exp_avg_sqs is None \
            else _as_list(exp_avg_sqs, "ClippedAdam")
        self.exp_avgs, self.exp_avg_sqs = [m.detach() for m in self.exp_avgs], [v.detach() for v in self.exp_avg_sqs]
        sizes = [p.numel() for p in self.params]
        for name, ts in (("params", self.params), ("exp_avgs", self.exp_avgs), ("exp_avg_sqs", self.exp_avg_sqs)):
            if [t.numel() for t in ts] != sizes:
                raise ValueError(f"ClippedAdam: {name} do not fit the parameters")
            if any(t.dtype != torch.float32 for t in ts):
                raise TypeError(f"ClippedAdam: {name} must be float32")
            if not all(t.is_contiguous() for t in ts):
                raise ValueError(f"ClippedAdam: {name} must be contiguous")
            if any(t.device != self.params[0].device for t in ts):
                raise ValueError("ClippedAdam: the tensors are on several devices")
        if not self.params[0].is_cuda:
            raise N.NativeError("ClippedAdam: tensors must live on the GPU (there is no CPU path)")

    def step(self, grads: Optional[Iterable[Optional[torch.Tensor]]] = None) -> torch.Tensor:
        """One update from `grads` (one per parameter; default: every ``p.grad``; None: that parameter stays as it is, and its moments too).
        Returns the gradients' global norm before clipping, a float32 scalar on the device."""
        if torch.cuda.is_current_stream_capturing():  # (its replays would all be the same step)
            raise RuntimeError("ClippedAdam.step: cannot be captured into a graph, the count of steps is the host's")
        b1, b2 = self.betas
        norm = N.binding().clipped_adam(self.params, self.exp_avgs, self.exp_avg_sqs, grads, self.lr, b1, b2, self.eps, self.max_norm or 0.0, self.steps_taken + 1)
        if norm is None:  # no gradient at all: no step
            return torch.zeros((), device=self.params[0].device)
        self.steps_taken += 1
        return norm
