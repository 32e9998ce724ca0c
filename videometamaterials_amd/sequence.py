"""Operators of sequence encoders: the gated linear recurrence (csrc/gated_scan.hip) and the gated feed-forward product (csrc/gated_ff.hip), each with its
gradients.  They stand beside the GRU of ``cond_att_GRU`` (vddp.py:546-549): a recurrence that is scanned in parallel over time, and the mixing of
channels behind it; ``Unet3D(cond_att_scan=True)`` builds its load-history encoder from them.
Checks, workspaces, launches and the autograd nodes are compiled (csrc/torch_binding.cpp).  Gradients are those of the backward pass; forward-mode derivatives,
the transforms of torch.func, tracing (torch.jit.trace, make_fx, torch.export) and tensors that stand in for others are refused (NotImplementedError); torch.compile
breaks its graph around a call.  Calls and their backward passes may be captured into a HIP graph; a captured backward whose leaves an eager graph on the default stream
still holds is refused (the capture would end the process).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native as N

ACTIVATIONS = {"silu": 0, "gelu": 1}


def gated_linear_scan(x: torch.Tensor, gate: torch.Tensor, h0: Optional[torch.Tensor] = None,
                      lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """h_t = f_t h_(t-1) + (1 - f_t) x_t with f = sigmoid(gate), over dimension 1 of x and gate (B, L, D); returns (all h_t, the last state).

    x, gate: float32, bfloat16 or float16, of one type and shape; any batch and time strides (they may be the halves of one projection's rows).
    h0 (B, D): the state in front of the first step, zero where not given.  States are float32, inside and out.
    lengths (B,), integers on the same device: behind a sequence's length the output is zero, the state stands still, and what the inputs hold there
    is not read; values outside 0 .. L are taken as the nearest of these.
    One token at a time: L = 1 with the last state as the next call's h0.  Differentiable (once) in x, gate and h0."""
    return N.binding().gated_linear_scan(x, gate, h0, lengths)


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
                       b_up: Optional[torch.Tensor] = None, activation: str = "silu") -> torch.Tensor:
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up) over the last dimension of x (..., K), in one kernel; returns (..., F).

    w_gate, w_up (F, K) and the biases (F,) (both or none) as torch.nn.Linear keeps them; activation "silu" or "gelu" (the erf form); everything float32,
    bfloat16 or float16 alike.  Sums are held in float32 for every type; the float32 products are made on the matrix cores from three bfloat16 parts of
    each value, to float32's own accuracy (an infinite operand gives NaN; an operand below 2^-110 is rounded to a multiple of 2^-133, bfloat16's smallest number).  Differentiable (once) in every tensor; the backward's dg and du are
    rounded to the type: 16-bit gradients of x and the weights are off by that rounding and their own (1.41 times their own alone), and with float16 the
    loss has to be scaled as for any float16 product."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"gated_feed_forward: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return N.binding().gated_feed_forward(x, w_gate, w_up, b_gate, b_up, act)
