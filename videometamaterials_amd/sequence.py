"""Operators of sequence encoders: the gated linear recurrence (csrc/gated_scan.hip) and the gated feed-forward product (csrc/gated_ff.hip), each with its
gradients.  They stand beside the GRU of ``cond_att_GRU`` (vddp.py:546-549): a recurrence that is scanned in parallel over time, and the mixing of
channels behind it; ``Unet3D(cond_att_scan=True)`` builds its load-history encoder from them.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _native as N
from .optim import TYPES, on_device, stream_of

ACTIVATIONS = {"silu": 0, "gelu": 1}


def _need_gpu(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise N.NativeError(f"{what}: tensors must live on the GPU (there is no CPU path)")


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with neighbouring values in its last dimension and rows less than 2^22 values apart, as the kernels' 32-bit offsets need them (else a copy)."""
    return t if (t.stride(-1) == 1 or t.shape[-1] == 1 and t.is_contiguous()) and t.stride(-2) < 1 << 22 else t.contiguous()


def _place(t: Optional[torch.Tensor]) -> tuple:
    return (None, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1))


# ---------------------------------------------------------------- gated linear recurrence


def _scan_desc(x, gate, h0, lengths, y=None, h_last=None, states=None, dy=None, dx=None, dgate=None, dh_last=None, dh0=None):
    B, L, D = x.shape
    return N.GatedScanDesc(*_place(x), *_place(gate), *_place(y), _ptr(h0), _ptr(h_last), _ptr(lengths), _ptr(states), *_place(dy), *_place(dx),
                           *_place(dgate), _ptr(dh_last), _ptr(dh0), None, L, B, D, TYPES[x.dtype])


def _scan_workspace(lib, d, backward: int, device) -> Optional[torch.Tensor]:
    size = lib.vmm_gated_scan_workspace(C.byref(d), backward)
    if size < 0:
        raise ValueError("gated_linear_scan: a size is out of range")
    if size == 0:
        return None
    work = torch.empty(size, dtype=torch.uint8, device=device)
    d.workspace = work.data_ptr()
    return work


def _scan_forward(x, gate, h0, lengths, keep: bool):
    B, L, D = x.shape
    lib = N.lib()
    with on_device(x.get_device()):
        y = torch.empty((B, L, D), dtype=x.dtype, device=x.device)
        h_last = torch.empty((B, D), dtype=torch.float32, device=x.device)
        d = _scan_desc(x, gate, h0, lengths, y=y, h_last=h_last)
        states = None
        if keep:
            states = torch.empty(max(lib.vmm_gated_scan_states(C.byref(d)), 0), dtype=torch.float32, device=x.device)
            d.states = states.data_ptr()
        work = _scan_workspace(lib, d, 0, x.device)  # noqa: F841 (alive until the launch is enqueued)
        N.check(lib.vmm_gated_scan(C.byref(d), stream_of(x.get_device())), "vmm_gated_scan")
    return y, h_last, states


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, lengths):
        ctx.set_materialize_grads(False)
        y, h_last, states = _scan_forward(x, gate, h0, lengths, True)
        ctx.save_for_backward(x, gate, lengths, states)
        return y, h_last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh_last):
        x, gate, lengths, states = ctx.saved_tensors
        if dy is None and dh_last is None:
            return None, None, None, None
        B, L, D = x.shape
        lib = N.lib()
        with on_device(x.get_device()):
            dy = None if dy is None else _rows(dy)
            dh_last = None if dh_last is None else dh_last.contiguous()
            dx, dgate = (torch.empty((B, L, D), dtype=x.dtype, device=x.device) if need else None for need in ctx.needs_input_grad[:2])
            dh0 = torch.empty((B, D), dtype=torch.float32, device=x.device) if ctx.needs_input_grad[2] else None
            d = _scan_desc(x, gate, None, lengths, states=states, dy=dy, dx=dx, dgate=dgate, dh_last=dh_last, dh0=dh0)
            work = _scan_workspace(lib, d, 1, x.device)  # noqa: F841
            N.check(lib.vmm_gated_scan_bwd(C.byref(d), stream_of(x.get_device())), "vmm_gated_scan_bwd")
        return dx, dgate, dh0, None


def gated_linear_scan(x: torch.Tensor, gate: torch.Tensor, h0: Optional[torch.Tensor] = None,
                      lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """h_t = f_t h_(t-1) + (1 - f_t) x_t with f = sigmoid(gate), over dimension 1 of x and gate (B, L, D); returns (all h_t, the last state).

    x, gate: float32, bfloat16 or float16, of one type and shape; any batch and time strides (they may be the halves of one projection's rows).
    h0 (B, D): the state in front of the first step, zero where not given.  States are float32, inside and out.
    lengths (B,), integers on the same device: behind a sequence's length the output is zero, the state stands still, and what the inputs hold there
    is not read; values outside 0 .. L are taken as the nearest of these.
    One token at a time: L = 1 with the last state as the next call's h0.  Differentiable (once) in x, gate and h0."""
    what = "gated_linear_scan"
    if x.dim() != 3 or gate.shape != x.shape:
        raise ValueError(f"{what}: x and gate must be (B, L, D) and alike, got {tuple(x.shape)} and {tuple(gate.shape)}")
    if x.dtype not in TYPES or gate.dtype != x.dtype:
        raise TypeError(f"{what}: x and gate must be float32, bfloat16 or float16 alike, got {x.dtype} and {gate.dtype}")
    _need_gpu(x, what)
    B, L, D = x.shape
    if h0 is not None:
        if h0.shape != (B, D) or not h0.is_floating_point():
            raise ValueError(f"{what}: h0 must be a floating ({B}, {D}), got {h0.dtype} {tuple(h0.shape)}")
        h0 = h0.float().contiguous()
    if lengths is not None:
        if lengths.shape != (B,) or lengths.is_floating_point() or lengths.is_complex() or lengths.dtype == torch.bool:
            raise ValueError(f"{what}: lengths must be ({B},) integers, got {lengths.dtype} {tuple(lengths.shape)}")
        lengths = lengths.contiguous() if lengths.dtype == torch.int32 else lengths.clamp(min=0, max=L).to(torch.int32)
    for t in (gate, h0, lengths):
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: all tensors must be on {x.device}")
    x, gate = _rows(x), _rows(gate)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(x, gate, h0, lengths)
    y, h_last, _ = _scan_forward(x, gate, h0, lengths, False)
    return y, h_last


# ---------------------------------------------------------------- gated feed-forward product


def _ff_desc(x, wg, wu, bg, bu, act, h=None, g_pre=None, u_pre=None, dh=None, dx=None, dwg=None, dwu=None, dbg=None, dbu=None):
    M, K = x.shape
    lead = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    return N.GatedFFDesc(_ptr(x), lead(x), _ptr(wg), _ptr(wu), _ptr(bg), _ptr(bu), _ptr(h), lead(h), _ptr(g_pre), _ptr(u_pre), _ptr(dh), lead(dh), _ptr(dx),
                         lead(dx), _ptr(dwg), _ptr(dwu), _ptr(dbg), _ptr(dbu), None, M, K, wg.shape[0], TYPES[x.dtype], act)


def _ff_workspace(lib, d, backward: int, device) -> Optional[torch.Tensor]:
    size = lib.vmm_gated_ff_workspace(C.byref(d), backward)
    if size < 0:
        raise ValueError("gated_feed_forward: a size is out of range")
    if size == 0:
        return None
    work = torch.empty(size, dtype=torch.uint8, device=device)
    d.workspace = work.data_ptr()
    return work


def _ff_forward(x, wg, wu, bg, bu, act: int, keep: bool):
    M, F = x.shape[0], wg.shape[0]
    lib = N.lib()
    with on_device(x.get_device()):
        h = torch.empty((M, F), dtype=x.dtype, device=x.device)
        # what the backward needs of the products stays in fp32: rounded to 16 bits they would put an error of their own into every gradient
        pre = torch.empty((2, M, F), dtype=torch.float32, device=x.device) if keep else (None, None)
        d = _ff_desc(x, wg, wu, bg, bu, act, h=h, g_pre=pre[0], u_pre=pre[1])
        work = _ff_workspace(lib, d, 0, x.device)  # noqa: F841 (alive until the launch is enqueued)
        N.check(lib.vmm_gated_ff(C.byref(d), stream_of(x.get_device())), "vmm_gated_ff")
    return h, pre if keep else None


class _GatedFF(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, act):
        h, pre = _ff_forward(x, wg, wu, bg, bu, act, True)
        ctx.act = act
        ctx.save_for_backward(x, wg, wu, pre)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, wg, wu, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        lib = N.lib()
        with on_device(x.get_device()):
            dh = _rows(dh)
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
            weights, biases = need[1] or need[2], need[3] or need[4]
            dwg, dwu = torch.empty((2,) + wg.shape, dtype=x.dtype, device=x.device) if weights else (None, None)
            dbg, dbu = torch.empty((2, wg.shape[0]), dtype=x.dtype, device=x.device) if biases else (None, None)
            d = _ff_desc(x, wg, wu, None, None, ctx.act, g_pre=pre[0], u_pre=pre[1], dh=dh, dx=dx, dwg=dwg, dwu=dwu, dbg=dbg, dbu=dbu)
            work = _ff_workspace(lib, d, 1, x.device)  # noqa: F841
            N.check(lib.vmm_gated_ff_bwd(C.byref(d), stream_of(x.get_device())), "vmm_gated_ff_bwd")
        return dx, *(t if n else None for t, n in zip((dwg, dwu, dbg, dbu), need[1:5])), None


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
                       b_up: Optional[torch.Tensor] = None, activation: str = "silu") -> torch.Tensor:
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up) over the last dimension of x (..., K), in one kernel; returns (..., F).

    w_gate, w_up (F, K) and the biases (F,) (both or none) as torch.nn.Linear keeps them; activation "silu" or "gelu" (the erf form); everything float32,
    bfloat16 or float16 alike.  Sums are held in float32 for every type; the float32 products are made on the matrix cores from three bfloat16 parts of
    each value, to float32's own accuracy (an infinite operand gives NaN).  Differentiable (once) in every tensor; the backward's dg and du are
    rounded to the type, so with float16 the loss has to be scaled as for any float16 product."""
    what = "gated_feed_forward"
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or x.shape[-1] != w_gate.shape[1] or 0 in w_gate.shape:
        raise ValueError(f"{what}: x (..., K) and weights (F, K) do not fit: {tuple(x.shape)}, {tuple(w_gate.shape)}, {tuple(w_up.shape)}")
    if (b_gate is None) != (b_up is None):
        raise ValueError(f"{what}: both biases or none")
    every = (x, w_gate, w_up) if b_gate is None else (x, w_gate, w_up, b_gate, b_up)
    for t in every[3:]:
        if t.shape != w_gate.shape[:1]:
            raise ValueError(f"{what}: biases must be ({w_gate.shape[0]},), got {tuple(t.shape)}")
    if x.dtype not in TYPES or any(t.dtype != x.dtype for t in every):
        raise TypeError(f"{what}: float32, bfloat16 or float16 tensors of one type, got {[str(t.dtype) for t in every]}")
    _need_gpu(x, what)
    if any(t.device != x.device for t in every):
        raise ValueError(f"{what}: all tensors must be on {x.device}")
    F, K = w_gate.shape
    rows = _rows(x.reshape(-1, K))
    wg, wu = w_gate.contiguous(), w_up.contiguous()
    bg, bu = (None, None) if b_gate is None else (b_gate.contiguous(), b_up.contiguous())
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t.requires_grad for t in every):
        h = _GatedFF.apply(rows, wg, wu, bg, bu, act)
    else:
        h, _ = _ff_forward(rows, wg, wu, bg, bu, act, False)
    return h.view(x.shape[:-1] + (F,))
