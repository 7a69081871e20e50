"""Gated activations that keep their inputs in 8 bits between the forward and the backward pass.

``swiglu`` and ``geglu`` save gate and up as they came, the two largest tensors an MLP block holds until its backward.
The functions here save them as int8 codes with one power-of-two step per 32 columns instead: 2.06 bytes for a pair
of elements where bf16 takes 4 and fp32 8.  The forward result is that of ``swiglu`` / ``geglu``, bit for bit;
the backward evaluates the derivative at the values the codes stand for, each within half a step of the input (at
most 1/127 of the largest magnitude among its 32 columns).  Nothing of the caller's is overwritten, and a graph can be
walked twice with ``retain_graph``.

    swiglu_ckpt8, swiglu_packed_ckpt8      autograd, as swiglu / swiglu_packed
    geglu_ckpt8, geglu_packed_ckpt8        autograd, as geglu / geglu_packed
    ckpt8_forward                          (h, kept) without autograd
    ckpt8_pack                             kept alone, for a block that has made h already
    ckpt8_backward                         (dgate, dup) from kept
    ckpt8_backward_recompute               (h, dgate, dup) from kept

The reference has no counterpart: it saves the inputs themselves (kernels/swiglu/swiglu.py:326-385,
kernels/geglu/geglu.py:380-575).  The kept form is defined at ``swiglu_b200_ckpt8_fwd`` in the C header.  A group that
holds an infinity or a NaN (or a magnitude within 1/256 of 2^128, which 8 bits round to infinity) is kept as NaN, so the
gradients of a step that overflowed are not finite either.
As elsewhere in this package there is no path for tensors that are not on a CUDA device.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .geglu import _check_approximate, geglu_forward, geglu_packed_forward
from .swiglu import (
    _DTYPE_CODE, _as_float, _check_cuda_dtype, _check_packed_input, _check_same_shape_inputs, _require_cuda, _stream,
    swiglu_forward, swiglu_packed_forward,
)

ACTIVATIONS = {"silu": 0, "gelu_tanh": 1, "gelu_exact": 2}
GROUP = 32


class Checkpoint8:
    """gate and up of one forward pass in 8 bits.

    ``codes`` int8 ``[2, rows, 32 * groups]`` and ``steps`` uint8 ``[2, rows, groups]`` (gate first), with the shape and
    dtype of the inputs and what the backward needs of the call: the activation and its multipliers."""

    __slots__ = ("codes", "steps", "shape", "dtype", "activation", "gate_multiplier", "down_multiplier")

    def __init__(self, codes, steps, shape, dtype, activation="silu", gate_multiplier=1.0, down_multiplier=1.0):
        self.codes = codes
        self.steps = steps
        self.shape = torch.Size(shape)
        self.dtype = dtype
        self.activation = _check_activation(activation)
        self.gate_multiplier, self.down_multiplier = _check_multipliers(activation, gate_multiplier, down_multiplier)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.steps.numel()

    def dequantize(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values that the codes of gate and up stand for, in fp32 and the inputs' shape."""
        exponent = self.steps.to(torch.int32)
        step = torch.where(exponent == 255, 0x7fc00000, exponent << 23).view(torch.float32)
        values = self.codes.view(*self.steps.shape, GROUP).to(torch.float32) * step.unsqueeze(-1)
        n_cols = self.shape[-1]
        values = values.view(self.codes.shape)[:, :, :n_cols].reshape(2, *self.shape)
        return values[0], values[1]


def _check_activation(activation: str) -> str:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    return activation


def _check_multipliers(activation: str, gate_multiplier, down_multiplier) -> Tuple[float, float]:
    gm = _as_float("gate_multiplier", gate_multiplier)
    dm = _as_float("down_multiplier", down_multiplier)
    if activation != "silu" and (gm != 1.0 or dm != 1.0):
        raise ValueError("the GELU activations have no multipliers")
    return gm, dm


def _check_inputs(gate: torch.Tensor, up: torch.Tensor) -> None:
    _check_same_shape_inputs(gate, up)
    _check_cuda_dtype(gate)
    _require_cuda(gate, "gate")
    if gate.dim() == 0:
        raise ValueError("gate and up need at least one dimension")


def _row_view(x: torch.Tensor) -> Optional[torch.Tensor]:
    """``x`` as ``[rows, cols]`` over its own storage when its rows lie in order without touching, else ``None``."""
    n_cols = x.shape[-1]
    rows = x.numel() // n_cols if n_cols else 0
    try:
        v = x.view(rows, n_cols)
    except RuntimeError:
        return None
    if v.numel() and ((n_cols > 1 and v.stride(1) != 1) or (rows > 1 and v.stride(0) < n_cols)):
        return None
    return v


def _rows(x: torch.Tensor) -> torch.Tensor:
    v = _row_view(x)
    return _row_view(x.contiguous()) if v is None else v


def _pitch(v: torch.Tensor) -> int:
    return v.stride(0) if v.shape[0] > 1 else v.shape[1]


def _input_rows(gate: torch.Tensor, up: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Both as rows of one pitch: in place when they are (two halves of a packed projection), else copied."""
    g, u = _row_view(gate), _row_view(up)
    if g is not None and u is not None and _pitch(g) == _pitch(u):
        return g, u
    return _row_view(gate.contiguous()), _row_view(up.contiguous())


def _keep(gate_2d, up_2d, shape, activation, gm, dm, want_h: bool, where: str):
    rows, n_cols = gate_2d.shape
    groups = (n_cols + GROUP - 1) // GROUP
    device, dtype = gate_2d.device, gate_2d.dtype
    codes = torch.empty((2, rows, groups * GROUP), dtype=torch.int8, device=device)
    steps = torch.empty((2, rows, groups), dtype=torch.uint8, device=device)
    h = torch.empty((rows, n_cols), dtype=dtype, device=device) if want_h else None
    plane, plane_steps = rows * groups * GROUP, rows * groups
    _lib.check(
        where,
        _lib.lib.swiglu_b200_ckpt8_fwd(
            h.data_ptr() if want_h else None, codes.data_ptr(), codes.data_ptr() + plane, steps.data_ptr(),
            steps.data_ptr() + plane_steps, gate_2d.data_ptr(), up_2d.data_ptr(), rows, n_cols, _pitch(gate_2d),
            n_cols, _DTYPE_CODE[dtype], ACTIVATIONS[activation], gm, dm, device.index, _stream(device),
        ),
    )
    return h, Checkpoint8(codes, steps, shape, dtype, activation, gm, dm)


def ckpt8_forward(gate: torch.Tensor, up: torch.Tensor, activation: str = "silu", gate_multiplier: float = 1.0,
                  down_multiplier: float = 1.0):
    """``(h, kept)``: ``h = act(gate * gm) * up * dm`` in the shape of ``gate``, and the ``Checkpoint8`` its backward
    needs.  One pass over gate and up; views with a common row pitch (the halves of a packed projection) are read in
    place."""
    _check_activation(activation)
    gm, dm = _check_multipliers(activation, gate_multiplier, down_multiplier)
    _check_inputs(gate, up)
    gate_2d, up_2d = _input_rows(gate, up)
    h, kept = _keep(gate_2d, up_2d, gate.shape, activation, gm, dm, True, "ckpt8_forward")
    return h.view(gate.shape), kept


def ckpt8_pack(gate: torch.Tensor, up: torch.Tensor, activation: str = "silu", gate_multiplier: float = 1.0,
               down_multiplier: float = 1.0) -> Checkpoint8:
    """The ``Checkpoint8`` alone, for a block whose own kernel has made ``h`` (the fused projections)."""
    _check_activation(activation)
    gm, dm = _check_multipliers(activation, gate_multiplier, down_multiplier)
    _check_inputs(gate, up)
    gate_2d, up_2d = _input_rows(gate, up)
    return _keep(gate_2d, up_2d, gate.shape, activation, gm, dm, False, "ckpt8_pack")[1]


def _check_dout(dout: torch.Tensor, kept: Checkpoint8) -> None:
    if dout.dtype != kept.dtype or dout.device != kept.device:
        raise TypeError("dout must have the dtype and device of gate and up")
    if dout.shape != kept.shape:
        raise ValueError(f"dout of shape {tuple(dout.shape)} does not match gate of shape {tuple(kept.shape)}")


def _gradients(dout_2d, kept: Checkpoint8, dgate, dup, grad_pitch: int, h, where: str) -> None:
    """Fills dgate and dup (addresses of rows ``grad_pitch`` apart), and ``h`` when it is given."""
    _, rows, groups = kept.steps.shape
    n_cols = kept.shape[-1]
    codes, steps = kept.codes.data_ptr(), kept.steps.data_ptr()
    device = kept.device
    _lib.check(
        where,
        _lib.lib.swiglu_b200_ckpt8_bwd(
            h.data_ptr() if h is not None else None, dgate, dup, dout_2d.data_ptr(), codes,
            codes + rows * groups * GROUP, steps, steps + rows * groups, rows, n_cols, grad_pitch, _pitch(dout_2d),
            _pitch(h) if h is not None else 0, _DTYPE_CODE[kept.dtype], ACTIVATIONS[kept.activation],
            kept.gate_multiplier, kept.down_multiplier, device.index, _stream(device),
        ),
    )


def ckpt8_backward(dout: torch.Tensor, kept: Checkpoint8):
    """``(dgate, dup)`` of a ``ckpt8_forward`` / ``ckpt8_pack``, in the inputs' shape."""
    _check_dout(dout, kept)
    dout_2d = _rows(dout)
    n_cols = kept.shape[-1]
    dgate, dup = (torch.empty(kept.shape, dtype=kept.dtype, device=kept.device) for _ in range(2))
    _gradients(dout_2d, kept, dgate.data_ptr(), dup.data_ptr(), n_cols, None, "ckpt8_backward")
    return dgate, dup


def ckpt8_backward_recompute(dout: torch.Tensor, kept: Checkpoint8, preserve_inputs: bool = False):
    """``(h, dgate, dup)`` in one pass: the gradients together with ``act(gate * gm) * up * dm`` of the kept values, as
    ``swiglu_backward_recompute`` gives them from gate and up.  Unless ``preserve_inputs`` is set, ``h`` is written
    over ``dout``, which must be contiguous then."""
    _check_dout(dout, kept)
    if preserve_inputs:
        dout_2d = _rows(dout)
        h = torch.empty(dout_2d.shape, dtype=kept.dtype, device=kept.device)
    else:
        if not dout.is_contiguous():
            raise ValueError("the in-place form needs a contiguous dout; pass preserve_inputs=True")
        dout_2d = h = _rows(dout)
    dgate, dup = (torch.empty(kept.shape, dtype=kept.dtype, device=kept.device) for _ in range(2))
    _gradients(dout_2d, kept, dgate.data_ptr(), dup.data_ptr(), kept.shape[-1], h, "ckpt8_backward_recompute")
    return (h.view(kept.shape) if preserve_inputs else dout), dgate, dup


class ForgeCkpt8Function(torch.autograd.Function):
    """``apply(gate, up, activation="silu", gate_multiplier=1.0, down_multiplier=1.0)``; saves the codes and steps."""

    @staticmethod
    def forward(ctx, gate, up, activation="silu", gate_multiplier=1.0, down_multiplier=1.0):
        h, kept = ckpt8_forward(gate, up, activation, gate_multiplier, down_multiplier)
        ctx.save_for_backward(kept.codes, kept.steps)
        ctx.call = (kept.shape, kept.dtype, kept.activation, kept.gate_multiplier, kept.down_multiplier)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        dgate, dup = ckpt8_backward(dout, Checkpoint8(*ctx.saved_tensors, *ctx.call))
        return dgate, dup, None, None, None


class ForgePackedCkpt8Function(torch.autograd.Function):
    """``apply(gate_up, activation="silu", gate_multiplier=1.0, down_multiplier=1.0)`` on the packed layout."""

    @staticmethod
    def forward(ctx, gate_up, activation="silu", gate_multiplier=1.0, down_multiplier=1.0):
        n_cols = gate_up.shape[-1] // 2
        # the two halves of one tensor share a row pitch: nothing is copied unless gate_up itself is not in rows
        packed = gate_up if _row_view(gate_up) is not None else gate_up.contiguous()
        h, kept = ckpt8_forward(packed[..., :n_cols], packed[..., n_cols:], activation, gate_multiplier,
                                down_multiplier)
        ctx.save_for_backward(kept.codes, kept.steps)
        ctx.call = (kept.shape, kept.dtype, kept.activation, kept.gate_multiplier, kept.down_multiplier)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        kept = Checkpoint8(*ctx.saved_tensors, *ctx.call)
        _check_dout(dout, kept)
        n_cols = kept.shape[-1]
        grad = torch.empty((*kept.shape[:-1], 2 * n_cols), dtype=kept.dtype, device=kept.device)
        base = grad.data_ptr()
        _gradients(_rows(dout), kept, base, base + n_cols * grad.element_size(), 2 * n_cols, None,
                   "packed ckpt8_backward")
        return grad, None, None, None


def _records(*inputs: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in inputs)


def swiglu_ckpt8(gate: torch.Tensor, up: torch.Tensor, gate_multiplier: float = 1.0,
                 down_multiplier: float = 1.0) -> torch.Tensor:
    """``swiglu`` that keeps gate and up in 8 bits for its backward (nothing is kept when no gradient is wanted)."""
    _check_same_shape_inputs(gate, up)
    _check_multipliers("silu", gate_multiplier, down_multiplier)
    _require_cuda(gate, "gate")
    if not _records(gate, up):
        return swiglu_forward(gate, up, gate_multiplier, down_multiplier)[0]
    return ForgeCkpt8Function.apply(gate, up, "silu", gate_multiplier, down_multiplier)


def swiglu_packed_ckpt8(gate_up: torch.Tensor, gate_multiplier: float = 1.0,
                        down_multiplier: float = 1.0) -> torch.Tensor:
    """``swiglu_packed`` that keeps both halves in 8 bits for its backward."""
    _check_packed_input(gate_up)
    _check_multipliers("silu", gate_multiplier, down_multiplier)
    _require_cuda(gate_up, "gate_up")
    if not _records(gate_up):
        return swiglu_packed_forward(gate_up, gate_multiplier, down_multiplier)[0]
    return ForgePackedCkpt8Function.apply(gate_up, "silu", gate_multiplier, down_multiplier)


def _gelu(approximate: str) -> str:
    return "gelu_tanh" if _check_approximate(approximate) else "gelu_exact"


def geglu_ckpt8(gate: torch.Tensor, up: torch.Tensor, approximate: str = "tanh") -> torch.Tensor:
    """``geglu`` that keeps gate and up in 8 bits for its backward (nothing is kept when no gradient is wanted)."""
    _check_same_shape_inputs(gate, up)
    activation = _gelu(approximate)
    _require_cuda(gate, "gate")
    if not _records(gate, up):
        return geglu_forward(gate, up, approximate)[0]
    return ForgeCkpt8Function.apply(gate, up, activation)


def geglu_packed_ckpt8(gate_up: torch.Tensor, approximate: str = "tanh") -> torch.Tensor:
    """``geglu_packed`` that keeps both halves in 8 bits for its backward."""
    _check_packed_input(gate_up)
    activation = _gelu(approximate)
    _require_cuda(gate_up, "gate_up")
    if not _records(gate_up):
        return geglu_packed_forward(gate_up, approximate)[0]
    return ForgePackedCkpt8Function.apply(gate_up, activation)
