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

    ``data`` is one uint8 buffer of ``Checkpoint8.size(shape)`` bytes: the codes of gate, the codes of up, the steps of
    gate, the steps of up.  With it go the shape and dtype of the inputs and what the backward needs of the call: the
    activation and its multipliers.  ``codes`` (int8 ``[2, rows, 32 * groups]``) and ``steps`` (uint8
    ``[2, rows, groups]``), gate first, are views of ``data``."""

    __slots__ = ("data", "shape", "dtype", "activation", "gate_multiplier", "down_multiplier")

    def __init__(self, data, shape, dtype, activation="silu", gate_multiplier=1.0, down_multiplier=1.0):
        shape = torch.Size(shape)
        if (data.dtype != torch.uint8 or data.dim() != 1 or data.numel() != Checkpoint8.size(shape)
                or not data.is_contiguous()):
            raise ValueError(f"the kept form of shape {tuple(shape)} is {Checkpoint8.size(shape)} bytes in a row")
        self.data = data
        self.shape = shape
        self.dtype = dtype
        self.activation = _check_activation(activation)
        self.gate_multiplier, self.down_multiplier = _check_multipliers(activation, gate_multiplier, down_multiplier)

    @staticmethod
    def _of(data, shape, dtype, activation, gm, dm) -> "Checkpoint8":
        """One whose parts have been checked."""
        kept = object.__new__(Checkpoint8)
        kept.data, kept.shape, kept.dtype = data, shape, dtype
        kept.activation, kept.gate_multiplier, kept.down_multiplier = activation, gm, dm
        return kept

    @staticmethod
    def size(shape) -> int:
        """Bytes of the kept form of gate and up of this shape."""
        rows, _, groups = _sizes(torch.Size(shape))
        return 2 * rows * groups * (GROUP + 1)

    @property
    def codes(self) -> torch.Tensor:
        rows, _, groups = _sizes(self.shape)
        return self.data[:2 * rows * groups * GROUP].view(torch.int8).view(2, rows, groups * GROUP)

    @property
    def steps(self) -> torch.Tensor:
        rows, _, groups = _sizes(self.shape)
        return self.data[2 * rows * groups * GROUP:].view(2, rows, groups)

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    def dequantize(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values that the codes of gate and up stand for, in fp32 and the inputs' shape."""
        rows, n_cols, groups = _sizes(self.shape)
        exponent = self.steps.to(torch.int32)
        step = torch.where(exponent == 255, 0x7fc00000, exponent << 23).view(torch.float32)
        values = self.codes.view(2, rows, groups, GROUP).to(torch.float32) * step.unsqueeze(-1)
        values = values.view(2, rows, groups * GROUP)[:, :, :n_cols].contiguous().view(2, *self.shape)
        return values[0], values[1]


def _sizes(shape: torch.Size) -> Tuple[int, int, int]:
    """Rows, columns and groups per row of inputs of this shape."""
    n_cols = shape[-1]
    return shape.numel() // n_cols if n_cols else 0, n_cols, (n_cols + GROUP - 1) // GROUP


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


def _rows(x: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """A tensor whose storage holds the rows of ``x`` in order (``x`` itself, or a copy), and their pitch."""
    if x.is_contiguous():
        return x, x.shape[-1]
    v = _row_view(x)
    return (x.contiguous(), x.shape[-1]) if v is None else (v, _pitch(v))


def _pitch(v: torch.Tensor) -> int:
    return v.stride(0) if v.shape[0] > 1 else v.shape[1]


def _input_rows(gate: torch.Tensor, up: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, int]:
    """Both as rows of one pitch: in place when they are (two halves of a packed projection), else copied."""
    if not (gate.is_contiguous() and up.is_contiguous()):
        g, u = _row_view(gate), _row_view(up)
        if g is not None and u is not None and _pitch(g) == _pitch(u):
            return g, u, _pitch(g)
        gate, up = gate.contiguous(), up.contiguous()
    return gate, up, gate.shape[-1]


def _keep(gate, up, activation, gm, dm, want_h: bool, where: str):
    _check_inputs(gate, up)
    shape, dtype, device = gate.shape, gate.dtype, gate.device
    rows, n_cols, groups = _sizes(shape)
    gate, up, pitch = _input_rows(gate, up)
    plane, plane_steps = rows * groups * GROUP, rows * groups
    data = torch.empty(2 * (plane + plane_steps), dtype=torch.uint8, device=device)
    h = torch.empty(shape, dtype=dtype, device=device) if want_h else None
    base = data.data_ptr()
    steps = base + 2 * plane
    _lib.check(
        where,
        _lib.lib.swiglu_b200_ckpt8_fwd(
            h.data_ptr() if want_h else None, base, base + plane, steps, steps + plane_steps, gate.data_ptr(),
            up.data_ptr(), rows, n_cols, pitch, n_cols, _DTYPE_CODE[dtype], ACTIVATIONS[activation], gm, dm,
            device.index, _stream(device),
        ),
    )
    return h, Checkpoint8._of(data, shape, dtype, activation, gm, dm)


def ckpt8_forward(gate: torch.Tensor, up: torch.Tensor, activation: str = "silu", gate_multiplier: float = 1.0,
                  down_multiplier: float = 1.0):
    """``(h, kept)``: ``h = act(gate * gm) * up * dm`` in the shape of ``gate``, and the ``Checkpoint8`` its backward
    needs.  One pass over gate and up; views with a common row pitch (the halves of a packed projection) are read in
    place."""
    _check_activation(activation)
    gm, dm = _check_multipliers(activation, gate_multiplier, down_multiplier)
    return _keep(gate, up, activation, gm, dm, True, "ckpt8_forward")


def ckpt8_pack(gate: torch.Tensor, up: torch.Tensor, activation: str = "silu", gate_multiplier: float = 1.0,
               down_multiplier: float = 1.0) -> Checkpoint8:
    """The ``Checkpoint8`` alone, for a block whose own kernel has made ``h`` (the fused projections)."""
    _check_activation(activation)
    gm, dm = _check_multipliers(activation, gate_multiplier, down_multiplier)
    return _keep(gate, up, activation, gm, dm, False, "ckpt8_pack")[1]


def _gradients(dout, kept: Checkpoint8, dgate: int, dup: int, grad_pitch: int, h, where: str) -> None:
    """Fills dgate and dup (addresses of rows ``grad_pitch`` apart), and ``h`` when it is given."""
    rows, n_cols, groups = _sizes(kept.shape)
    dout, pitch = _rows(dout)
    codes, plane, plane_steps = kept.data.data_ptr(), rows * groups * GROUP, rows * groups
    steps = codes + 2 * plane
    device = kept.device
    _lib.check(
        where,
        _lib.lib.swiglu_b200_ckpt8_bwd(
            h.data_ptr() if h is not None else None, dgate, dup, dout.data_ptr(), codes, codes + plane, steps,
            steps + plane_steps, rows, n_cols, grad_pitch, pitch, n_cols, _DTYPE_CODE[kept.dtype],
            ACTIVATIONS[kept.activation], kept.gate_multiplier, kept.down_multiplier, device.index, _stream(device),
        ),
    )


def _check_dout(dout: torch.Tensor, kept: Checkpoint8) -> None:
    if dout.dtype != kept.dtype or dout.device != kept.device:
        raise TypeError("dout must have the dtype and device of gate and up")
    if dout.shape != kept.shape or kept.data.numel() != Checkpoint8.size(kept.shape):
        raise ValueError(f"dout of shape {tuple(dout.shape)} does not match gate of shape {tuple(kept.shape)}")
    _require_cuda(dout, "dout")


def ckpt8_backward(dout: torch.Tensor, kept: Checkpoint8):
    """``(dgate, dup)`` of a ``ckpt8_forward`` / ``ckpt8_pack``, in the inputs' shape."""
    _check_dout(dout, kept)
    dgate, dup = dout.new_empty(kept.shape), dout.new_empty(kept.shape)
    _gradients(dout, kept, dgate.data_ptr(), dup.data_ptr(), kept.shape[-1], None, "ckpt8_backward")
    return dgate, dup


def ckpt8_backward_recompute(dout: torch.Tensor, kept: Checkpoint8, preserve_inputs: bool = False):
    """``(h, dgate, dup)`` in one pass: the gradients together with ``act(gate * gm) * up * dm`` of the kept values, as
    ``swiglu_backward_recompute`` gives them from gate and up.  Unless ``preserve_inputs`` is set, ``h`` is written
    over ``dout``, which must be contiguous then."""
    if not (preserve_inputs or dout.is_contiguous()):
        raise ValueError("the in-place form needs a contiguous dout; pass preserve_inputs=True")
    _check_dout(dout, kept)
    h = dout.new_empty(kept.shape) if preserve_inputs else dout
    dgate, dup = dout.new_empty(kept.shape), dout.new_empty(kept.shape)
    _gradients(dout, kept, dgate.data_ptr(), dup.data_ptr(), kept.shape[-1], h, "ckpt8_backward_recompute")
    return h, dgate, dup


class ForgeCkpt8Function(torch.autograd.Function):
    """``apply(gate, up, activation="silu", gate_multiplier=1.0, down_multiplier=1.0)``; saves the kept form."""

    @staticmethod
    def forward(ctx, gate, up, activation="silu", gate_multiplier=1.0, down_multiplier=1.0):
        h, kept = ckpt8_forward(gate, up, activation, gate_multiplier, down_multiplier)
        ctx.save_for_backward(kept.data)
        ctx.call = (kept.shape, kept.dtype, kept.activation, kept.gate_multiplier, kept.down_multiplier)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        dgate, dup = ckpt8_backward(dout, Checkpoint8._of(*ctx.saved_tensors, *ctx.call))
        return dgate, dup, None, None, None


class ForgePackedCkpt8Function(torch.autograd.Function):
    """``apply(gate_up, activation="silu", gate_multiplier=1.0, down_multiplier=1.0)`` on the packed layout."""

    @staticmethod
    def forward(ctx, gate_up, activation="silu", gate_multiplier=1.0, down_multiplier=1.0):
        _check_packed_input(gate_up)
        n_cols = gate_up.shape[-1] // 2
        # the two halves of one tensor share a row pitch: nothing is copied unless gate_up itself is not in rows
        packed = gate_up if _row_view(gate_up) is not None else gate_up.contiguous()
        h, kept = ckpt8_forward(packed[..., :n_cols], packed[..., n_cols:], activation, gate_multiplier,
                                down_multiplier)
        ctx.save_for_backward(kept.data)
        ctx.call = (kept.shape, kept.dtype, kept.activation, kept.gate_multiplier, kept.down_multiplier)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        kept = Checkpoint8._of(*ctx.saved_tensors, *ctx.call)
        _check_dout(dout, kept)
        n_cols = kept.shape[-1]
        grad = dout.new_empty((*kept.shape[:-1], 2 * n_cols))
        base = grad.data_ptr()
        _gradients(dout, kept, base, base + n_cols * grad.element_size(), 2 * n_cols, None,
                   "packed ckpt8_backward")
        return grad, None, None, None


def _records(*inputs: torch.Tensor) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in inputs)


def swiglu_ckpt8(gate: torch.Tensor, up: torch.Tensor, gate_multiplier: float = 1.0,
                 down_multiplier: float = 1.0) -> torch.Tensor:
    """``swiglu`` that keeps gate and up in 8 bits for its backward (nothing is kept when no gradient is wanted)."""
    if not _records(gate, up):
        gm, dm = _check_multipliers("silu", gate_multiplier, down_multiplier)
        return swiglu_forward(gate, up, gm, dm)[0]
    return ForgeCkpt8Function.apply(gate, up, "silu", gate_multiplier, down_multiplier)


def swiglu_packed_ckpt8(gate_up: torch.Tensor, gate_multiplier: float = 1.0,
                        down_multiplier: float = 1.0) -> torch.Tensor:
    """``swiglu_packed`` that keeps both halves in 8 bits for its backward."""
    _check_packed_input(gate_up)
    if not _records(gate_up):
        gm, dm = _check_multipliers("silu", gate_multiplier, down_multiplier)
        return swiglu_packed_forward(gate_up, gm, dm)[0]
    return ForgePackedCkpt8Function.apply(gate_up, "silu", gate_multiplier, down_multiplier)


def _gelu(approximate: str) -> str:
    return "gelu_tanh" if _check_approximate(approximate) else "gelu_exact"


def geglu_ckpt8(gate: torch.Tensor, up: torch.Tensor, approximate: str = "tanh") -> torch.Tensor:
    """``geglu`` that keeps gate and up in 8 bits for its backward (nothing is kept when no gradient is wanted)."""
    activation = _gelu(approximate)
    if not _records(gate, up):
        return geglu_forward(gate, up, approximate)[0]
    return ForgeCkpt8Function.apply(gate, up, activation)


def geglu_packed_ckpt8(gate_up: torch.Tensor, approximate: str = "tanh") -> torch.Tensor:
    """``geglu_packed`` that keeps both halves in 8 bits for its backward."""
    _check_packed_input(gate_up)
    activation = _gelu(approximate)
    if not _records(gate_up):
        return geglu_packed_forward(gate_up, approximate)[0]
    return ForgePackedCkpt8Function.apply(gate_up, activation)
