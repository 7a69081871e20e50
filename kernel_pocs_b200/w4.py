"""Gated MLP with 4-bit weights for one to a few hundred tokens: the frozen projections of a block that generates.

With one token, or one per sequence of a small batch, an MLP costs what it takes to read its weights.  Here they are
4-bit codes with a scale (and, optionally, a zero point) for every ``group_size`` columns, and are turned back into
numbers inside the kernel that multiplies them:

    w4_linear(x, w)                      x W^T
    w4_gate_up(x, w_gate, w_up, ...)     act(x Wg^T * gm) * (x Wu^T) * dm in one launch
    w4_mlp(x, w_gate, w_up, w_down, ...) both, one after the other
    quantize_w4(weight, ...)             a ``W4Weight`` from a bf16 / fp16 matrix
    W4Weight(packed, scales, zeros, ...) one from codes that exist already

W[n, k] is ``(code - zero) * scale``; products with x are summed in fp32 and scaled in fp32, and the result is rounded
once to the dtype of x, with any number of tokens.  Up to ``LINEAR_ROWS`` / ``GATE_UP_ROWS`` tokens take these kernels;
more (a prompt) take the weights written out in 16 bits by ``W4Weight.dequantize``, one more rounding per weight (half a
unit of the 16-bit type), and a library product or, for bf16 gate and up, the tensor-core projections of ``fused_mlp`` /
``geglu``.  Those are not for a graph capture, nor for ``k % 8`` or ``n % 16``: the library takes their place there, with
sums in another order, so that a captured prompt may differ from an eager one in the last bit.
Forward only: weights are frozen and an input that wants a gradient is refused.  The reference has no counterpart (its
inference path is bf16, kernels/lora_mlp/experiments/v5/lora_mlp_kernel_v5.py:451-454).  There is no path for tensors that
are not on a CUDA device.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .checkpoint8 import ACTIVATIONS, _check_activation, _check_multipliers, _rows
from .swiglu import _DTYPE_CODE, _stream

DTYPES = (torch.bfloat16, torch.float16)
GROUP_SIZES = (32, 64, 128)
TILE_ROWS, TILE_COLS, CODE_BYTES = 16, 128, 1024
# Tokens up to which the 4-bit kernels are the faster side, bf16 on B200 (4-bit / 16-bit, us; the 4-bit side goes through
# the weights again for every 64 tokens).  Linear 14336 -> 4096: 39.6 / 56.0 with 256 tokens, 70.5 / 65.9 with 384; 4096
# -> 4096: 16.3 / 17.9 and 25.9 / 20.0.  Gate and up 4096 -> 14336: 149.3 / 154.5 with 448, 171.0 / 155.0 with 512.
LINEAR_ROWS, GATE_UP_ROWS = 256, 448
# Tokens of a prompt whose fp32 projections are held at a time where the library makes them.  In 16 bits the projections
# would take less time (fp16 gate and up 4096 -> 11008: 116 instead of 131 us with 512 tokens, 325 instead of 367 with
# 2048), but they would be rounded before the activation, and Inf above 65504.
PIECE_ROWS = 4096


def _ceil(a: int, b: int) -> int:
    return (a + b - 1) // b


# Nibbles of a 32-bit word: the plain order is by column, in a block columns (0, 2, 4, 6, 1, 3, 5, 7).
_TO_BLOCK = (0, 2, 4, 6, 1, 3, 5, 7)
_FROM_BLOCK = (0, 4, 1, 5, 2, 6, 3, 7)


def _shuffle(p: torch.Tensor, order) -> torch.Tensor:
    """Bytes in words of four along the last dimension, with nibble ``order[i]`` of each word moved to place i."""
    q = torch.stack((p & 15, p >> 4), dim=-1).flatten(-2)[..., list(order)]
    return q[..., 0::2] | (q[..., 1::2] << 4)


class W4Weight:
    """A ``[out_features, in_features]`` matrix in 4 bits.

    ``packed``  uint8 ``[n, 16 * ceil(k / 32)]``: byte j of a row holds the codes of columns 2j (low half) and 2j + 1;
    ``scales``  bf16 or fp16 ``[n, ceil(k / group_size)]``, the dtype of the tokens it multiplies;
    ``zeros``   uint8 of the shape of ``scales``, 0..15, or ``None`` for 8 everywhere.

    The constructor lays them out once in ``blocks``, the form the kernels read (``swiglu_b200_w4_linear`` in the C
    header), and keeps only that; ``packed``, ``scales`` and ``zeros`` are rebuilt on request."""

    __slots__ = ("_blocks", "dtype", "out_features", "in_features", "group_size", "has_zeros")

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *,
                 in_features: int, group_size: int = 128):
        if group_size not in GROUP_SIZES:
            raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size}")
        if packed.dim() != 2 or packed.shape[0] < 1 or in_features < 1:
            raise ValueError("packed must be a [n, bytes] matrix of at least one row and one column")
        n, k = packed.shape[0], int(in_features)
        if packed.dtype != torch.uint8:
            raise TypeError(f"packed must be uint8, got {packed.dtype}")
        if packed.shape[1] != 16 * _ceil(k, 32):
            raise ValueError(f"packed needs {16 * _ceil(k, 32)} bytes per row for {k} columns, got {packed.shape[1]}")
        if scales.dtype not in DTYPES:
            raise TypeError(f"scales must be bf16 or fp16, got {scales.dtype}")
        if scales.shape != (n, _ceil(k, group_size)):
            raise ValueError(f"scales must be of shape {(n, _ceil(k, group_size))}, got {tuple(scales.shape)}")
        if zeros is not None:
            if zeros.dtype != torch.uint8:
                raise TypeError(f"zeros must be uint8, got {zeros.dtype}")
            if zeros.shape != scales.shape:
                raise ValueError(f"zeros must be of shape {tuple(scales.shape)}, got {tuple(zeros.shape)}")
            if int(zeros.max()) > 15:
                raise ValueError("zeros must lie in 0..15")
        if any(t is not None and t.device != packed.device for t in (scales, zeros)):
            raise ValueError("packed, scales and zeros must be on one device")
        self.dtype, self.out_features, self.in_features, self.group_size = scales.dtype, n, k, group_size
        self.has_zeros = zeros is not None
        rows, cols = self._tiles()
        # [row tile, 2, 8, column tile, word u, lane t, byte] -> [row tile, column tile, 2, 8, t, u, byte]
        p = torch.nn.functional.pad(packed, (0, 64 * cols - packed.shape[1], 0, TILE_ROWS * rows - n))
        p = _shuffle(p.reshape(rows, 2, 8, cols, 4, 4, 4), _TO_BLOCK)
        parts = [p.permute(0, 3, 1, 2, 5, 4, 6).reshape(rows, cols, -1), self._tile_groups(scales)]
        if zeros is not None:
            parts.append(self._tile_groups(zeros))
        self._blocks = torch.cat(parts, dim=2)

    @property
    def blocks(self) -> torch.Tensor:
        """uint8 ``[row tiles, column tiles, bytes of a block]``."""
        return self._blocks

    def _operand(self):
        # the address is asked for at every call: a copy of this object has blocks of its own
        return self._blocks.data_ptr(), self.has_zeros

    def _tiles(self):
        return _ceil(self.out_features, TILE_ROWS), _ceil(self.in_features, TILE_COLS)

    def _tile_groups(self, t: torch.Tensor) -> torch.Tensor:
        """[n, groups] -> bytes [row tile, column tile, (8, group, 2)], zero past the matrix."""
        (rows, cols), per = self._tiles(), TILE_COLS // self.group_size
        t = torch.nn.functional.pad(t, (0, cols * per - t.shape[1], 0, TILE_ROWS * rows - t.shape[0]))
        t = t.reshape(rows, 2, 8, cols, per).permute(0, 3, 2, 4, 1).reshape(rows, cols, -1)
        return t.contiguous().view(torch.uint8)

    def _untile_groups(self, lo: int, dtype: torch.dtype) -> torch.Tensor:
        (rows, cols), per = self._tiles(), TILE_COLS // self.group_size
        t = self._blocks[:, :, lo:lo + 16 * per * dtype.itemsize].contiguous().view(dtype)
        t = t.view(rows, cols, 8, per, 2).permute(0, 4, 2, 1, 3).reshape(TILE_ROWS * rows, cols * per)
        return t[:self.out_features, :_ceil(self.in_features, self.group_size)].contiguous()

    @property
    def packed(self) -> torch.Tensor:
        rows, cols = self._tiles()
        p = self._blocks[:, :, :CODE_BYTES].reshape(rows, cols, 2, 8, 4, 4, 4).permute(0, 2, 3, 1, 5, 4, 6)
        p = _shuffle(p, _FROM_BLOCK).reshape(TILE_ROWS * rows, 64 * cols)
        return p[:self.out_features, :16 * _ceil(self.in_features, 32)].contiguous()

    @property
    def scales(self) -> torch.Tensor:
        return self._untile_groups(CODE_BYTES, self.dtype)

    @property
    def zeros(self) -> Optional[torch.Tensor]:
        if not self.has_zeros:
            return None
        return self._untile_groups(CODE_BYTES + 32 * (TILE_COLS // self.group_size), torch.uint8)

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.out_features, self.in_features))

    @property
    def device(self) -> torch.device:
        return self._blocks.device

    @property
    def nbytes(self) -> int:
        """Bytes the kernels read of it."""
        return self._blocks.numel()

    def to(self, device) -> "W4Weight":
        """This weight on ``device`` (itself when it is there already).  Its type cannot be changed."""
        if not isinstance(device, (str, int, torch.device)):
            raise TypeError(f"W4Weight.to takes a device, got {device!r}")
        moved = self._blocks.to(torch.device(device))
        if moved is self._blocks:
            return self
        other = object.__new__(W4Weight)
        for name in ("dtype", "out_features", "in_features", "group_size", "has_zeros"):
            setattr(other, name, getattr(self, name))
        other._blocks = moved
        return other

    def dequantize(self) -> torch.Tensor:
        """``[out_features, in_features]`` in the dtype of the scales: ``(code - zero) * scale`` rounded once."""
        if not self._blocks.is_cuda:
            raise RuntimeError("W4Weight.dequantize has a CUDA (sm_100a) kernel only; there is no CPU fallback")
        n, k = self.shape
        out = torch.empty((n, k), dtype=self.dtype, device=self.device)
        _lib.check(
            "W4Weight.dequantize",
            _lib.lib.swiglu_b200_w4_dequantize(out.data_ptr(), *self._operand(), n, k, k, self.group_size,
                                               _DTYPE_CODE[self.dtype], self.device.index, _stream(self.device)),
        )
        return out


def quantize_w4(weight: torch.Tensor, group_size: int = 128, zero_points: bool = False,
                dtype: Optional[torch.dtype] = None) -> W4Weight:
    """``weight`` ``[n, k]`` in 4 bits, rounded to nearest.  Every ``group_size`` columns of a row share a scale of
    ``dtype`` (the weight's own by default): the group's largest magnitude over 7, or with ``zero_points`` its range
    (zero included) over 15."""
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size}")
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be a non-empty matrix, got shape {tuple(weight.shape)}")
    dtype = weight.dtype if dtype is None else dtype
    if dtype not in DTYPES or not weight.is_floating_point():
        raise TypeError(f"4-bit weights carry bf16 or fp16 scales, got {dtype}")
    n, k = weight.shape
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("weight holds values that are not finite")
    groups, pitch = _ceil(k, group_size), 32 * _ceil(k, 32)
    packed = torch.empty((n, pitch // 2), dtype=torch.uint8, device=weight.device)
    scales = torch.empty((n, groups), dtype=dtype, device=weight.device)
    zeros = torch.empty((n, groups), dtype=torch.uint8, device=weight.device) if zero_points else None
    step = max(1, (1 << 26) // (groups * group_size))  # rows at a time: a quarter of a gigabyte of fp32
    for lo in range(0, n, step):
        w = weight[lo:lo + step].detach().to(torch.float32)
        rows = w.shape[0]
        w = torch.nn.functional.pad(w, (0, groups * group_size - k)).view(rows, groups, group_size)
        if zero_points:
            low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
            scale = ((high - low) / 15).to(dtype)
        else:
            scale = (w.abs().amax(-1) / 7).to(dtype)
        if not bool(torch.isfinite(scale).all()):
            raise ValueError(f"weight holds magnitudes whose scale is not a finite {dtype}")
        # 1 / scale leaves fp32 for scales below 2^-128: these are lifted, with their weights, by a power of two
        lift = torch.where(scale < 2.0 ** -100, 2.0 ** 60, 1.0).to(torch.float32)
        inverse = torch.where(scale > 0, 1.0 / (scale.to(torch.float32) * lift), 0.0)
        if zero_points:
            zero = torch.round(-(low * lift) * inverse).clamp(0, 15)
            zeros[lo:lo + step] = zero.to(torch.uint8)
        else:
            zero = torch.full_like(inverse, 8.0)
        code = (torch.round(w * lift.unsqueeze(-1) * inverse.unsqueeze(-1)) + zero.unsqueeze(-1)).clamp(0, 15).to(torch.uint8)
        code = torch.nn.functional.pad(code.view(rows, -1), (0, max(0, pitch - groups * group_size)))[:, :pitch]
        packed[lo:lo + step] = code[:, 0::2] | (code[:, 1::2] << 4)
        scales[lo:lo + step] = scale
    return W4Weight(packed, scales, zeros, in_features=k, group_size=group_size)


def _check_tokens(x: torch.Tensor, w: W4Weight, what: str) -> None:
    if not (x.is_cuda and w._blocks.is_cuda):
        raise RuntimeError(f"{what} has a CUDA (sm_100a) kernel only; there is no CPU fallback")
    if x.device != w.device:
        raise ValueError(f"x is on {x.device}, the weight on {w.device}")
    if x.dtype != w.dtype:
        raise TypeError(f"x is {x.dtype}, the weight's scales are {w.dtype}")
    if x.dim() == 0 or x.shape[-1] != w.in_features:
        raise ValueError(f"x of shape {tuple(x.shape)} does not end in the weight's {w.in_features} features")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError(f"{what} is forward only (frozen 4-bit weights): call it under torch.no_grad()")


def _aligned_rows(x: torch.Tensor):
    """The rows of ``x`` where every row starts on a 16-byte boundary, as the kernels need them, and their pitch; copied
    into padded rows when they do not."""
    rows, pitch = _rows(x)
    if rows.data_ptr() % 16 == 0 and (pitch % 8 == 0 or x.shape[:-1].numel() == 1):
        return rows, pitch
    k = x.shape[-1]
    pitch = 8 * _ceil(k, 8)
    rows = x.new_empty((*x.shape[:-1], pitch))
    rows[..., :k] = x
    return rows, pitch


def w4_linear(x: torch.Tensor, weight: W4Weight) -> torch.Tensor:
    """``x W^T`` for ``x`` ``[..., in_features]`` of the weight's dtype."""
    _check_tokens(x, weight, "w4_linear")
    n, k = weight.out_features, weight.in_features
    m = x.numel() // k
    if m > LINEAR_ROWS:
        with torch.autocast("cuda", enabled=False):  # which does not reach the 4-bit kernels either
            return x @ weight.dequantize().t()
    y = x.new_empty((m, n) if x.dim() == 2 else (*x.shape[:-1], n))
    x, pitch = _aligned_rows(x)
    device = x.device
    _lib.check(
        "w4_linear",
        _lib.lib.swiglu_b200_w4_linear(y.data_ptr(), x.data_ptr(), *weight._operand(), m, n, k, pitch, n,
                                       weight.group_size, _DTYPE_CODE[x.dtype], device.index, _stream(device)),
    )
    return y


def _gate_up_16bit(x, w_gate, w_up, activation, gm, dm):
    """The same stage from weights written out in 16 bits, for more tokens than the 4-bit kernels are for.  Here too the
    projections stay in fp32 up to the activation."""
    from .fused_mlp import gate_up_swiglu_forward
    from .geglu import gate_up_geglu_forward, geglu_forward
    from .swiglu import swiglu_forward

    wg, wu = w_gate.dequantize(), w_up.dequantize()
    n, k = wg.shape
    approximate = "tanh" if activation == "gelu_tanh" else "none"
    # the fused projections report through status words that belong to launches, not to a graph's replays
    if x.dtype == torch.bfloat16 and k % 8 == 0 and n % 16 == 0 and not torch.cuda.is_current_stream_capturing():
        if x.data_ptr() % 16:
            x = x.clone(memory_format=torch.contiguous_format)  # they start at 16-byte boundaries
        if activation == "silu":
            return gate_up_swiglu_forward(x, wg, wu, gm, dm)
        return gate_up_geglu_forward(x, wg, wu, approximate)
    h = x.new_empty((*x.shape[:-1], n))
    with torch.autocast("cuda", enabled=False):
        for rows, out in zip(x.reshape(-1, k).split(PIECE_ROWS), h.view(-1, n).split(PIECE_ROWS)):
            gate, up = (torch.mm(rows, w.t(), out_dtype=torch.float32) for w in (wg, wu))
            out.copy_((swiglu_forward(gate, up, gm, dm) if activation == "silu" else
                       geglu_forward(gate, up, approximate))[0])
    return h


def w4_gate_up(x: torch.Tensor, w_gate: W4Weight, w_up: W4Weight, activation: str = "silu",
               gate_multiplier: float = 1.0, down_multiplier: float = 1.0) -> torch.Tensor:
    """``act(x Wg^T * gate_multiplier) * (x Wu^T) * down_multiplier``; both projections and the activation (``"silu"``,
    ``"gelu_tanh"`` or ``"gelu_exact"``; the GELU forms have no multipliers) in one launch up to ``GATE_UP_ROWS`` tokens;
    the projections are not rounded to 16 bits on the way, however many there are."""
    _check_activation(activation)
    gm, dm = _check_multipliers(activation, gate_multiplier, down_multiplier)
    n, k = w_gate.out_features, w_gate.in_features
    if (n != w_up.out_features or k != w_up.in_features or w_gate.group_size != w_up.group_size
            or w_gate.dtype != w_up.dtype or w_gate.device != w_up.device):
        raise ValueError("w_gate and w_up must agree in shape, group size, dtype and device")
    _check_tokens(x, w_gate, "w4_gate_up")
    m = x.numel() // k
    if m > GATE_UP_ROWS:
        return _gate_up_16bit(x, w_gate, w_up, activation, gm, dm)
    h = x.new_empty((m, n) if x.dim() == 2 else (*x.shape[:-1], n))
    x, pitch = _aligned_rows(x)
    device = x.device
    _lib.check(
        "w4_gate_up",
        _lib.lib.swiglu_b200_w4_gate_up(
            h.data_ptr(), x.data_ptr(), *w_gate._operand(), *w_up._operand(), m, n, k, pitch, n, w_gate.group_size,
            _DTYPE_CODE[x.dtype], ACTIVATIONS[activation], gm, dm, device.index, _stream(device),
        ),
    )
    return h


def w4_mlp(x: torch.Tensor, w_gate: W4Weight, w_up: W4Weight, w_down: W4Weight,
           activation: str = "silu") -> torch.Tensor:
    """``down(act(gate(x)) * up(x))`` with all three projections in 4 bits: two launches for a few tokens."""
    return w4_linear(w4_gate_up(x, w_gate, w_up, activation), w_down)
