"""Activations kept in 8 bits between the forward and the backward pass.

``save8`` keeps a tensor as e4m3 with one fp32 scale for each 128 elements of its last dimension (``ops/fp8.py``, row
blocks): 1.03 bytes an element instead of 2 or 4, relative error at most 2 ** -4 of a normal e4m3 value.
``silu8`` and ``swiglu8`` are the activations of an MLP with such a copy of their input in place of the input itself: the
output is computed from the input as it is, the gradient from the copy (kernels: ``csrc/kernels/fp8_act.cu``).  The pairs
``silu8_forward`` / ``silu8_backward`` and ``swiglu8_forward`` / ``swiglu8_backward`` are for callers that write their own
backward pass, as ``models/tp_mlp.py`` does.

The reference has no activations and no autograd (README.md:5).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .fp8 import ACT_BACKWARD, ACT_FORWARD, DTYPES, _call, _check_float, _check_scale, _native, _new_payload, _new_scale, _payload
from .fp8 import _rows, _scale_shape, _up16, dequantize_fp8, quantize_fp8


class Saved8(NamedTuple):
    """What ``save8`` keeps: payload and scales of the tensor as a matrix (its last dimension by all others)."""
    data: torch.Tensor
    scale: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.data.numel() + 4 * self.scale.numel()

    def restore(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The tensor again, contiguous, in its own type or ``dtype``."""
        x = dequantize_fp8(self.data, self.scale, "row", dtype or self.dtype)
        return x if len(self.shape) == 2 else x.view(self.shape)


def _matrix(x: torch.Tensor) -> torch.Tensor:
    if x.dim() == 2:
        return x
    cols = x.shape[-1] if x.dim() else 1
    return x.reshape(x.numel() // cols if cols else 0, cols)


def save8(x: torch.Tensor) -> Saved8:
    """Keep ``x`` (fp32, fp16 or bf16, any shape and strides) in 8 bits."""
    _check_float(x, "x")
    return Saved8(*quantize_fp8(_matrix(x.detach()), "row"), x.shape, x.dtype)


def _forward(h: torch.Tensor, u: Optional[torch.Tensor]):
    _check_float(h, "the input")
    if u is not None and (u.shape != h.shape or u.dtype != h.dtype or u.device != h.device):
        raise ValueError("gate and up must be of one shape, type and device")
    h2, u2 = _matrix(h), None if u is None else _matrix(u)
    if not _native(*((h2,) if u is None else (h2, u2))):
        with torch.no_grad():
            hf = h.float()
            y = hf / (1 + torch.exp(-hf))
            y = (y if u is None else y * u.float()).to(h.dtype)
            return y, save8(h), None if u is None else save8(u)
    (rows, cols), dev = h2.shape, h.device
    hd, hs = _new_payload(rows, cols, h2), _new_scale(rows, cols, "row", dev)
    y = h2.new_empty(h.shape)
    h2, ldh = _rows(h2)
    if u is None:
        ud = us = None
        up = 0, 0, 0, 0
    else:
        ud, us = _new_payload(rows, cols, h2), _new_scale(rows, cols, "row", dev)
        u2, ldu = _rows(u2)
        up = u2.data_ptr(), ldu, ud.data_ptr(), us.data_ptr()
    if y.numel():
        _call(ACT_FORWARD, y.get_device(), DTYPES[h.dtype], h2.data_ptr(), ldh, up[0], up[1], rows, cols, y.data_ptr(), cols, _up16(cols),
              hd.data_ptr(), hs.data_ptr(), up[2], up[3])
    return y, Saved8(hd, hs, h.shape, h.dtype), None if u is None else Saved8(ud, us, h.shape, h.dtype)


def _backward(h: Saved8, u: Optional[Saved8], dy: torch.Tensor, act: bool):
    if dy.shape != h.shape or dy.dtype != h.dtype or dy.device != h.data.device:
        raise ValueError("dy must have the shape, type and device of the activation")
    if u is not None and (u.shape != h.shape or u.dtype != h.dtype or u.data.device != h.data.device):
        raise ValueError("gate and up must be of one shape, type and device")
    dy2 = _matrix(dy)
    rows, cols = dy2.shape
    kept = (h,) if u is None else (h, u)
    for k in kept:
        if tuple(k.data.shape) != (rows, cols):
            raise ValueError("the saved payload does not have its tensor's shape")
        _check_scale(k.scale, _scale_shape(rows, cols, "row"), k.data, "scale")
    if not _native(dy2, *(t for k in kept for t in (k.data, k.scale))):
        with torch.no_grad():
            d, x = dy.float(), h.restore(torch.float32)
            p = 1 / (1 + torch.exp(-x))
            slope, s = p * (1 + x * (1 - p)), x * p
            v = torch.ones_like(x) if u is None else u.restore(torch.float32)
            return (d * v * slope).to(dy.dtype), None if u is None else (d * s).to(dy.dtype), (s * v).to(dy.dtype) if act else None
    dy2, ld = _rows(dy2)
    new = lambda want: dy2.new_empty(dy.shape) if want else None      # noqa: E731
    dh, du, y = new(True), new(u is not None), new(act)
    if dh.numel():
        pitch, ins, live = _up16(cols), [], []
        for k in kept:
            data, _ = _payload(k.data, "the saved payload", vectors=True, apart=pitch)     # what was kept may come back otherwise
            live.append(data)
            ins += [data.data_ptr(), k.scale.data_ptr(), *k.scale.stride()]
        if u is None:
            ins += [0, 0, 0, 0]
        _call(ACT_BACKWARD, dh.get_device(), DTYPES[dy.dtype], pitch, *ins, dy2.data_ptr(), ld, rows, cols, dh.data_ptr(),
              du.data_ptr() if u is not None else 0, y.data_ptr() if act else 0)
    return dh, du, y


def silu8_forward(h: torch.Tensor) -> Tuple[torch.Tensor, Saved8]:
    """``(silu(h), h kept in 8 bits)`` in one pass; fp32, fp16 or bf16, any shape."""
    y, saved, _ = _forward(h, None)
    return y, saved


def silu8_backward(saved: Saved8, dy: torch.Tensor, act: bool = False):
    """``dy * silu'(h)`` from the kept copy of ``h``; with ``act`` ``(that, silu(h))``."""
    dh, _, y = _backward(saved, None, dy, act)
    return (dh, y) if act else dh


def swiglu8_forward(gate: torch.Tensor, up: torch.Tensor) -> Tuple[torch.Tensor, Tuple[Saved8, Saved8]]:
    """``(silu(gate) * up, both kept in 8 bits)`` in one pass.  The inputs may be strided, such as the halves of one tensor."""
    y, kg, ku = _forward(gate, up)
    return y, (kg, ku)


def swiglu8_backward(saved: Tuple[Saved8, Saved8], dy: torch.Tensor, act: bool = False):
    """``(dgate, dup)`` from the kept copies; with ``act`` the activation again as a third."""
    dg, du, y = _backward(saved[0], saved[1], dy, act)
    return (dg, du, y) if act else (dg, du)


class _Silu8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h):
        y, saved = silu8_forward(h)
        ctx.save_for_backward(saved.data, saved.scale)
        ctx.meta = saved.shape, saved.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return silu8_backward(Saved8(*ctx.saved_tensors, *ctx.meta), dy)


class _Swiglu8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        y, (kg, ku) = swiglu8_forward(gate, up)
        ctx.save_for_backward(kg.data, kg.scale, ku.data, ku.scale)
        ctx.meta = kg.shape, kg.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        t = ctx.saved_tensors
        return swiglu8_backward((Saved8(t[0], t[1], *ctx.meta), Saved8(t[2], t[3], *ctx.meta)), dy)


def silu8(h: torch.Tensor) -> torch.Tensor:
    """``silu(h)`` that keeps ``h`` in 8 bits for its gradient."""
    _check_float(h, "h")
    return _Silu8.apply(h)


def swiglu8(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` that keeps both in 8 bits for their gradients."""
    _check_float(gate, "gate")
    return _Swiglu8.apply(gate, up)
