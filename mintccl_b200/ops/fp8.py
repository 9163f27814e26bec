"""e4m3 matrices with one fp32 scale per block of 128, their products, and a linear layer trained with them.

Format: an e4m3 payload (``uint8``, or ``torch.float8_e4m3fn`` where a caller has it so) and an fp32 scale for every block of

* ``"row"``: 1 x 128 elements along a row; activations and gradients, scales ``[rows, ceil(cols / 128)]``;
* ``"tile"``: 128 x 128 elements; weights, scales ``[ceil(rows / 128), ceil(cols / 128)]``;
* ``"col"``: 128 x 1 elements down a column; gradients that are summed over their rows, scales ``[ceil(rows / 128), cols]``.

An element stands for payload times scale.  ``quantize_fp8`` takes the smallest power of two (``2 ** -126`` at least) with
which the block's largest finite magnitude is at most 448, the largest e4m3 value, and 1 for a block of zeros: dividing by
it is exact, so the rounding to e4m3 is the only one.  Infinities and NaN become NaN and leave the rest of their block as it
is.  ``gemm_fp8`` takes scales of any value, as checkpoints bring them.

MXFP8 (``ops/mxfp8.py``) has a scale of 8 bits for each 32 elements instead, which the tensor cores apply themselves.
The reference has no fp8 path; it is on its roadmap (README.md:58-60).
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from .. import _native as N
from .mxfp8 import _QUANT_DT as DTYPES
from .mxfp8 import _on_device, _plain_cuda

BLOCK = 128
BLOCKS = {"row": (1, BLOCK), "col": (BLOCK, 1), "tile": (BLOCK, BLOCK)}
Quantized = Tuple[torch.Tensor, torch.Tensor]


def _cdiv(a: int, b: int) -> int:
    return -(-a // b)


def _scale_shape(rows: int, cols: int, block: str) -> Tuple[int, int]:
    br, bc = BLOCKS[block]
    return _cdiv(rows, br), _cdiv(cols, bc)


def _new_payload(rows: int, cols: int, device) -> torch.Tensor:
    """Rows a multiple of 16 bytes apart, as the kernels (and TMA) want them; the padding is not part of the result."""
    pitch = _cdiv(cols, 16) * 16
    buf = torch.empty(rows, pitch, device=device, dtype=torch.uint8)
    return buf if pitch == cols else buf[:, :cols]


def _new_scale(rows: int, cols: int, block: str, device) -> torch.Tensor:
    r, c = _scale_shape(rows, cols, block)
    if block == "row":   # neighbouring rows next to one another: what a warp of the product reads at once
        return torch.empty(c, r, device=device, dtype=torch.float32).t()
    return torch.empty(r, c, device=device, dtype=torch.float32)


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else 0


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` (2-D) with adjacent columns."""
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _payload(t: torch.Tensor, name: str) -> Tuple[torch.Tensor, int]:
    """A payload as the kernels take it, and the bytes between its rows: copied where its rows are not on 16-byte boundaries."""
    if t.dtype not in (torch.uint8, torch.float8_e4m3fn) or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D uint8 or float8_e4m3fn tensor")
    rows, cols = t.shape
    t = t.view(torch.uint8)
    if cols <= 1 or t.stride(1) == 1:
        pitch = t.stride(0) if rows > 1 else _cdiv(cols, 16) * 16
        end = t.storage_offset() + max(rows - 1, 0) * pitch + _cdiv(cols, 16) * 16      # the last row is read in whole vectors too
        if t.data_ptr() % 16 == 0 and pitch % 16 == 0 and pitch >= cols and end <= t.untyped_storage().nbytes():
            return t, pitch
    buf = _new_payload(rows, cols, t.device)
    buf.copy_(t)
    return buf, _cdiv(cols, 16) * 16


def _plain_scale(s: torch.Tensor, shape: Tuple[int, int], like: torch.Tensor, name: str) -> torch.Tensor:
    if s.dtype != torch.float32 or tuple(s.shape) != shape or s.device != like.device:
        raise ValueError(f"{name} must be a float32 tensor of shape {shape} on {like.device}")
    return s


def _check_float(x: torch.Tensor, name: str) -> None:
    if x.dtype not in DTYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")


# ---- encoding and decoding -----------------------------------------------------------------------------------------
def quantize_fp8(x: torch.Tensor, block: str = "row") -> Quantized:
    """fp32 / fp16 / bf16 ``[rows, cols]`` -> (payload uint8 ``[rows, cols]``, scales).  Payload rows are a multiple of 16
    bytes apart; the scales of row blocks are held with neighbouring rows adjacent (strides ``(1, rows)``)."""
    return quantize_fp8_many(x, (block,))[0]


def quantize_fp8_many(x: torch.Tensor, blocks: Sequence[str]) -> List[Quantized]:
    """``[quantize_fp8(x, b) for b in blocks]`` from one pass over ``x``."""
    if x.dim() != 2:
        raise ValueError("x must be 2-D")
    _check_float(x, "x")
    if not blocks or len(set(blocks)) != len(blocks) or any(b not in BLOCKS for b in blocks):
        raise ValueError(f"blocks must be different ones of {sorted(BLOCKS)}")
    if not _plain_cuda(x):
        return [_torch_quantize(x, b) for b in blocks]
    rows, cols = x.shape
    out = {b: (_new_payload(rows, cols, x.device), _new_scale(rows, cols, b, x.device)) for b in blocks}
    if x.numel():
        x = _rows(x)
        ptrs = []
        for b in ("row", "col", "tile"):
            ptrs += [out[b][0].data_ptr(), out[b][1].data_ptr()] if b in out else [None, None]
        _on_device(x, N.lib().mt_fp8_quantize, DTYPES[x.dtype], x.data_ptr(), _row_stride(x), rows, cols, _cdiv(cols, 16) * 16, *ptrs)
    return [out[b] for b in blocks]


def _spread(scale: torch.Tensor, rows: int, cols: int, block: str) -> torch.Tensor:
    """The scale of every element."""
    br, bc = BLOCKS[block]
    return scale.repeat_interleave(br, 0)[:rows].repeat_interleave(bc, 1)[:, :cols]


def _torch_quantize(x: torch.Tensor, block: str) -> Quantized:
    """The same in torch expressions: the path of CPU tensors and the oracle of the kernels."""
    x = x.detach().float()
    rows, cols = x.shape
    br, bc = BLOCKS[block]
    finite = x.isfinite()
    mag = torch.nn.functional.pad(torch.where(finite, x.abs(), torch.zeros_like(x)), (0, -cols % bc, 0, -rows % br))
    r, c = _scale_shape(rows, cols, block)
    m, e = torch.frexp(mag.reshape(r, br, c, bc).amax((1, 3)) if x.numel() else mag.new_zeros(r, c))
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)      # 448 = 0.875 * 2 ** 9
    scale = torch.where(m > 0, ((e + 127) << 23).view(torch.float32), torch.ones_like(m))
    q = torch.where(finite, x / _spread(scale, rows, cols, block), torch.full_like(x, float("nan"))).to(torch.float8_e4m3fn)
    data = _new_payload(rows, cols, x.device).copy_(q.view(torch.uint8))
    return data, (scale.t().contiguous().t() if block == "row" else scale)


def dequantize_fp8(data: torch.Tensor, scale: torch.Tensor, block: str = "row", dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Payload times scale in ``dtype``, contiguous.  A finite value that rounding took past the type's largest stays there."""
    if block not in BLOCKS:
        raise ValueError(f"block must be one of {sorted(BLOCKS)}")
    if dtype not in DTYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    if data.dtype not in (torch.uint8, torch.float8_e4m3fn) or data.dim() != 2:
        raise ValueError("data must be a 2-D uint8 or float8_e4m3fn tensor")
    rows, cols = data.shape
    _plain_scale(scale, _scale_shape(rows, cols, block), data, "scale")
    if not (_plain_cuda(data) and _plain_cuda(scale)):
        top = torch.finfo(dtype).max
        return (data.view(torch.float8_e4m3fn).float() * _spread(scale, rows, cols, block)).clamp(-top, top).to(dtype)
    out = torch.empty(rows, cols, device=data.device, dtype=dtype)
    if out.numel():
        data, pitch = _payload(data, "data")
        br, bc = BLOCKS[block]
        _on_device(data, N.lib().mt_fp8_dequantize, DTYPES[dtype], data.data_ptr(), pitch, scale.data_ptr(), scale.stride(0),
                   scale.stride(1), rows, cols, br, bc, out.data_ptr(), cols)
    return out


# ---- products ------------------------------------------------------------------------------------------------------
def gemm_fp8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, ta: bool = False, tb: bool = False,
             out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16, nctas: int = 0) -> torch.Tensor:
    """``op(a) @ op(b)`` of quantised matrices as they are stored, any sizes (kernel: ``csrc/kernels/gemm_fp8.cu``):

    * ``a [M, K] @ b[N, K].T``: a layer's output; ``a`` in row blocks, ``b`` (the weight) in tiles;
    * ``tb``: ``a [M, K] @ b [K, N]``: the gradient of its input; ``a`` in row blocks, ``b`` in tiles;
    * ``ta`` and ``tb``: ``a[K, M].T @ b [K, N]``: the gradient of its weight; ``a`` in column blocks, ``b`` in tiles.

    Sums are fp32 with one rounding to ``dtype`` (fp32, fp16 or bf16; that of ``out`` where it is given) at the end."""
    if ta and not tb:
        raise ValueError("gemm_fp8: ta goes with tb")
    for t, name in ((a, "a"), (a_scale, "a_scale"), (b, "b"), (b_scale, "b_scale")):
        if not _plain_cuda(t):
            raise ValueError(f"{name} must be a plain CUDA tensor")
        if t.device != a.device:
            raise ValueError("operands must be on one device")
    a, lda = _payload(a, "a")
    b, ldb = _payload(b, "b")
    M, K = (a.shape[1], a.shape[0]) if ta else a.shape
    Nn, K2 = (b.shape[1], b.shape[0]) if tb else b.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    _plain_scale(a_scale, _scale_shape(*a.shape, "col" if ta else "row"), a, "a_scale")
    _plain_scale(b_scale, _scale_shape(*b.shape, "tile"), b, "b_scale")
    if out is None:
        if dtype not in DTYPES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        out = torch.empty(M, Nn, device=a.device, dtype=dtype)
    elif (tuple(out.shape) != (M, Nn) or out.dtype not in DTYPES or out.device != a.device or not _plain_cuda(out)
          or (Nn > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < Nn)):
        raise ValueError("out must be a float32, float16 or bfloat16 CUDA tensor [M, N] with adjacent columns")
    if not out.numel():
        return out
    if K == 0:
        return out.zero_()
    sa_m, sa_k = (a_scale.stride(1), a_scale.stride(0)) if ta else a_scale.stride()
    sb_n, sb_k = (b_scale.stride(1), b_scale.stride(0)) if tb else b_scale.stride()
    _on_device(a, N.lib().mt_gemm_fp8, a.data_ptr(), lda, a_scale.data_ptr(), sa_m, sa_k, b.data_ptr(), ldb, b_scale.data_ptr(),
               sb_n, sb_k, out.data_ptr(), out.stride(0) if M > 1 else Nn, DTYPES[out.dtype], M, Nn, K, int(ta), int(tb), nctas)
    return out


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, w_data, w_scale, keep):
        x2 = x.reshape(-1, x.shape[-1])
        # keep: the weight has a gradient, which contracts over the tokens; what is kept of x for it are tiles, in 8 bits
        q = quantize_fp8_many(x2, ("row", "tile") if keep else ("row",))
        if w_data is None:
            w_data, w_scale = quantize_fp8(w, "tile")
        y = gemm_fp8(*q[0], w_data, w_scale, dtype=x.dtype)
        ctx.save_for_backward(*(q[1] if keep else (None, None)), w_data, w_scale)
        ctx.dtypes = x.dtype, w.dtype
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        xt, xt_scale, w_data, w_scale = ctx.saved_tensors
        want_x, want_w = ctx.needs_input_grad[:2]
        blocks = [b for b, want in (("row", want_x), ("col", want_w)) if want]
        if not blocks:
            return None, None, None, None, None
        q = dict(zip(blocks, quantize_fp8_many(dy.reshape(-1, dy.shape[-1]), blocks)))
        dx = dw = None
        if want_x:
            dx = gemm_fp8(*q["row"], w_data, w_scale, tb=True, dtype=ctx.dtypes[0]).view(*dy.shape[:-1], w_data.shape[1])
        if want_w:
            dw = gemm_fp8(*q["col"], xt, xt_scale, ta=True, tb=True, dtype=ctx.dtypes[1])
        return dx, dw, None, None, None


def linear_fp8(x: torch.Tensor, w: torch.Tensor, w_fp8: Optional[Quantized] = None) -> torch.Tensor:
    """``x [..., K] @ w[N, K].T`` through 8 bits, in ``x``'s type, with both gradients:

        y = row(x) @ tile(w).T      dx = row(dy) @ tile(w)      dw = col(dy).T @ tile(x)

    where row, col and tile are trips through ``quantize_fp8``.  Between the passes ``x`` and ``w`` are kept in 8 bits.
    ``w_fp8``: ``quantize_fp8(w, "tile")`` where the caller has it (one weight, several micro-batches)."""
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError("x must be [..., K] and w [N, K]")
    _check_float(x, "x")
    _check_float(w, "w")
    if not x.is_cuda or x.device != w.device:
        raise ValueError("x and w must be on one CUDA device")
    if 0 in w.shape:
        raise ValueError("w has no elements")
    data, scale = w_fp8 if w_fp8 is not None else (None, None)
    if data is not None and tuple(data.shape) != tuple(w.shape):
        raise ValueError("w_fp8 does not belong to w")
    return _LinearFp8.apply(x, w, data, scale, torch.is_grad_enabled() and w.requires_grad)
