"""e4m3 matrices with one fp32 scale per block of 128, their products, and a linear layer trained with them.

Format: an e4m3 payload (``uint8``, or ``torch.float8_e4m3fn`` where a caller has it so) and an fp32 scale for every block of

* ``"row"``: 1 x 128 elements along a row; activations and gradients, scales ``[rows, ceil(cols / 128)]``;
* ``"tile"``: 128 x 128 elements; weights, scales ``[ceil(rows / 128), ceil(cols / 128)]``;
* ``"col"``: 128 x 1 elements down a column; gradients that are summed over their rows, scales ``[ceil(rows / 128), cols]``.

An element stands for payload times scale.  ``quantize_fp8`` takes the smallest power of two (``2 ** -126`` at least) with
which the block's largest finite magnitude is at most 448, the largest e4m3 value, and 1 for a block of zeros: dividing by
it is exact, so the rounding to e4m3 is the only one.  Infinities and NaN become NaN and leave the rest of their block as it
is.  ``gemm_fp8`` takes scales of any value, as checkpoints bring them.

Waits inside the product kernels are bounded, as in the collectives: one that runs out ends the kernel, whose output is then
not valid.  ``check`` says so, as ``Communicator.check`` does for collectives.

MXFP8 (``ops/mxfp8.py``) has a scale of 8 bits for each 32 elements instead, which the tensor cores apply themselves.
The reference has no fp8 path; it is on its roadmap (README.md:58-60).
"""
from __future__ import annotations

import struct
from typing import List, Optional, Sequence, Tuple, Union

import torch

from .. import _native as N
from .mxfp8 import _QUANT_DT as DTYPES
from .mxfp8 import _bits, _plain_cuda

BLOCK = 128
BLOCKS = {"row": (1, BLOCK), "col": (BLOCK, 1), "tile": (BLOCK, BLOCK)}
Quantized = Tuple[torch.Tensor, torch.Tensor]
QUANTIZE, DEQUANTIZE, ACT_FORWARD, ACT_BACKWARD, GEMM, LINEAR_FORWARD, LINEAR_BACKWARD = range(7)
_PACK = [struct.Struct(f"{n}q").pack for n in range(24)]
_U8 = (torch.uint8, torch.float8_e4m3fn)
_TYPES = (torch.Tensor, torch.nn.Parameter)
_packed = None


def _call(op: int, device: int, *args: int) -> None:
    """Operation ``op`` (``mt_fp8_packed``) on the current stream of ``device``, with that device current."""
    global _packed
    if _packed is None:
        _packed = N.lib().mt_fp8_packed
    if device == torch._C._cuda_getDevice():
        rc = _packed(N.raw_stream(device), op, _PACK[len(args)](*args))
    else:
        with torch.cuda.device(device):
            rc = _packed(N.raw_stream(device), op, _PACK[len(args)](*args))
    if rc < 0:
        raise RuntimeError(f"mt_fp8 operation {op}: {N.last_error()}")


def _address(t: torch.Tensor) -> int:
    """Where ``t`` is on a GPU, or 0: it is elsewhere, has no elements, or does not stand for its own memory (what vmap,
    functionalisation and lazy zeros make has no address or none to be asked for)."""
    if type(t) not in _TYPES or not t.is_cuda or t.is_neg():
        return 0
    try:
        return t.data_ptr()
    except RuntimeError:
        return 0


def _native(*ts: torch.Tensor) -> bool:
    """Whether kernels may be pointed at all of these; tensors without elements count."""
    if torch._C._get_tracing_state() is not None or torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() != 0:
        return False        # somebody records or replaces operations: a kernel launched from here would be missing from the record
    for t in ts:
        if not (_address(t) or (t.numel() == 0 and _plain_cuda(t))):
            return False
    return True


def _up16(n: int) -> int:
    return (n + 15) & ~15


def _scale_shape(rows: int, cols: int, block: str) -> Tuple[int, int]:
    br, bc = BLOCKS[block]
    return -(-rows // br), -(-cols // bc)


def _new_payload(rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    """On ``like``'s device.  Rows a multiple of 16 bytes apart, as the kernels (and TMA) want them; the padding is not part of
    the result."""
    pitch = (cols + 15) & ~15
    buf = like.new_empty((rows, pitch), dtype=torch.uint8)
    return buf if pitch == cols else buf[:, :cols]


def _new_scale(rows: int, cols: int, block: str, device) -> torch.Tensor:
    r, c = _scale_shape(rows, cols, block)
    # row blocks: neighbouring rows next to one another, what a warp of the product reads at once
    return torch.empty_strided((r, c), (1, r) if block == "row" else (c, 1), device=device, dtype=torch.float32)


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """``t`` (2-D) with adjacent columns, and the elements between its rows."""
    (rows, cols), (ld, inner) = t.shape, t.stride()
    if cols > 1 and inner != 1:
        return t.contiguous(), cols
    return t, ld if rows > 1 else 0


def _payload(t: torch.Tensor, name: str, vectors: bool = False, apart: int = 0) -> Tuple[torch.Tensor, int]:
    """A payload as the kernels take it, and the bytes between its rows: copied where its rows are not on 16-byte boundaries,
    not ``apart`` bytes apart (the kernel wants its payloads alike), or (``vectors``: the kernel reads whole ones) where the
    last row's padding is not there to be read."""
    if t.dtype not in _U8 or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D uint8 or float8_e4m3fn tensor")
    (rows, cols), (pitch, inner) = t.shape, t.stride()
    if rows <= 1:
        pitch = _up16(cols)
    if (cols <= 1 or inner == 1) and pitch % 16 == 0 and pitch >= cols and t.data_ptr() % 16 == 0 and apart in (0, pitch):
        if not vectors or cols % 16 == 0:
            return t, pitch
        if t.storage_offset() + (rows - 1) * pitch + _up16(cols) <= t.untyped_storage().nbytes():
            return t, pitch
    buf = _new_payload(rows, cols, t)
    buf.copy_(t.view(torch.uint8))      # bytes: from float8 a copy would convert
    return buf, _up16(cols)


def _check_scale(s: torch.Tensor, shape: Tuple[int, int], like: torch.Tensor, name: str) -> torch.Tensor:
    if s.dtype != torch.float32 or s.shape != shape or s.device != like.device:
        raise ValueError(f"{name} must be a float32 tensor of shape {shape} on {like.device}")
    return s


def _check_float(x: torch.Tensor, name: str) -> None:
    if x.dtype not in DTYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")


# ---- encoding and decoding -----------------------------------------------------------------------------------------
def quantize_fp8(x: torch.Tensor, block: str = "row") -> Quantized:
    """fp32 / fp16 / bf16 ``[rows, cols]`` -> (payload uint8 ``[rows, cols]``, scales).  Payload rows are a multiple of 16
    bytes apart; the scales of row blocks are held with neighbouring rows adjacent (strides ``(1, rows)``)."""
    if block == "row" and x.dim() == 2 and x.dtype in DTYPES and _native(x):    # as below, for the small calls of a decode step
        rows, cols = x.shape
        kb = -(-cols // BLOCK)
        data, scale = _new_payload(rows, cols, x), torch.empty_strided((rows, kb), (1, rows), device=x.device, dtype=torch.float32)
        if rows and cols:
            x, ld = _rows(x)
            _call(QUANTIZE, x.get_device(), DTYPES[x.dtype], x.data_ptr(), ld, rows, cols, (cols + 15) & ~15, data.data_ptr(),
                  scale.data_ptr(), 0, 0, 0, 0)
        return data, scale
    return quantize_fp8_many(x, (block,))[0]


def quantize_fp8_many(x: torch.Tensor, blocks: Sequence[str]) -> List[Quantized]:
    """``[quantize_fp8(x, b) for b in blocks]`` from one pass over ``x``."""
    if x.dim() != 2:
        raise ValueError("x must be 2-D")
    _check_float(x, "x")
    if not blocks or len(set(blocks)) != len(blocks) or any(b not in BLOCKS for b in blocks):
        raise ValueError(f"blocks must be different ones of {sorted(BLOCKS)}")
    if not _native(x):
        return [_torch_quantize(x, b) for b in blocks]
    rows, cols = x.shape
    out = {b: (_new_payload(rows, cols, x), _new_scale(rows, cols, b, x.device)) for b in blocks}
    if x.numel():
        x, ld = _rows(x)
        ptrs = [0] * 6
        for b, (data, scale) in out.items():
            at = 0 if b == "row" else 2 if b == "col" else 4
            ptrs[at], ptrs[at + 1] = data.data_ptr(), scale.data_ptr()
        _call(QUANTIZE, x.get_device(), DTYPES[x.dtype], x.data_ptr(), ld, rows, cols, _up16(cols), *ptrs)
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
    scale = torch.where(m > 0, _bits((e + 127) << 23, torch.float32), torch.ones_like(m))
    q = torch.where(finite, x / _spread(scale, rows, cols, block), torch.full_like(x, float("nan"))).to(torch.float8_e4m3fn)
    data = _new_payload(rows, cols, x).copy_(_bits(q, torch.uint8))
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
    _check_scale(scale, _scale_shape(rows, cols, block), data, "scale")
    if not _native(data, scale):
        top = torch.finfo(dtype).max
        return (_bits(data, torch.float8_e4m3fn).float() * _spread(scale, rows, cols, block)).clamp(-top, top).to(dtype)
    out = data.new_empty((rows, cols), dtype=dtype)
    if out.numel():
        data, pitch = _payload(data, "data", vectors=True)
        br, bc = BLOCKS[block]
        _call(DEQUANTIZE, out.get_device(), DTYPES[dtype], data.data_ptr(), pitch, scale.data_ptr(), *scale.stride(), rows, cols, br, bc,
              out.data_ptr(), cols)
    return out


# ---- products ------------------------------------------------------------------------------------------------------
def gemm_fp8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, ta: bool = False, tb: bool = False,
             out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16, nctas: int = 0,
             power_of_two: bool = False) -> torch.Tensor:
    """``op(a) @ op(b)`` of quantised matrices as they are stored, any sizes (kernel: ``csrc/kernels/gemm_fp8.cu``):

    * ``a [M, K] @ b[N, K].T``: a layer's output; ``a`` in row blocks, ``b`` (the weight) in tiles;
    * ``tb``: ``a [M, K] @ b [K, N]``: the gradient of its input; ``a`` in row blocks, ``b`` in tiles;
    * ``ta`` and ``tb``: ``a[K, M].T @ b [K, N]``: the gradient of its weight; ``a`` in column blocks, ``b`` in tiles.

    Sums are fp32, and the product of two blocks' scales has to be in that range too, with one rounding to ``dtype`` (fp32,
    fp16 or bf16; that of ``out`` where it is given) at the end.  ``power_of_two``: the caller's word that every scale is one
    (``quantize_fp8`` makes no others), which large products are faster for, the tensor cores then apply them; a scale that is
    not may make what it belongs to NaN.  There are no torch expressions behind the products: under a dispatch mode (a flop
    counter, selective checkpointing) and for tensors that do not stand for their own memory they raise ``ValueError``."""
    if ta and not tb:
        raise ValueError("gemm_fp8: ta goes with tb")
    if not _native(a, a_scale, b, b_scale):
        raise ValueError("operands must be plain CUDA tensors, and nobody recording")
    device = a.device
    a, lda = _payload(a, "a")
    b, ldb = _payload(b, "b")
    if b.device != device:
        raise ValueError("operands must be on one device")
    sa, sb = a.shape, b.shape
    M, K = (sa[1], sa[0]) if ta else sa
    Nn, K2 = (sb[1], sb[0]) if tb else sb
    if K != K2:
        raise ValueError("inner dimensions differ")
    kb = -(-K // BLOCK)
    _check_scale(a_scale, (kb, M) if ta else (M, kb), a, "a_scale")
    _check_scale(b_scale, _scale_shape(*sb, "tile"), b, "b_scale")
    if out is None:
        if dtype not in DTYPES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        out, ldc = a.new_empty((M, Nn), dtype=dtype), Nn
    else:
        ldc = out.stride(0) if out.dim() == 2 and M > 1 else Nn
        if (tuple(out.shape) != (M, Nn) or out.dtype not in DTYPES or out.device != device or not _native(out)
                or (Nn > 1 and out.stride(1) != 1) or ldc < Nn):
            raise ValueError("out must be a float32, float16 or bfloat16 CUDA tensor [M, N] with adjacent columns")
    if not out.numel():
        return out
    if K == 0:
        return out.zero_()
    sa_r, sa_c = a_scale.stride()
    sb_r, sb_c = b_scale.stride()
    _call(GEMM, out.get_device(), a.data_ptr(), lda, a_scale.data_ptr(), *((sa_c, sa_r) if ta else (sa_r, sa_c)), b.data_ptr(), ldb,
          b_scale.data_ptr(), *((sb_c, sb_r) if tb else (sb_r, sb_c)), out.data_ptr(), ldc, DTYPES[out.dtype], M, Nn, K, int(ta), int(tb),
          nctas, int(power_of_two))
    return out


def check(device: Optional[Union[int, str, torch.device]] = None) -> None:
    """Raises ``RuntimeError`` if a wait inside a product (``gemm_fp8``, either pass of ``linear_fp8``) ran out on ``device`` (the
    current one by default) since the last check: something that was returned since then is not valid.  Waits for all work on
    the device: for the end of a step, not for a captured one."""
    if device is not None:
        with torch.cuda.device(device):
            return check()
    rc = N.lib().mt_gemm_fp8_error()
    if rc < 0:
        raise RuntimeError(f"mt_gemm_fp8_error: {N.last_error()}")
    if rc:
        raise RuntimeError("a wait inside a block-scaled product ran out: results since the last check are not valid")


# ---- the linear layer ----------------------------------------------------------------------------------------------
def _check_encoded(data: torch.Tensor, scale: torch.Tensor, shape: Tuple[int, int], like: torch.Tensor) -> None:
    if data.shape != shape or data.dtype not in _U8 or not _native(data, scale) or data.device != like.device:
        raise ValueError("w_fp8 does not belong to w")
    _check_scale(scale, _scale_shape(*shape, "tile"), data, "the scales of w_fp8")


def _room(nbytes: int) -> int:
    """Areas of one buffer start 256 bytes apart: allocating each by itself is most of a small layer's time."""
    return (nbytes + 255) & ~255


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, w_data, w_scale, keep, power_of_two):
        # keep: the weight has a gradient, which contracts over the tokens; what is kept of x for it are tiles, in 8 bits
        n, k = w.shape
        x2, ldx = _rows(x if x.dim() == 2 else x.reshape(-1, k))
        t, pk, kb, own = x2.shape[0], (k + 15) & ~15, -(-k // BLOCK), w_data is None
        # one buffer: x's tiles and their scales, w's tiles and theirs
        xs = _room(t * pk) if keep else 0
        wd = xs + (_room(4 * -(-t // BLOCK) * kb) if keep else 0)
        ws = wd + (_room(n * pk) if own else 0)
        size = ws + (4 * -(-n // BLOCK) * kb if own else 0)
        kept = x2.new_empty(size, dtype=torch.uint8) if size else None
        base = kept.data_ptr() if size else 0
        ctx.sizes = t, n, k, xs, wd, ws, size, x.dtype, w.dtype, power_of_two
        ctx.save_for_backward(kept, w_data, w_scale)
        y = x2.new_empty((t, n) if x.dim() == 2 else (*x.shape[:-1], n))
        if own:
            w2, ldw = _rows(w)
            wq = w2.data_ptr(), ldw, base + wd, pk, base + ws, kb, 1
        else:
            w2, pitch = _payload(w_data, "w_fp8")
            wq = 0, 0, w2.data_ptr(), pitch, w_scale.data_ptr(), *w_scale.stride()
        if t:
            rows = x2.new_empty(_room(t * pk) + 4 * t * kb, dtype=torch.uint8)      # x's row blocks, for this product only
            at = rows.data_ptr()
            _call(LINEAR_FORWARD, y.get_device(), DTYPES[x.dtype], x2.data_ptr(), ldx, t, k, DTYPES[w.dtype], wq[0], wq[1], n, at,
                  at + _room(t * pk), base if keep else 0, base + xs if keep else 0, *wq[2:], y.data_ptr(), int(power_of_two))
        elif own:
            _call(QUANTIZE, y.get_device(), DTYPES[w.dtype], wq[0], wq[1], n, k, pk, 0, 0, 0, 0, wq[2], wq[4])
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        kept, w_data, w_scale = ctx.saved_tensors
        t, n, k, xs, wd, ws, size, x_dtype, w_dtype, power_of_two = ctx.sizes
        want_x, want_w = ctx.needs_input_grad[:2]
        if not _native(dy):
            raise ValueError("the gradient must be a plain CUDA tensor, and nobody recording")
        base = 0
        if size:   # what a saved-tensor hook made of it
            if kept.dtype != torch.uint8 or kept.numel() != size or kept.device != dy.device or not _native(kept):
                raise ValueError("what was kept for the gradient came back as another tensor")
            kept = kept.contiguous()
            if kept.data_ptr() % 16:
                kept = kept.clone()
            base = kept.data_ptr()
        if w_data is None:
            w2, wq = None, (base + wd, (k + 15) & ~15, base + ws, -(-k // BLOCK), 1)
        else:
            _check_encoded(w_data, w_scale, (n, k), dy)
            w2, pitch = _payload(w_data, "w_fp8")
            wq = w2.data_ptr(), pitch, w_scale.data_ptr(), *w_scale.stride()
        dx = dy.new_empty((*dy.shape[:-1], k), dtype=x_dtype) if want_x else None
        dw = dy.new_empty((n, k), dtype=w_dtype) if want_w else None
        if t and (want_x or want_w):
            dy2, ld = _rows(dy if dy.dim() == 2 else dy.reshape(-1, n))
            # dy's row blocks and their scales, its column blocks and theirs
            pn = (n + 15) & ~15
            rs = _room(t * pn) if want_x else 0
            cd = rs + (_room(4 * t * -(-n // BLOCK)) if want_x else 0)
            cs = cd + (_room(t * pn) if want_w else 0)
            tmp = dy2.new_empty(cs + (4 * -(-t // BLOCK) * n if want_w else 0), dtype=torch.uint8)
            at = tmp.data_ptr()
            _call(LINEAR_BACKWARD, dy2.get_device(), DTYPES[x_dtype], dy2.data_ptr(), ld, t, n, k, at, at + rs, *wq,
                  dx.data_ptr() if want_x else 0, at + cd, at + cs, base, base + xs, dw.data_ptr() if want_w else 0, DTYPES[w_dtype],
                  int(power_of_two))
        elif want_w:
            dw.zero_()
        return dx, dw, None, None, None, None


def linear_fp8(x: torch.Tensor, w: torch.Tensor, w_fp8: Optional[Quantized] = None, power_of_two: bool = True) -> torch.Tensor:
    """``x [..., K] @ w[N, K].T`` through 8 bits, in ``x``'s type, with both gradients:

        y = row(x) @ tile(w).T      dx = row(dy) @ tile(w)      dw = col(dy).T @ tile(x)

    where row, col and tile are trips through ``quantize_fp8``.  Between the passes ``x`` and ``w`` are kept in 8 bits.
    ``w_fp8``: ``quantize_fp8(w, "tile")`` where the caller has it (one weight, several micro-batches), or a checkpoint's tiles.

    ``power_of_two``: that of ``gemm_fp8`` for the three products.  False where ``w_fp8`` has scales that are not (large
    products make NaN of them otherwise), or where the rounding of sums matters more than a fifth of the time: the tensor core
    truncates a sum to 32 bits at every 32 products, without it each block of 128 is rounded to nearest."""
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError("x must be [..., K] and w [N, K]")
    _check_float(x, "x")
    _check_float(w, "w")
    if not x.is_cuda or x.device != w.device:
        raise ValueError("x and w must be on one CUDA device")
    if 0 in w.shape:
        raise ValueError("w has no elements")
    if not _native(x, w):
        raise ValueError("x and w must be plain CUDA tensors, and nobody recording")
    data, scale = w_fp8 if w_fp8 is not None else (None, None)
    if data is not None:
        _check_encoded(data, scale, tuple(w.shape), w)
    return _LinearFp8.apply(x, w, data, scale, torch.is_grad_enabled() and w.requires_grad, power_of_two)
