"""Products of 8-bit floats with one scale per block of 128, and activations kept in 8 bits for the backward pass.

The format: e4m3 payloads, one fp32 scale for each block, a power of two where this library quantises: the smallest with
which the block's largest finite magnitude is at most 448.  Blocks are 1 x 128 along a row ("row": activations, gradients),
128 x 128 ("tile": weights) or 128 x 1 along a column ("col": gradients whose rows are summed over).

Four kinds of work:

* ``pack``: an activation goes to 8 bits and comes back (row blocks).
* ``gemm``: the product of two quantised matrices.  ``form`` "fwd": ``a[M, K] @ b[N, K].T``, "dgrad": ``a[M, K] @ b[K, N]``,
  "wgrad": ``a[K, M].T @ b[K, N]``.
* ``linear``: one training step of a linear layer, forward and both gradients.  The forward product reads the input in row
  blocks; what is kept of it for the weight's gradient are its tiles, in 8 bits too.
* ``act``: silu (or silu(gate) * up) whose input is kept in 8 bits, and its gradient from what was kept.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
B = 128


def listed():
    return [
        # the activations of one decode step of a small batch: latency and nothing else
        {"name": "pack_16x4096_bf16", "kind": "pack", "rows": 16, "cols": 4096, "dtype": "bf16"},
        # the hidden states of a training step
        {"name": "pack_8192x4096_bf16", "kind": "pack", "rows": 8192, "cols": 4096, "dtype": "bf16"},
        # a linear layer for one token
        {"name": "gemm_1x4096x4096", "kind": "gemm", "form": "fwd", "m": 1, "n": 4096, "k": 4096, "out": "bf16"},
        # the down projection of a decode step with a batch of 128
        {"name": "gemm_128x4096x1792", "kind": "gemm", "form": "fwd", "m": 128, "n": 4096, "k": 1792, "out": "bf16"},
        # the up projection of a prefill or training step
        {"name": "gemm_8192x1792x4096", "kind": "gemm", "form": "fwd", "m": 8192, "n": 1792, "k": 4096, "out": "bf16"},
        # a padded-free batch into a projection whose sizes fit nothing, back to its input
        {"name": "gemm_dgrad_1001x1111x2050", "kind": "gemm", "form": "dgrad", "m": 1001, "n": 1111, "k": 2050, "out": "fp16"},
        # the gradient of the up projection's weight, summed over the tokens of a step, for a 32-bit master copy
        {"name": "gemm_wgrad_1792x4096x8192", "kind": "gemm", "form": "wgrad", "m": 1792, "n": 4096, "k": 8192, "out": "fp32"},
        # a short ragged sequence through a small layer: forward and backward of many small kernels
        {"name": "linear_333x1000x1792_fp16", "kind": "linear", "tokens": 333, "fin": 1000, "fout": 1792, "dtype": "fp16"},
        # one training step of the up projection
        {"name": "linear_8192x4096x1792_bf16", "kind": "linear", "tokens": 8192, "fin": 4096, "fout": 1792, "dtype": "bf16"},
        # the activation between the projections of one rank of a tensor-parallel MLP, a ragged batch
        {"name": "act_1001x1792_fp16", "kind": "act", "rows": 1001, "cols": 1792, "dtype": "fp16", "gated": False},
        # the same, all tokens of a training step and the whole MLP
        {"name": "act_8192x14336_bf16", "kind": "act", "rows": 8192, "cols": 14336, "dtype": "bf16", "gated": False},
        # the gated form
        {"name": "act_gated_8192x7168_bf16", "kind": "act", "rows": 8192, "cols": 7168, "dtype": "bf16", "gated": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["pack", "gemm", "gemm", "linear", "act"])
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    if kind in ("pack", "act"):
        c = {"kind": kind, "rows": _log(rng, 1, 8192), "cols": _log(rng, 1, 14336), "dtype": dtype}
        if kind == "act":
            c["gated"] = rng.random() < 0.5
        return c
    most = 8192 * 4096 * 1792
    if kind == "linear":
        c = {"kind": kind, "tokens": _log(rng, 1, 8192), "fin": _log(rng, 64, 8192), "fout": _log(rng, 64, 8192), "dtype": dtype}
        while c["tokens"] * c["fin"] * c["fout"] > most:
            c["tokens"] = c["tokens"] // 2 + 1
        return c
    c = {"kind": kind, "form": rng.choice(["fwd", "fwd", "dgrad", "wgrad"]), "m": _log(rng, 1, 8192), "n": _log(rng, 64, 14336),
         "k": _log(rng, 64, 8192), "out": dtype}
    while c["m"] * c["n"] * c["k"] > most:
        c["m"] = c["m"] // 2 + 1
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _blocks(n):
    return -(-n // B)


def _payload(g, rows, cols):
    """e4m3 values as quantisation leaves them (the largest of a block between 224 and 448), rows on 16-byte boundaries."""
    buf = torch.zeros(rows, -(-cols // 16) * 16, device="cuda", dtype=torch.uint8)
    v = (torch.randn(rows, cols, generator=g, device="cuda") * 96.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    buf[:, :cols] = v.view(torch.uint8)
    return buf[:, :cols]


def _scales(g, rows, cols, around):
    """Scales between half and twice ``around``: of any value, as checkpoints bring them."""
    return around * torch.exp2(torch.rand(rows, cols, generator=g, device="cuda") * 2.0 - 1.0)


def _inputs(c, seed):
    g = _gen(seed)
    kind = c["kind"]
    if kind == "pack":
        # hidden states: some channels are much larger than the others
        x = _randn(g, (c["rows"], c["cols"]), torch.float32)
        return ((x * torch.exp(torch.randn(c["cols"], generator=g, device="cuda"))).to(_DT[c["dtype"]]),)
    if kind == "gemm":
        m, n, k, form = c["m"], c["n"], c["k"], c["form"]
        # row-block scales are held with the rows next to one another, as quantisation returns them
        sa = _scales(g, _blocks(k), m, 0.01)
        if form == "wgrad":
            a = _payload(g, k, m)
        else:
            a, sa = _payload(g, m, k), sa.t()
        if form == "fwd":
            return a, sa, _payload(g, n, k), _scales(g, _blocks(n), _blocks(k), 2e-4)
        return a, sa, _payload(g, k, n), _scales(g, _blocks(k), _blocks(n), 2e-4)
    dt = _DT[c["dtype"]]
    if kind == "linear":
        return (_randn(g, (c["tokens"], c["fin"]), dt), _randn(g, (c["fout"], c["fin"]), dt, 0.02),
                _randn(g, (c["tokens"], c["fout"]), dt, 0.01))
    shape = (c["rows"], c["cols"])
    if c["gated"]:
        # one projection makes both: gate and up are the halves of its rows
        both = _randn(g, (c["rows"], 2 * c["cols"]), dt, 1.5)
        return both[:, :c["cols"]], both[:, c["cols"]:], _randn(g, shape, dt, 0.01)
    return _randn(g, shape, dt, 1.5), _randn(g, shape, dt, 0.01)


def prepare(case, seed):
    tensors = _inputs(case, seed)
    if case["kind"] == "linear":
        tensors[0].requires_grad_(True)
        tensors[1].requires_grad_(True)
    return {"case": case, "tensors": tensors}


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(state):
    c, t = state["case"], state["tensors"]
    if own:
        return _own(c, t)
    return _plain(c, t)


def _own(c, t):
    from mintccl_b200.ops import checkpoint8, fp8
    kind = c["kind"]
    if kind == "pack":
        return checkpoint8.save8(t[0]).restore()
    if kind == "gemm":
        a, sa, b, sb = t
        return fp8.gemm_fp8(a, sa, b, sb, ta=c["form"] == "wgrad", tb=c["form"] != "fwd", dtype=_DT[c["out"]])
    if kind == "linear":
        x, w, dy = t
        y = fp8.linear_fp8(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        return y.detach(), dx, dw
    if c["gated"]:
        gate, up, dy = t
        y, saved = checkpoint8.swiglu8_forward(gate, up)
        dgate, dup = checkpoint8.swiglu8_backward(saved, dy)
        return y, dgate, dup
    h, dy = t
    y, saved = checkpoint8.silu8_forward(h)
    return y, checkpoint8.silu8_backward(saved, dy)


def _spread(s, shape, block):
    """The scale of every element."""
    if block in ("tile", "col"):
        s = s.repeat_interleave(B, 0)[:shape[0]]
    if block in ("tile", "row"):
        s = s.repeat_interleave(B, 1)[:, :shape[1]]
    return s


def _dequant(q, s, block):
    return q.view(torch.float8_e4m3fn).float() * _spread(s, q.shape, block)


def _amax(x, block):
    """Largest finite magnitude of every block."""
    r, c = x.shape
    x = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x))
    x = torch.nn.functional.pad(x, (0, -c % B if block != "col" else 0, 0, -r % B if block != "row" else 0))
    if block == "row":
        return x.view(r, -1, B).amax(2)
    if block == "col":
        return x.view(-1, B, c).amax(1)
    return x.view(x.shape[0] // B, B, -1, B).amax((1, 3))


def _quantised(x, block):
    """``x`` after a trip through 8 bits, in fp32."""
    x = x.float()
    m, e = torch.frexp(_amax(x, block))
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    s = torch.where(m > 0, ((e + 127) << 23).view(torch.float32), torch.ones_like(m))       # 2 ** e, exactly
    s = _spread(s, x.shape, block)
    q = torch.where(x.isfinite(), x / s, torch.full_like(x, math.nan)).to(torch.float8_e4m3fn)
    return q.float() * s


def _plain(c, t):
    kind = c["kind"]
    if kind == "pack":
        return _quantised(t[0], "row").to(t[0].dtype)
    if kind == "gemm":
        a, sa, b, sb = t
        a = _dequant(a, sa, "col").t() if c["form"] == "wgrad" else _dequant(a, sa, "row")
        b = _dequant(b, sb, "tile")
        return (a @ (b.t() if c["form"] == "fwd" else b)).to(_DT[c["out"]])
    if kind == "linear":
        with torch.no_grad():
            x, w, dy = t
            xq, wq = _quantised(x, "row"), _quantised(w, "tile")
            dw = _quantised(dy, "col").t() @ _quantised(x, "tile")
            return (xq @ wq.t()).to(x.dtype), (_quantised(dy, "row") @ wq).to(x.dtype), dw.to(w.dtype)
    dt = t[0].dtype
    if c["gated"]:
        g, u, dy = (v.float() for v in t)
        y = g / (1 + torch.exp(-g)) * u
        g, u = _quantised(g, "row"), _quantised(u, "row")
        p = 1 / (1 + torch.exp(-g))
        return y.to(dt), (dy * u * p * (1 + g * (1 - p))).to(dt), (dy * g * p).to(dt)
    h, dy = (v.float() for v in t)
    y = h / (1 + torch.exp(-h))
    h = _quantised(h, "row")
    p = 1 / (1 + torch.exp(-h))
    return y.to(dt), (dy * p * (1 + h * (1 - p))).to(dt)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    c, kind = case, case["kind"]
    if kind == "pack":
        # the activation is read, payload and scales are written and read again, the activation is written
        n, blocks = c["rows"] * c["cols"], c["rows"] * _blocks(c["cols"])
        return {"bytes": 2 * (n * (_SIZE[c["dtype"]] + 1) + 4 * blocks), "flops": 3 * n}
    if kind == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k + n * k + _SIZE[c["out"]] * m * n + 4 * _blocks(k) * (m + _blocks(n)), "flops": 2 * m * n * k}
    if kind == "linear":
        # x and w are read for the forward pass and dy for the backward one, y, dx and dw are written; in between x is kept
        # in 8 bits
        t, i, o = c["tokens"], c["fin"], c["fout"]
        s = _SIZE[c["dtype"]]
        return {"bytes": s * (t * i + o * i + t * o) + 2 * t * i + s * (t * o + t * i + o * i), "flops": 6 * t * i * o}
    # forward: h in, y and the 8-bit copy out; backward: the copy and dy in, dh out
    n, blocks = c["rows"] * c["cols"], c["rows"] * _blocks(c["cols"])
    ins = 2 if c["gated"] else 1
    return {"bytes": n * _SIZE[c["dtype"]] * (2 * ins + 2) + 2 * ins * (n + 4 * blocks), "flops": 20 * ins * n}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def _e4m3_values(bits):
    """The values of e4m3 bit patterns, from the format: sign, 4 bits of exponent (bias 7), 3 of mantissa, no infinities."""
    code = torch.arange(256, dtype=torch.float64)
    mag = code % 128
    ex, man = torch.div(mag, 8, rounding_mode="floor"), mag % 8
    v = torch.where(ex == 0, man * 2.0 ** -9, (1 + man / 8) * torch.pow(torch.tensor(2.0, dtype=torch.float64), ex - 7))
    v = torch.where(mag == 127, torch.full_like(v, math.nan), v)
    v = torch.where(code >= 128, -v, v).to(bits.device)
    return v[bits.view(torch.uint8).long()]


def _two_to(e):
    """2 ** e in 64 bits, exactly: pow() need not be."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _whole_blocks(n):
    return torch.arange(n, device="cuda") // B


def _round8(x, block):
    """``x`` (64 bits) after a trip through 8 bits, by the definition: the smallest power of two s with max |x| <= 448 s over
    the block, then the nearest multiple of the e4m3 step at |x| / s, ties to even."""
    r, c = x.shape
    rb = _whole_blocks(r) if block in ("tile", "col") else torch.arange(r, device="cuda")
    cb = _whole_blocks(c) if block in ("tile", "row") else torch.arange(c, device="cuda")
    nrb, ncb = int(rb[-1]) + 1, int(cb[-1]) + 1
    mag = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    top = torch.zeros(r, ncb, dtype=torch.float64, device="cuda").scatter_reduce_(1, cb.expand(r, c), mag, "amax")
    top = torch.zeros(nrb, ncb, dtype=torch.float64, device="cuda").scatter_reduce_(0, rb[:, None].expand(r, ncb), top, "amax")
    e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, 448.0)) / 448.0))
    e = torch.where(top > 448.0 * _two_to(e), e + 1, e)              # where the logarithm was rounded
    e = torch.where(top <= 448.0 * _two_to(e - 1), e - 1, e)
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=-126)
    s = _two_to(e)[rb][:, cb]
    v = x / s
    step = _two_to((torch.frexp(v)[1] - 1).clamp(min=-6) - 3)
    q = torch.round(v / step) * step
    return torch.where(torch.isfinite(x), q * s, torch.full_like(x, math.nan))


def exact(case, seed):
    c = case
    t = _inputs(c, seed)
    kind = c["kind"]
    if kind == "pack":
        return _round8(t[0].double(), "row")
    if kind == "gemm":
        a, sa, b, sb = t
        m, n, k, form = c["m"], c["n"], c["k"], c["form"]
        kb, nb = _whole_blocks(k), _whole_blocks(n)
        a = _e4m3_values(a) * (sa.double()[kb] if form == "wgrad" else sa.double()[:, kb])
        b = _e4m3_values(b) * (sb.double()[nb][:, kb] if form == "fwd" else sb.double()[kb][:, nb])
        return torch.matmul(a.t() if form == "wgrad" else a, b.t() if form == "fwd" else b)
    if kind == "linear":
        x, w, dy = (v.double() for v in t)
        w = _round8(w, "tile")
        return (torch.matmul(_round8(x, "row"), w.t()), torch.matmul(_round8(dy, "row"), w),
                torch.matmul(_round8(dy, "col").t(), _round8(x, "tile")))
    v = [u.double() for u in t]
    kept = [_round8(u, "row") for u in v[:-1]]
    dy, h, hk = v[-1], v[0], kept[0]
    sig = torch.sigmoid(hk)
    slope = sig + hk * sig * torch.sigmoid(-hk)
    if c["gated"]:
        return h * torch.sigmoid(h) * v[1], dy * kept[1] * slope, dy * hk * sig
    return h * torch.sigmoid(h), dy * slope
