"""e4m3 with a scale per block of 128, on the CPU: the encoding against its definition in 64 bits, the activations kept in 8
bits against the formula and against differences, and what the entry points refuse."""
import math

import pytest
import torch

from mintccl_b200.ops import checkpoint8 as c8
from mintccl_b200.ops import fp8

BLOCKS = ["row", "col", "tile"]


def values(shape, dtype, seed=0):
    """Magnitudes over many powers of two, ties of e4m3, zero blocks, and values that are not finite."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float64)
    top = {torch.float32: 120.0, torch.bfloat16: 120.0, torch.float16: 12.0}[dtype]
    x = x * torch.exp2((torch.rand(shape[0], 1, generator=g, dtype=torch.float64) * 2 - 1) * top)
    x = x.to(dtype)
    flat = x.view(-1)
    flat[::7] = 0.0
    flat[3::11] = -0.0
    if flat.numel() > 400:
        flat[50] = float("inf")
        flat[61] = float("-inf")
        flat[72] = float("nan")
        flat[300] = torch.finfo(dtype).max
        flat[301] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return x


def by_definition(x, block):
    """Scales and values in 64 bits: a loop over blocks, the e4m3 values enumerated."""
    codes = torch.arange(127, dtype=torch.float64)
    ex, man = torch.div(codes, 8, rounding_mode="floor"), codes % 8
    mags = torch.where(ex == 0, man / 512, (1 + man / 8) * torch.exp2(ex - 7))          # 0 ... 448, ascending
    x = x.double()
    br, bc = fp8.BLOCKS[block]
    rows, cols = x.shape
    want = torch.full_like(x, math.nan)
    scales = torch.empty(-(-rows // br), -(-cols // bc), dtype=torch.float64)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            b = x[i * br:(i + 1) * br, j * bc:(j + 1) * bc]
            amax = b[b.isfinite()].abs().max().item() if b.isfinite().any() else 0.0
            e = 0
            if amax > 0:
                e = math.frexp(amax)[1] - 9
                e = max(-126, e if amax <= 448.0 * 2.0 ** e else e + 1)
            s = scales[i, j] = 2.0 ** e
            v = (b / s).abs()
            at = torch.searchsorted(mags, v.contiguous()).clamp(max=126)
            lo, hi = (at - 1).clamp(min=0), at
            dl, dh = (v - mags[lo]).abs(), (v - mags[hi]).abs()
            even = torch.where(lo % 2 == 0, lo, hi)
            idx = torch.where(dl < dh, lo, torch.where(dh < dl, hi, even))
            want[i * br:(i + 1) * br, j * bc:(j + 1) * bc] = torch.where(b.isfinite(), torch.sign(b) * mags[idx] * s, math.nan)
    return scales, want


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 129), (128, 1), (129, 257), (260, 40)])
def test_encoding_is_the_definition(shape, block, dtype):
    x = values(shape, dtype)
    data, scale = fp8.quantize_fp8(x, block)
    want_scale, want = by_definition(x, block)
    assert data.shape == x.shape and data.dtype is torch.uint8 and data.stride(0) % 16 == 0
    assert torch.equal(scale.double(), want_scale)
    got = data.view(torch.float8_e4m3fn).double() * fp8._spread(scale, *shape, block).double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    # restored in the tensor's own type: one rounding, and no infinity from a finite value
    back = fp8.dequantize_fp8(data, scale, block, dtype)
    top = torch.finfo(dtype).max
    assert torch.equal(back.nan_to_num(nan=1.0), want.nan_to_num(nan=1.0).clamp(-top, top).to(dtype))


def test_empty_tensors():
    for shape in ((0, 5), (5, 0), (0, 0)):
        for block in BLOCKS:
            data, scale = fp8.quantize_fp8(torch.zeros(shape), block)
            assert tuple(data.shape) == shape and tuple(scale.shape) == fp8._scale_shape(*shape, block)
            assert tuple(fp8.dequantize_fp8(data, scale, block).shape) == shape


@pytest.mark.parametrize("shape", [(), (1,), (300,), (2, 3, 130), (0, 4), (4, 0)])
def test_saved_tensors_come_back(shape):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=g).to(torch.bfloat16)
    s = c8.save8(x)
    y = s.restore()
    assert y.shape == x.shape and y.dtype is x.dtype
    # a rounding to e4m3 is half a step (2 ** -4 relative) of a normal value, 2 ** -10 times the scale below; the scale is
    # at most 2 ** -7 of the largest magnitude
    if x.numel():
        assert bool(((y.double() - x.double()).abs() <= x.double().abs() * 2.0 ** -4 + x.double().abs().max() * 2.0 ** -17).all())
    assert s.nbytes == x.numel() + 4 * s.scale.numel()
    assert s.restore(torch.float32).dtype is torch.float32


@pytest.mark.parametrize("gated", [False, True])
def test_gradient_is_the_formulas_and_that_of_differences(gated):
    g = torch.Generator().manual_seed(2)
    h, u, dy = (torch.randn(4, 200, generator=g) for _ in range(3))
    ins = [t.requires_grad_(True) for t in ((h, u) if gated else (h,))]
    y = c8.swiglu8(*ins) if gated else c8.silu8(*ins)
    hd, ud = h.detach().double(), u.detach().double() if gated else torch.ones(4, 200, dtype=torch.float64)
    # 32 bits: a few roundings
    torch.testing.assert_close(y.detach().double(), hd * torch.sigmoid(hd) * ud, rtol=2.0 ** -20, atol=2.0 ** -24)
    y.backward(dy)
    x = [c8.save8(t.detach()).restore().double().requires_grad_(True) for t in ins]
    f = lambda a, b: a * torch.sigmoid(a) * b                                              # noqa: E731
    ref = torch.autograd.grad(f(x[0], x[1] if gated else torch.ones_like(x[0])), x, dy.double())
    for t, r in zip(ins, ref):
        torch.testing.assert_close(t.grad.double(), r, rtol=2.0 ** -19, atol=2.0 ** -22)
    # central differences in 64 bits at the kept values; the third derivative of silu is below 1: error step ** 2
    step = 1e-4
    b = x[1].detach() if gated else torch.ones(4, 200, dtype=torch.float64)
    a = x[0].detach()
    torch.testing.assert_close(ins[0].grad.double(), dy.double() * (f(a + step, b) - f(a - step, b)) / (2 * step), rtol=1e-5, atol=1e-6)


def test_activation_at_the_ends_of_the_range():
    h = torch.tensor([[-3e38, -200.0, -88.0, -0.0, 0.0, 88.0, 200.0, 3e38]])
    y, saved = c8.silu8_forward(h)
    assert torch.equal(y[0, [1, 3, 4, 6, 7]], torch.tensor([0.0, 0.0, 0.0, 200.0, 3e38]).where(torch.tensor([1, 0, 1, 1, 1]).bool(), torch.tensor(-0.0)))
    d = c8.silu8_backward(saved, torch.ones_like(h))
    assert d.isfinite().all() and d[0, -1] == 1 and d[0, 0] == 0


def test_strided_and_expanded_gradients():
    h = torch.randn(6, 150, requires_grad=True)
    c8.silu8(h).sum().backward()
    assert h.grad.shape == h.shape
    both = torch.randn(2, 3, 260, requires_grad=True)
    y = c8.swiglu8(both[..., :130], both[..., 130:])
    y.transpose(0, 1).contiguous().sum().backward()
    assert both.grad.isfinite().all() and y.shape == (2, 3, 130)


def test_refusals():
    x = torch.randn(4, 8)
    for bad in (lambda: fp8.quantize_fp8(x, "rows"), lambda: fp8.quantize_fp8(x[0]), lambda: fp8.quantize_fp8(x.double()),
                lambda: fp8.quantize_fp8_many(x, ()), lambda: fp8.quantize_fp8_many(x, ("row", "row")),
                lambda: fp8.dequantize_fp8(*fp8.quantize_fp8(x), block="tiles"),
                lambda: fp8.dequantize_fp8(*fp8.quantize_fp8(x), block="col"),
                lambda: fp8.dequantize_fp8(*fp8.quantize_fp8(x), dtype=torch.float64),
                lambda: fp8.dequantize_fp8(x, torch.ones(4, 1)),
                lambda: c8.save8(x.long()), lambda: c8.silu8(x.int()), lambda: c8.swiglu8(x, x[:2]),
                lambda: c8.swiglu8(x, x.half()), lambda: c8.silu8_backward(c8.save8(x), x[:2]),
                lambda: c8.silu8_backward(c8.save8(x), x.half()),
                lambda: fp8.gemm_fp8(*fp8.quantize_fp8(x), *fp8.quantize_fp8(x, "tile")),       # CPU tensors
                lambda: fp8.gemm_fp8(*fp8.quantize_fp8(x), *fp8.quantize_fp8(x, "tile"), ta=True),
                lambda: fp8.linear_fp8(x, x), lambda: fp8.linear_fp8(x, x[:, :4]), lambda: fp8.linear_fp8(x.double(), x.double())):
        with pytest.raises(ValueError):
            bad()


def test_native_checks_come_before_any_launch():
    """The C entry points refuse with an error code what a kernel could not run on; nothing here needs a GPU."""
    from mintccl_b200 import _native as N
    L = N.lib()
    p = 1 << 20
    assert L.mt_fp8_quantize(None, 0, p, 8, 0, 8, 16, p, p, None, None, None, None) < 0            # no rows
    assert L.mt_fp8_quantize(None, 3, p, 8, 4, 8, 16, p, p, None, None, None, None) < 0            # type
    assert L.mt_fp8_quantize(None, 0, p, 8, 4, 8, 24, p, p, None, None, None, None) < 0            # payload pitch
    assert L.mt_fp8_quantize(None, 0, p, 8, 4, 8, 16, p + 8, p, None, None, None, None) < 0        # payload alignment
    assert L.mt_fp8_quantize(None, 0, p, 8, 4, 8, 16, p, None, None, None, None, None) < 0         # no scales
    assert L.mt_fp8_quantize(None, 0, p, 8, 4, 8, 16, None, None, None, None, None, None) < 0      # nothing wanted
    assert L.mt_fp8_dequantize(None, 0, p, 16, p, 1, 1, 4, 8, 1, 64, p, 8) < 0                     # block size
    assert L.mt_fp8_dequantize(None, 0, p, 16, p, 1, 1, 4, 8, 1, 128, p, 7) < 0                    # rows of out overlap
    assert L.mt_fp8_act_forward(None, 0, p, 8, p, 8, 4, 8, p, 8, 16, p, p, None, None) < 0         # a gate without its copy
    assert L.mt_fp8_act_backward(None, 0, 16, p, p, 1, 1, None, None, 0, 0, p, 8, 4, 8, p, p, None) < 0
    ok = (None, p, 16, p, 1, 1, p, 16, p, 1, 1, p, 8, 0, 4, 8, 16, 0, 0, 0)
    for i, v in ((1, None), (2, 8), (7, 0), (12, 7), (13, 5), (14, 0), (16, -1), (17, 1)):
        assert L.mt_gemm_fp8(*ok[:i], v, *ok[i + 1:]) < 0, i
    assert N.last_error()


@pytest.mark.parametrize("between", [0, 1], ids=["backward_at_once", "two_in_flight"])
def test_mlp_of_two_ranks_with_its_activation_input_in_8_bits(between, monkeypatch):
    """The autograd wiring on two ranks (threads; plans and GEMMs as torch expressions): gradients are those of the block with
    the activation's input replaced by its kept copy, passed straight through."""
    import threading

    import test_cpu_tp_mlp as two
    from mintccl_b200.models import tp_mlp

    class Gather(two.FakeGather):
        def __call__(self, x, w):
            return self.call_silu(x, w)[0]

    monkeypatch.setattr(tp_mlp, "gemm_t", lambda a, b, ta=False, tb=False: (a.t() if ta else a) @ (b if tb else b.t()))
    g = torch.Generator().manual_seed(between)
    N, T, H, F = two.N, two.T, two.H, two.F
    ups, downs = torch.randn(N, F, H, generator=g), torch.randn(N, H, F, generator=g)
    xs, dys = torch.randn(2, T, H, generator=g), torch.randn(2, T, H, generator=g)
    used, got, errors, bus, per = [0] if between == 0 else [0, 1], {}, [], two.Bus(), T // N

    def rank(r):
        try:
            m, rows = two.mlp_of(two.Comm(bus, r), ups[r], downs[r]), slice(r * per, (r + 1) * per)
            assert m.checkpoint is None
            m.checkpoint, m.ag_gemm = "fp8", Gather(m.comm)
            shards = [xs[i][rows].clone().requires_grad_(True) for i in used]
            outs = [m(s) for s in shards]
            got[r] = [(y.detach(), *torch.autograd.grad(y, [s, m.w_up, m.w_down], dys[i][rows]))
                      for i, s, y in zip(used, shards, outs)]
        except Exception as e:
            errors.append(e)
            bus.bar.abort()

    threads = [threading.Thread(target=rank, args=(r,)) for r in range(N)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors, errors
    for k, i in enumerate(used):
        x = xs[i].clone().requires_grad_(True)
        u, d = ups.clone().requires_grad_(True), downs.clone().requires_grad_(True)
        h = [x @ u[r].t() for r in range(N)]
        y = sum(torch.nn.functional.silu(h[r]) @ d[r].t() for r in range(N))
        kept = [h[r] + (c8.save8(h[r]).restore() - h[r].detach()) for r in range(N)]
        z = sum(torch.nn.functional.silu(kept[r]) @ d[r].t() for r in range(N))
        dx, du, dd = torch.autograd.grad(z, [x, u, d], dys[i])
        for r in range(N):
            rows = slice(r * per, (r + 1) * per)
            for a, b in zip(got[r][k], (y.detach()[rows], dx[rows], du[r], dd[r])):
                torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)     # fp32 sums of at most 20 terms


@pytest.mark.parametrize("order", [("fp8", None), (None, "fp8")], ids=str)
def test_mlp_whose_checkpoint_is_changed_between_the_passes(order, monkeypatch):
    """The backward pass follows what its own forward pass has kept."""
    import threading

    import test_cpu_tp_mlp as two
    from mintccl_b200.models import tp_mlp

    class Gather(two.FakeGather):
        def __call__(self, x, w):
            return self.call_silu(x, w)[0]

    monkeypatch.setattr(tp_mlp, "gemm_t", lambda a, b, ta=False, tb=False: (a.t() if ta else a) @ (b if tb else b.t()))
    monkeypatch.setattr(tp_mlp, "gemm_dsilu", two.dsilu)
    g = torch.Generator().manual_seed(5)
    N, T, H, F = two.N, two.T, two.H, two.F
    ups, downs = torch.randn(N, F, H, generator=g), torch.randn(N, H, F, generator=g)
    xs, dys = torch.randn(T, H, generator=g), torch.randn(T, H, generator=g)
    got, errors, per = {}, [], T // N

    def rank(r, bus, change):
        try:
            m, rows = two.mlp_of(two.Comm(bus, r), ups[r], downs[r]), slice(r * per, (r + 1) * per)
            m.checkpoint, m.ag_gemm = order[0], Gather(m.comm)
            s = xs[rows].clone().requires_grad_(True)
            y = m(s)
            if change:
                m.checkpoint = order[1]
            got[r, change] = torch.autograd.grad(y, [s, m.w_up, m.w_down], dys[rows])
        except Exception as e:
            errors.append(e)
            bus.bar.abort()

    for change in (False, True):
        bus = two.Bus()
        threads = [threading.Thread(target=rank, args=(r, bus, change)) for r in range(N)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
        assert not errors, errors
    for r in range(N):
        assert all(torch.equal(a, b) for a, b in zip(got[r, True], got[r, False]))


def test_mlp_refuses_unknown_checkpoints():
    from mintccl_b200.models import tp_mlp

    class Comm:
        world_size = 1
    with pytest.raises(ValueError):
        tp_mlp.TensorParallelMLP(Comm(), 128, 256, 256, checkpoint="fp4")


@pytest.mark.parametrize("kind", [torch.uint8, torch.float8_e4m3fn], ids=str)
def test_payloads_are_copied_by_their_bytes(kind):
    """Where a kernel cannot take a payload as it lies, it gets a copy of the bytes, whatever type they have."""
    g = torch.Generator().manual_seed(4)
    wide = torch.randint(0, 256, (7, 96), generator=g, dtype=torch.uint8)
    for t, apart in ((wide[:, :30], 32), (wide[:, 3:33], 0), (wide[:, :60:2], 0), (wide[:1, 1:31], 0), (wide[:, 64:94], 32),
                     (wide.t()[:30], 0)):
        got, pitch = fp8._payload(t.view(kind) if t.is_contiguous() else wide.view(kind).as_strided(t.shape, t.stride(), t.storage_offset()),
                                  "payload", vectors=True, apart=apart)
        assert pitch == 32 if t.shape[1] == 30 else pitch % 16 == 0
        assert torch.equal(got.view(torch.uint8), t)
    kept = wide[:, :32].view(kind)
    assert fp8._payload(kept, "payload", vectors=True)[0] is kept
    again, pitch = fp8._payload(kept, "payload", vectors=True, apart=32)
    assert pitch == 32 and torch.equal(again.view(torch.uint8), wide[:, :32])


def test_a_wait_that_ran_out_is_reported(monkeypatch):
    import types
    for rc, raises in ((0, False), (1, True), (-1, True)):
        monkeypatch.setattr(fp8.N, "lib", lambda: types.SimpleNamespace(mt_gemm_fp8_error=lambda: rc, mt_last_error=lambda: b"why"))
        if raises:
            with pytest.raises(RuntimeError, match="ran out" if rc > 0 else "why"):
                fp8.check()
        else:
            fp8.check()


@pytest.mark.parametrize("block", BLOCKS)
def test_encoding_under_vmap(block):
    """Batched by torch: the bytes and values of the matrices one by one."""
    xs = torch.stack([values((3, 260), torch.float32, seed=i) for i in range(4)]).view(2, 2, 3, 260)
    enc = lambda t: fp8.quantize_fp8(t, block)                                          # noqa: E731
    dec = lambda d, s: fp8.dequantize_fp8(d, s, block, torch.bfloat16)                  # noqa: E731
    data, scale = torch.vmap(torch.vmap(enc))(xs)
    back = torch.vmap(torch.vmap(dec))(data, scale)
    for i in range(2):
        for j in range(2):
            d, s = enc(xs[i, j])
            assert torch.equal(data[i, j], d) and torch.equal(scale[i, j], s)
            assert torch.equal(back[i, j].nan_to_num(), dec(d, s).nan_to_num())
    data, scale = torch.vmap(enc, in_dims=2)(xs[0].transpose(0, 2))
    for i in range(2):
        assert torch.equal(data[i], enc(xs[0, i].t())[0])


def test_activations_and_their_gradients_under_vmap():
    g = torch.Generator().manual_seed(6)
    gate, up, dy = torch.randn(3, 5, 4, 200, generator=g)

    def both(a, b, d):
        y, saved = c8.swiglu8_forward(a, b)
        one = c8.silu8_forward(a)[1]
        return y, *c8.swiglu8_backward(saved, d), c8.silu8_backward(one, d), c8.save8(a).restore()

    got = torch.vmap(both)(gate, up, dy)
    for i in range(5):
        for a, b in zip(got, both(gate[i], up[i], dy[i])):
            torch.testing.assert_close(a[i], b, rtol=2.0 ** -22, atol=2.0 ** -24)      # fp32 exponentials may differ with the layout


def test_packed_calls_report_what_they_cannot_run():
    import ctypes
    from mintccl_b200 import _native as N
    for op, args in ((99, b"\0" * 64), (-1, b"\0" * 64), (fp8.QUANTIZE, b"\0" * 96), (fp8.GEMM, b"\0" * 160), (fp8.LINEAR_FORWARD, b"\0" * 160),
                     (fp8.LINEAR_BACKWARD, b"\0" * 168), (fp8.GEMM, None)):
        assert N.lib().mt_fp8_packed(None, op, args and ctypes.create_string_buffer(args, len(args)).raw) < 0, op
        assert N.last_error()
