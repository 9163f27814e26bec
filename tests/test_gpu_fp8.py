"""The kernels for e4m3 with a scale per block of 128: the encoding gives the bytes of the torch expressions (which the CPU
tests hold to the definition), products and gradients are held to 64 bits."""
import pytest
import torch

from mintccl_b200 import _native as N
from mintccl_b200.ops import checkpoint8 as c8
from mintccl_b200.ops import fp8
from test_cpu_fp8 import values

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def same_encoding(got, x, block):
    want_data, want_scale = fp8._torch_quantize(x.cpu(), block)
    assert torch.equal(got[1].cpu(), want_scale)
    assert torch.equal(got[0].cpu(), want_data)


# ---- encoding, decoding -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 127), (1, 4096), (3, 129), (31, 256), (32, 128), (33, 1000), (128, 128), (129, 257),
                                   (300, 640), (1000, 16)])
def test_encoding_gives_the_bytes_of_the_torch_path(shape, dtype):
    x = values(shape, dtype, seed=shape[1]).cuda()
    for block in fp8.BLOCKS:
        same_encoding(fp8.quantize_fp8(x, block), x, block)
    for blocks in (("row", "col"), ("row", "tile"), ("tile", "col"), ("col", "row", "tile")):
        for block, got in zip(blocks, fp8.quantize_fp8_many(x, blocks)):
            same_encoding(got, x, block)


@pytest.mark.parametrize("dtype", DTYPES)
def test_encoding_takes_any_layout(dtype):
    base = values((70, 700), dtype).cuda()
    for x in (base[:, 1:600], base[:, 8:520], base[::2, 16:272], base.t(), base[:, ::3], base[:1].expand(40, 700), base[3:4, 5:],
              base[:, 5:6]):
        for block in fp8.BLOCKS:
            same_encoding(fp8.quantize_fp8(x, block), x, block)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", list(fp8.BLOCKS))
@pytest.mark.parametrize("shape", [(1, 1), (1, 300), (33, 1000), (129, 256), (256, 17)])
def test_decoding_gives_the_values_of_the_torch_path(shape, block, dtype):
    x = values(shape, dtype, seed=3)
    data, scale = fp8.quantize_fp8(x, block)
    want = fp8.dequantize_fp8(data, scale, block, dtype)
    for d, s in ((data.cuda(), scale.cuda()),                                             # copies lose the padding
                 fp8.quantize_fp8(x.cuda(), block),
                 (data.cuda().view(torch.float8_e4m3fn), scale.cuda().t().contiguous().t())):
        got = fp8.dequantize_fp8(d, s, block, dtype)
        assert got.is_contiguous() and torch.equal(got.cpu().nan_to_num(nan=1.0), want.nan_to_num(nan=1.0))
        assert torch.equal(got.cpu().isnan(), want.isnan())


def test_a_long_tensor_and_a_long_row():
    g = torch.Generator(device="cuda").manual_seed(0)
    for shape in ((2_300_000_000 // 4096, 4096), (1, 70_000_001)):          # offsets past 31 bits; one row of many blocks
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
        s = c8.save8(x)
        last = (slice(-3, None), slice((shape[1] - 1) // 128 * 128 - 1024, None))        # whole blocks, then what is left
        tail = x[last]
        want = fp8._torch_quantize(tail, "row")
        assert torch.equal(s.data[last], want[0])
        assert torch.equal(s.restore()[last], fp8.dequantize_fp8(*want, "row", torch.bfloat16))
        del x, s, tail


# ---- products ----------------------------------------------------------------------------------------------------------
def operands(form, M, N, K, seed=0, spread=1.0):
    """Payloads and scales on the GPU, and the matrices they stand for in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed + M + 3 * N + 5 * K)

    def one(rows, cols, block):
        data = fp8._new_payload(rows, cols, torch.empty(0, device="cuda"))
        v = (torch.randn(rows, cols, generator=g, device="cuda") * 100).clamp(-448, 448)
        data.copy_(v.to(torch.float8_e4m3fn).view(torch.uint8))
        scale = fp8._new_scale(rows, cols, block, "cuda")
        scale.copy_(torch.exp2((torch.rand(scale.shape, generator=g, device="cuda") * 2 - 1) * spread) * 0.01)
        return data, scale, data.view(torch.float8_e4m3fn).double() * fp8._spread(scale, rows, cols, block).double()

    a = one(K, M, "col") if form == "wgrad" else one(M, K, "row")
    b = one(N, K, "tile") if form == "fwd" else one(K, N, "tile")
    return a[:2], b[:2], a[2].t() if form == "wgrad" else a[2], b[2].t() if form == "fwd" else b[2]


def product(form, a, b, **kw):
    return fp8.gemm_fp8(*a, *b, ta=form == "wgrad", tb=form != "fwd", **kw)


def check_product(got, a64, b64):
    """Roundings to 32 bits: one for each block's scale product and one for each addition of a block, 2 ** -24 each; inside
    a block four steps of 32 products, for which the tensor core keeps at least 24 bits below the largest (32 * 2 ** -27 at
    the 27 bits measured, 4 * 2 ** -23 for the steps' own roundings): together (K / 128 + 16) * 2 ** -23 of the sum of
    magnitudes.  Then one rounding to the output's type, or half of its smallest value."""
    want, mag = a64 @ b64, a64.abs() @ b64.abs()
    info = torch.finfo(got.dtype)
    blocks = -(-a64.shape[1] // 128)
    tol = mag * ((blocks + 16) * 2.0 ** -23) * (1 + info.eps) + want.abs() * info.eps / 2 + info.smallest_normal * info.eps
    bad = ((got.double() - want).abs() > tol).nonzero()
    assert not len(bad), (bad[:4].tolist(), len(bad))


def check_product_pow2(got, a64, b64):
    """With scales that the tensor core applies: four steps of 32 products a block, each of which rounds the sum so far
    (2 ** -23, a truncation) and keeps 27 bits or more below the largest product (32 * 2 ** -27); then the output's rounding."""
    want, mag = a64 @ b64, a64.abs() @ b64.abs()
    info = torch.finfo(got.dtype)
    steps = 4 * -(-a64.shape[1] // 128)
    tol = mag * (steps * 3 * 2.0 ** -23) * (1 + info.eps) + want.abs() * info.eps / 2 + info.smallest_normal * info.eps
    # past the largest value and half a step (fp16: 65520) rounding gives infinity
    over = (want.abs() + tol >= info.max * (1 + info.eps / 4)) & (got.double() == want.sign() * float("inf"))
    bad = (((got.double() - want).abs() > tol) & ~over).nonzero()
    assert not len(bad), (bad[:4].tolist(), len(bad))


SIZES = [(1, 1, 1), (1, 128, 128), (3, 5, 7), (1, 4096, 4096), (17, 300, 129), (64, 1000, 512), (127, 129, 257), (128, 256, 384),
         (130, 1000, 1111), (257, 515, 2050), (300, 127, 16), (2050, 1800, 260), (512, 4096, 1792), (129, 20000, 100)]


@pytest.mark.parametrize("form", ["fwd", "dgrad", "wgrad"])
@pytest.mark.parametrize("size", SIZES)
def test_product_against_64_bits(size, form):
    a, b, a64, b64 = operands(form, *size, spread=4.0)
    for dtype in DTYPES:
        check_product(product(form, a, b, dtype=dtype), a64, b64)
    assert N.lib().mt_gemm_fp8_error() == 0


@pytest.mark.parametrize("form", ["fwd", "dgrad", "wgrad"])
@pytest.mark.parametrize("size", [(64, 100, 300), (2050, 1800, 260), (1500, 2301, 129), (2304, 2048, 1111), (300, 16384, 2050), (5000, 1000, 7), (1030, 4100, 4100), (8200, 520, 2100)])
def test_product_with_scales_that_are_powers_of_two(size, form):
    a, b, *_ = operands(form, *size, spread=6.0)
    for _, s in (a, b):
        s.copy_(torch.exp2(torch.round(torch.log2(s))))
    a64 = a[0].view(torch.float8_e4m3fn).double() * fp8._spread(a[1], *a[0].shape, "col" if form == "wgrad" else "row").double()
    b64 = b[0].view(torch.float8_e4m3fn).double() * fp8._spread(b[1], *b[0].shape, "tile").double()
    a64, b64 = a64.t() if form == "wgrad" else a64, b64.t() if form == "fwd" else b64
    for dtype in DTYPES:
        check_product_pow2(product(form, a, b, dtype=dtype, power_of_two=True), a64, b64)
    first = product(form, a, b, dtype=torch.float32, power_of_two=True)
    for _ in range(3):
        assert torch.equal(product(form, a, b, dtype=torch.float32, power_of_two=True), first)
    assert N.lib().mt_gemm_fp8_error() == 0


@pytest.mark.parametrize("form", ["fwd", "dgrad", "wgrad"])
@pytest.mark.parametrize("size, nctas", [((600, 700, 8200), 16), ((600, 600, 8200), 16), ((1792, 4096, 6200), 0), ((1030, 4996, 9000), 0)])
def test_product_with_a_last_wave_of_few_tiles(size, nctas, form):
    """Long sums and one or a few tiles more than whole waves, the last of them partly behind the matrix."""
    a, b, a64, b64 = operands(form, *size, spread=4.0)
    c, d = (x[0].clone() for x in (a, b))
    sc, sd = (torch.exp2(torch.round(torch.log2(x[1]))) for x in (a, b))
    c64 = c.view(torch.float8_e4m3fn).double() * fp8._spread(sc, *c.shape, "col" if form == "wgrad" else "row").double()
    d64 = d.view(torch.float8_e4m3fn).double() * fp8._spread(sd, *d.shape, "tile").double()
    c64, d64 = c64.t() if form == "wgrad" else c64, d64.t() if form == "fwd" else d64
    for dtype in (torch.float32, torch.bfloat16):
        whole = torch.full((size[0] + 130, size[1] + 8), 7.0, device="cuda", dtype=dtype)
        got = product(form, a, b, out=whole[:size[0], :size[1]], nctas=nctas)
        check_product(got, a64, b64)
        assert bool((whole[size[0]:] == 7).all()) and bool((whole[:, size[1]:] == 7).all())
        assert torch.equal(product(form, a, b, dtype=dtype, nctas=nctas), got)
        check_product_pow2(product(form, (c, sc), (d, sd), dtype=dtype, nctas=nctas, power_of_two=True), c64, d64)
    assert N.lib().mt_gemm_fp8_error() == 0


def test_scales_at_the_ends_of_the_range_and_others_than_promised():
    M, Nn, K = 2304, 2048, 384
    a, b, *_ = operands("fwd", M, Nn, K)
    a[1].fill_(1.0)
    b[1].fill_(1.0)
    plain = product("fwd", a, b, dtype=torch.float32, power_of_two=True)
    assert torch.equal(plain, product("fwd", a, b, dtype=torch.float32)) or bool(((plain - product("fwd", a, b, dtype=torch.float32)).abs()
                                                                                   <= plain.abs() * 2.0 ** -18 + 2.0 ** -4).all())
    a[1][3] = 2.0 ** -126
    a[1][5] = 2.0 ** 100
    b[1][2] = 2.0 ** -20
    got = product("fwd", a, b, dtype=torch.float32, power_of_two=True)
    scale = torch.ones(M, Nn, device="cuda", dtype=torch.float64)
    scale[3] *= 2.0 ** -126
    scale[5] *= 2.0 ** 100
    scale[:, 256:384] *= 2.0 ** -20
    want = plain.double() * scale
    # powers of two change nothing but the exponents, except where sums fall below 2 ** -126 (row 3 times the small tile): they
    # are then multiples of 2 ** -149, and each of the four steps of the three blocks may cut up to one off
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -23 + 12 * 2.0 ** -149).all())
    a[1][7, 1] = 3.0        # not a power of two
    a[1][9, 2] = float("nan")
    got = product("fwd", a, b, dtype=torch.float32, power_of_two=True)
    assert bool(got[7].isnan().all()) and bool(got[9].isnan().all())
    keep = [i for i in range(M) if i not in (7, 9)]
    assert bool(got[keep].isfinite().all())


@pytest.mark.parametrize("form", ["fwd", "dgrad", "wgrad"])
def test_product_takes_any_layout(form):
    M, Nn, K = 200, 333, 500
    a, b, a64, b64 = operands(form, M, Nn, K)
    wide = torch.zeros(M, 512, device="cuda", dtype=torch.float16)
    for out in (wide[:, 8:8 + Nn], wide[:, 3:3 + Nn], wide[:, :Nn]):
        wide.zero_()
        got = product(form, a, b, out=out)
        assert got is out
        check_product(got, a64, b64)
        assert int((wide != 0).sum()) == int((out != 0).sum())            # nothing beside the output is written
    # tight rows (not on 16-byte boundaries), float8 views, transposed storage, scales in another order
    tight = [(d.contiguous().view(torch.float8_e4m3fn), s.t().contiguous().t()) for d, s in (a, b)]
    check_product(product(form, *tight), a64, b64)
    turned = [(d.t().contiguous().t(), s.contiguous()) for d, s in (a, b)]
    check_product(product(form, *turned, nctas=3), a64, b64)
    assert torch.equal(product(form, *tight), product(form, a, b))


def test_rows_behind_the_output_are_left_alone():
    a, b, a64, b64 = operands("fwd", 100, 200, 300)
    buf = torch.full((140, 208), 7.0, device="cuda", dtype=torch.bfloat16)
    check_product(product("fwd", a, b, out=buf[20:120, :200]), a64, b64)
    buf[20:120, :200] = 7.0
    assert bool((buf == 7.0).all())


def test_empty_products():
    z = lambda *s: torch.zeros(s, device="cuda", dtype=torch.uint8)                                  # noqa: E731
    f = lambda *s: torch.zeros(s, device="cuda")                                                     # noqa: E731
    assert fp8.gemm_fp8(z(0, 64), f(0, 1), z(32, 64), f(1, 1)).shape == (0, 32)
    got = fp8.gemm_fp8(z(0, 64), f(0, 64), z(0, 32), f(0, 1), ta=True, tb=True, out=torch.ones(64, 32, device="cuda"))
    assert got.shape == (64, 32) and bool((got == 0).all())


def test_values_that_are_not_finite_stay_in_their_rows():
    a, b, a64, b64 = operands("fwd", 130, 260, 300)
    a[0].view(torch.uint8)[5, 7] = 0x7f
    a[1][9, 1] = float("inf")
    got = product("fwd", a, b)
    assert bool(got[5].isnan().all()) and not bool(got[9].isfinite().any())
    keep = [i for i in range(130) if i not in (5, 9)]
    check_product(got[keep], a64[keep], b64)


def test_product_offsets_past_31_bits():
    M, Nn, K = 70_016, 32_768 + 8, 128
    a, b, a64, b64 = operands("fwd", M, Nn, K)
    got = product("fwd", a, b)
    rows = [0, 1, 65_535, 65_536, M - 1]
    check_product(got[rows], a64[rows], b64)


def test_product_gives_the_same_bits_again():
    a, b, *_ = operands("fwd", 1000, 1111, 2050)
    first = product("fwd", a, b, dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(product("fwd", a, b, dtype=torch.float32), first)


def test_products_on_two_streams_and_in_a_graph():
    a, b, a64, b64 = operands("fwd", 300, 700, 900)
    c, d, c64, d64 = operands("dgrad", 500, 600, 1000)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            outs.append((product("fwd", a, b), a64, b64))
        with torch.cuda.stream(s2):
            outs.append((product("dgrad", c, d), c64, d64))
    torch.cuda.synchronize()
    for o in outs:
        check_product(*o)
    x = torch.randn(100, 384, device="cuda", dtype=torch.bfloat16)
    w = fp8.quantize_fp8(torch.randn(256, 384, device="cuda"), "tile")
    step = lambda t: fp8.gemm_fp8(*fp8.quantize_fp8(t), *w)                                          # noqa: E731
    step(x)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step(x)
        graphs.append((g, y))
    x.copy_(torch.randn_like(x) * 3)
    with torch.cuda.stream(s1):
        s1.wait_stream(torch.cuda.default_stream())
        graphs[0][0].replay()
    with torch.cuda.stream(s2):
        s2.wait_stream(torch.cuda.default_stream())
        graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], step(x)) and torch.equal(graphs[1][1], step(x))


def test_refusals_on_the_gpu():
    x = torch.randn(64, 128, device="cuda")
    a, sa = fp8.quantize_fp8(x)
    b, sb = fp8.quantize_fp8(x, "tile")
    for bad in (lambda: fp8.gemm_fp8(a, sb, b, sb), lambda: fp8.gemm_fp8(a, sa, b, sa), lambda: fp8.gemm_fp8(a, sa.double(), b, sb),
                lambda: fp8.gemm_fp8(a, sa, b[:, :64], sb), lambda: fp8.gemm_fp8(x, sa, b, sb), lambda: fp8.gemm_fp8(a, sa, b, sb, ta=True),
                lambda: fp8.gemm_fp8(a, sa, b, sb, dtype=torch.float64), lambda: fp8.gemm_fp8(a, sa.cpu(), b, sb),
                lambda: fp8.gemm_fp8(a, sa, b, sb, out=torch.empty(64, 65, device="cuda")),
                lambda: fp8.gemm_fp8(a, sa, b, sb, out=torch.empty(64, 64, device="cuda").t()),
                lambda: fp8.gemm_fp8(a, sa, b, sb, out=torch.empty(64, 64)), lambda: fp8.dequantize_fp8(a, sa.cpu()),
                lambda: fp8.linear_fp8(x, x.cpu()), lambda: fp8.linear_fp8(x, x, w_fp8=(b[:32], sb))):
        with pytest.raises(ValueError):
            bad()


# ---- the linear layer ------------------------------------------------------------------------------------------------
def trip(t, block):
    return fp8.dequantize_fp8(*fp8.quantize_fp8(t.detach(), block), block).double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,fin,fout", [((1,), 64, 64), ((2, 65), 300, 130), ((1000,), 512, 1000), ((3, 1, 7), 129, 257)])
def test_linear_layer_and_its_gradients(lead, fin, fout, dtype):
    g = torch.Generator(device="cuda").manual_seed(fin)
    x = torch.randn(*lead, fin, generator=g, device="cuda").to(dtype).requires_grad_(True)
    w = (torch.randn(fout, fin, generator=g, device="cuda") * 0.05).to(dtype).requires_grad_(True)
    dy = torch.randn(*lead, fout, generator=g, device="cuda").to(dtype)
    y = fp8.linear_fp8(x, w)
    assert y.dtype is dtype and y.shape == (*lead, fout)
    y.backward(dy)
    x2, dy2 = x.detach().reshape(-1, fin), dy.reshape(-1, fout)
    check_product(y.detach().reshape(-1, fout), trip(x2, "row"), trip(w, "tile").t())
    check_product(x.grad.reshape(-1, fin), trip(dy2, "row"), trip(w, "tile"))
    check_product(w.grad, trip(dy2, "col").t(), trip(x2, "tile"))
    # with the weight's encoding at hand, and only one of the gradients
    q = fp8.quantize_fp8(w.detach(), "tile")
    (dx,) = torch.autograd.grad(fp8.linear_fp8(x, w.detach(), w_fp8=q), (x,), dy)
    (dw,) = torch.autograd.grad(fp8.linear_fp8(x.detach(), w, w_fp8=q), (w,), dy)
    assert torch.equal(dx, x.grad) and torch.equal(dw, w.grad)


def test_linear_layer_follows_differences():
    """The gradients against those of the layer in 64 bits without any 8-bit trip: two operands off by 2 ** -4 of each
    value at most (2 ** -10 of the block's largest below that) leave the products' errors independent, so the norms agree to
    2 ** -4 * sqrt(2) at the very most; central differences of a bilinear map are the map itself."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(256, 384, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    w = (torch.randn(200, 384, generator=g, device="cuda") * 0.05).requires_grad_(True)
    dy = torch.randn(256, 200, generator=g, device="cuda", dtype=torch.bfloat16)
    fp8.linear_fp8(x, w).backward(dy)
    f = lambda a, b: ((a @ b.t()) * dy.double()).sum()                                               # noqa: E731
    x0, w0 = x.detach().double(), w.detach().double()
    for grad, direction in ((x.grad, 0), (w.grad, 1)):
        v = torch.randn(x0.shape if direction == 0 else w0.shape, generator=g, device="cuda").double()
        v = v + grad.double() / grad.double().norm() * v.norm()             # a direction along which the slope is not small
        h = 0.5
        up, down = (f(x0 + h * v, w0), f(x0 - h * v, w0)) if direction == 0 else (f(x0, w0 + h * v), f(x0, w0 - h * v))
        slope = float((up - down) / (2 * h))
        assert abs(float((grad.double() * v).sum()) - slope) <= 2.0 ** -4 * 2 ** 0.5 * abs(slope)


def test_linear_layer_without_tokens_and_without_gradients():
    w = torch.randn(64, 96, device="cuda", requires_grad=True)
    x = torch.randn(0, 96, device="cuda", requires_grad=True)
    y = fp8.linear_fp8(x, w)
    y.sum().backward()
    assert y.shape == (0, 64) and x.grad.shape == (0, 96) and bool((w.grad == 0).all())
    with torch.no_grad():
        assert not fp8.linear_fp8(torch.randn(5, 96, device="cuda"), w).requires_grad


def test_saved_tensor_hooks_may_change_the_layout():
    x = torch.randn(130, 300, device="cuda", requires_grad=True)
    w = torch.randn(70, 300, device="cuda", requires_grad=True)
    dy = torch.randn(130, 70, device="cuda")
    want = torch.autograd.grad(c8.silu8(fp8.linear_fp8(x, w)), (x, w), dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.t().contiguous().cuda().t()):
        y = c8.silu8(fp8.linear_fp8(x, w))
    for a, b in zip(torch.autograd.grad(y, (x, w), dy), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("unpack", [lambda t: t.cpu(), lambda t: t[:-1] if t.dim() == 1 else t[:, :-1], lambda t: t.float()],
                         ids=["host", "shorter", "type"])
@pytest.mark.parametrize("given", [False, True], ids=["weight", "encoded_weight"])
def test_saved_tensors_that_come_back_wrong_are_refused(given, unpack):
    x = torch.randn(130, 300, device="cuda", requires_grad=True)
    w = torch.randn(70, 300, device="cuda", requires_grad=not given)
    encoded = fp8.quantize_fp8(w, "tile") if given else None      # then it is all that is kept
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = fp8.linear_fp8(x, w, encoded)
    with pytest.raises(ValueError):
        y.sum().backward()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = c8.silu8(x)
    with pytest.raises((ValueError, RuntimeError)):
        y.sum().backward()


def test_training_step_in_a_graph():
    """Forward and backward captured once and replayed on other data give what the eager step gives."""
    g = torch.Generator(device="cuda").manual_seed(5)
    w1 = (torch.randn(256, 384, generator=g, device="cuda") * 0.05).bfloat16().requires_grad_(True)
    w2 = (torch.randn(384, 256, generator=g, device="cuda") * 0.05).bfloat16().requires_grad_(True)
    x = torch.randn(100, 384, generator=g, device="cuda").bfloat16()
    dy = torch.randn(100, 384, generator=g, device="cuda").bfloat16()
    step = lambda: torch.autograd.grad(fp8.linear_fp8(c8.silu8(fp8.linear_fp8(x, w1)), w2), (w1, w2), dy)   # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(torch.randn(100, 384, generator=g, device="cuda") * 2)
    dy.copy_(torch.randn(100, 384, generator=g, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    kept = [t.clone() for t in got]
    for a, b in zip(kept, step()):
        assert torch.equal(a, b)


# ---- activations kept in 8 bits --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (1, 5000), (5, 129), (33, 1001), (2, 17, 256), (300, 1792)])
def test_activation_against_64_bits(shape, gated, dtype):
    g = torch.Generator(device="cuda").manual_seed(shape[-1])
    both = (torch.randn(*shape[:-1], 2 * shape[-1], generator=g, device="cuda") * 4).to(dtype)
    h, u = (both[..., :shape[-1]], both[..., shape[-1]:]) if gated else (both[..., :shape[-1]].contiguous(), None)
    dy = torch.randn(shape, generator=g, device="cuda").to(dtype)
    if gated:
        y, saved = c8.swiglu8_forward(h, u)
        dh, du, again = c8.swiglu8_backward(saved, dy, act=True)
        kept = saved
    else:
        y, saved = c8.silu8_forward(h)
        dh, again = c8.silu8_backward(saved, dy, act=True)
        kept = (saved,)
    for k, t in zip(kept, (h, u)):
        same_encoding((k.data, k.scale), t.reshape(-1, shape[-1]), "row")
    info = torch.finfo(dtype)
    # fp32 tensors: about ten roundings of 2 ** -24; 16-bit ones: exponential and quotient within 1e-5
    rel = 2.0 ** -20 if dtype is torch.float32 else 1e-5

    def close(got, want, mag):
        tol = mag * rel * (1 + info.eps) + want.abs() * info.eps / 2 + info.smallest_normal * info.eps + 1e-37
        assert bool(((got.double() - want).abs() <= tol).all())

    hd, ud = h.double(), u.double() if gated else 1.0
    close(y, hd * torch.sigmoid(hd) * ud, (hd * torch.sigmoid(hd) * ud).abs())
    hk = kept[0].restore(torch.float32).double()
    uk = kept[1].restore(torch.float32).double() if gated else torch.ones_like(hk)
    p = torch.sigmoid(hk)
    d = dy.double() * uk
    close(dh, d * (p + hk * p * (1 - p)), d.abs() * (p + hk.abs() * p))
    close(again, hk * p * uk, (hk * p * uk).abs())
    if gated:
        close(du, dy.double() * hk * p, (dy.double() * hk * p).abs())
    # the autograd forms are the same kernels
    ins = [t.detach().clone().requires_grad_(True) for t in ((h, u) if gated else (h,))]
    z = c8.swiglu8(*ins) if gated else c8.silu8(*ins)
    z.backward(dy)
    assert torch.equal(z.detach(), y) and torch.equal(ins[0].grad, dh)


@pytest.mark.parametrize("dtype", DTYPES)
def test_activation_of_extreme_values(dtype):
    top = torch.finfo(dtype).max
    h = torch.tensor([[-top, -200.0, -88.0, -0.0, 0.0, 88.0, 200.0, top] * 40], dtype=dtype, device="cuda")
    y, saved = c8.silu8_forward(h)
    assert bool(y.isfinite().all()) and float(y[0, -1]) == top
    d = c8.silu8_backward(saved, torch.ones_like(h))
    assert bool(d.isfinite().all())
    h[0, 200] = float("nan")
    h[0, 3] = float("inf")
    y, saved = c8.silu8_forward(h)
    back = saved.restore()
    assert int(y.isnan().sum()) == 1 and int(back.isnan().sum()) == 2 and bool(back[0, 3].isnan())
    assert int(c8.silu8_backward(saved, torch.ones_like(h)).isnan().sum()) == 2


def test_activation_on_another_stream():
    s = torch.cuda.Stream()
    h = torch.randn(500, 700, device="cuda", dtype=torch.bfloat16)
    want = c8.silu8_forward(h)[0]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [c8.silu8_forward(h)[0] for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got)


# ---- the MLP block -----------------------------------------------------------------------------------------------------
def test_mlp_with_its_activation_input_in_8_bits():
    """Against 64 bits from the kept copy.  Roundings to bf16, half a step 2 ** -9 each (and 5 % for what is second order or
    fp32): the activation and the output for w_down's gradient; dy @ w_down, dh and the output for the others."""
    import mintccl_b200
    from mintccl_b200 import Config
    from mintccl_b200.models.tp_mlp import TensorParallelMLP
    from mintccl_b200.parallel.rendezvous import SingleControl
    cfg = Config.from_env(max_channels=2, num_blocks=2, buff_size=1 << 20, heap_bytes=64 << 20, scratch_bytes=1 << 20,
                          wait_timeout_ms=4000)
    comm = mintccl_b200.Communicator(control=SingleControl(), device=0, config=cfg)
    T, H, F = 384, 256, 512
    plain, mlp = TensorParallelMLP(comm, T, H, F), TensorParallelMLP(comm, T, H, F, checkpoint="fp8")
    assert torch.equal(plain.w_up, mlp.w_up)
    g = torch.Generator(device="cuda").manual_seed(2)
    with torch.no_grad():
        mlp.w_up.mul_(3.0)
        plain.w_up.copy_(mlp.w_up)
    x, dy, x2 = (torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16).requires_grad_(True) for _ in range(3))
    dy = dy.detach()
    saved = []

    def pack(t):
        saved.append(t)
        return t

    def unpack(t):      # a hook may hand a tensor back in another layout or off the 16-byte grid
        return t.t().contiguous().t() if t.dtype is torch.uint8 else torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y, other = mlp(x), mlp(x2)      # another pass in between
        operands = [t.data_ptr() for t in (x, x2, mlp.w_up, mlp.w_down)]
        assert sum(t.numel() * t.element_size() for t in saved if t.data_ptr() not in operands) == 2 * T * (F + 4 * (F // 128))
        got = torch.autograd.grad(y, [x, mlp.w_up, mlp.w_down], dy)
    comm.check()
    # the same output but for the last place of the activation (exponential and quotient within 1e-5)
    want = plain(x).detach().double()
    h = plain.ag_gemm(x.detach(), mlp.w_up.detach()).double()
    act = (h * torch.sigmoid(h)).abs()
    tol = (act @ mlp.w_down.detach().double().abs().t()) * 2.0 ** -8 * 1.05 + want.abs() * 2.0 ** -8 + 1e-30
    assert bool(((y.detach().double() - want).abs() <= tol).all())
    hk = c8.save8(h.bfloat16()).restore().double()
    p = torch.sigmoid(hk)
    slope = p * (1 + hk * (1 - p))
    d, up, down, xd = dy.double(), mlp.w_up.detach().double(), mlp.w_down.detach().double(), x.detach().double()
    dh, a, half = (d @ down) * slope, hk * p, 2.0 ** -9 * 1.05
    for t, ref, mag in ((got[2], d.t() @ a, (d.abs().t() @ a.abs()) * half),
                        (got[1], dh.t() @ xd, (dh.abs().t() @ xd.abs()) * 2 * half),
                        (got[0], dh @ up, (dh.abs() @ up.abs()) * 2 * half)):
        # dh's error is relative to dy @ w_down's rounding, not to a sum: the fp32 sums under it add 2 ** -16 of magnitudes
        extra = 2.0 ** -16 * mag.max()
        assert bool(((t.double() - ref).abs() <= mag + ref.abs() * half + extra).all())
    assert other.isfinite().all()
    comm.close()


# ---- calls that the documentation allows ------------------------------------------------------------------------------
def test_layer_takes_vectors_and_strided_operands():
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(96, 160, generator=g, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(7, 320, generator=g, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(fp8.linear_fp8(x[0, :160], w), fp8.linear_fp8(x[:1, :160].contiguous(), w)[0])
    for xs, ws in ((x[:, ::2], w), (x[:, 1:161], w.t().contiguous().t()), (x[::3, 160:], w), (x[:1, :160].expand(5, 160), w[::2])):
        a = [t.detach().requires_grad_(True) for t in (xs, ws)]
        b = [t.detach().contiguous().clone().requires_grad_(True) for t in (xs, ws)]
        ya, yb = fp8.linear_fp8(*a), fp8.linear_fp8(*b)
        dy = torch.randn(ya.shape, generator=g, device="cuda").bfloat16()
        assert torch.equal(ya, yb)
        for p, q in zip(torch.autograd.grad(ya, a, dy), torch.autograd.grad(yb, b, dy)):
            assert torch.equal(p, q)
    # gradients that are expanded or strided
    y = fp8.linear_fp8(x[:, :160].detach().requires_grad_(True), w)
    y.sum().backward()


def test_layer_refuses_what_it_cannot_follow():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    w = torch.randn(32, 64, device="cuda", requires_grad=True)
    y = fp8.linear_fp8(x, w)
    with pytest.raises(Exception):      # batched gradients have no address
        torch.autograd.grad(y, (x, w), torch.ones(3, 4, 32, device="cuda"), is_grads_batched=True)
    (dx,) = torch.autograd.grad(fp8.linear_fp8(x, w), x, torch.ones(4, 32, device="cuda"), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(ValueError):
        make_fx(lambda t: fp8.linear_fp8(t, w.detach()))(x.detach())
    q = fp8.quantize_fp8(x.detach())
    with pytest.raises(ValueError):
        make_fx(lambda t: fp8.gemm_fp8(t, q[1], *fp8.quantize_fp8(w.detach(), "tile")))(q[0])


def test_traced_encoding_replays_on_other_inputs():
    """A recorded graph of the encoding holds the operations: it gives other inputs their own bytes."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, y = torch.randn(2, 130, 300, device="cuda")
    for block in fp8.BLOCKS:
        for a, b in zip(make_fx(lambda t: fp8.quantize_fp8(t, block))(x)(y), fp8.quantize_fp8(y, block)):
            assert torch.equal(a, b)
    h = make_fx(lambda t: c8.silu8_forward(t)[0])(x)(y)
    torch.testing.assert_close(h, torch.nn.functional.silu(y), rtol=2.0 ** -20, atol=2.0 ** -24)


def test_batched_gradients_of_the_activation():
    h = torch.randn(5, 200, device="cuda", requires_grad=True)
    d = torch.randn(3, 5, 200, device="cuda")
    y = c8.silu8(h)
    (got,) = torch.autograd.grad(y, h, d, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        (want,) = torch.autograd.grad(y, h, d[i], retain_graph=True)
        torch.testing.assert_close(got[i], want, rtol=2.0 ** -18, atol=2.0 ** -20)


def test_first_calls_of_a_process_may_be_captured():
    """Nothing is set up outside the capture: a new process whose first use of the kernels is inside a graph."""
    import subprocess
    import sys
    code = """
import torch
from mintccl_b200.ops import checkpoint8 as c8, fp8
x, w = torch.randn(300, 512, device="cuda"), torch.randn(2000, 512, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = c8.silu8_forward(fp8.gemm_fp8(*fp8.quantize_fp8(x), *fp8.quantize_fp8(w, "tile"), dtype=torch.float32))[1].restore()
g.replay()
torch.cuda.synchronize()
z = c8.silu8_forward(fp8.gemm_fp8(*fp8.quantize_fp8(x), *fp8.quantize_fp8(w, "tile"), dtype=torch.float32))[1].restore()
assert torch.equal(y, z)
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120,
                       cwd=str(N.lib_path().parents[2]))
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_layers_on_two_streams_at_once():
    g = torch.Generator(device="cuda").manual_seed(9)
    sets = []
    for t, k, n in ((300, 512, 1000), (37, 1000, 640)):
        x = torch.randn(t, k, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
        w = (torch.randn(n, k, generator=g, device="cuda") * 0.05).bfloat16().requires_grad_(True)
        dy = torch.randn(t, n, generator=g, device="cuda", dtype=torch.bfloat16)
        y = fp8.linear_fp8(x, w)
        sets.append((x, w, dy, (y.detach(), *torch.autograd.grad(y, (x, w), dy))))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for i, (x, w, dy, _) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                y = fp8.linear_fp8(x, w)
                got[i].append((y.detach(), *torch.autograd.grad(y, (x, w), dy)))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, sets[i][3]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape, pitch", [((5, 100), 512), ((130, 16), 256), ((129, 1), 128), ((3, 250), 320), ((40, 129), 144), ((129, 384), 1024)])
def test_encoding_leaves_what_lies_between_payload_rows(shape, pitch, dtype):
    """The C entry with payload rows further apart than their padding to 16 bytes, as in a slice of a wider buffer: nothing
    else is written, behind the last row either."""
    rows, cols = shape
    pad = fp8._up16(cols)
    base = values((rows, cols + 1), dtype, seed=cols).cuda()
    for x in (base[:, :cols], base[:, 1:], base[:, :cols].contiguous()):
        for blocks in (("row",), ("col",), ("tile",), ("row", "col"), ("row", "tile"), ("col", "tile"), ("row", "col", "tile")):
            bufs, ptrs = {}, [0] * 6
            for b in blocks:
                bufs[b] = torch.full((rows + 1, pitch), 0xab, device="cuda", dtype=torch.uint8), fp8._new_scale(rows, cols, b, "cuda")
                at = 2 * ("row", "col", "tile").index(b)
                ptrs[at:at + 2] = (t.data_ptr() for t in bufs[b])
            rc = N.lib().mt_fp8_quantize(N.raw_stream(0), fp8.DTYPES[dtype], x.data_ptr(), x.stride(0), rows, cols, pitch,
                                         *(p or None for p in ptrs))
            assert rc == 0, N.last_error()
            for b, (data, scale) in bufs.items():
                same_encoding((data[:rows, :cols], scale), x, b)
                assert bool((data[:rows, cols:pad] == 0).all())
                assert bool((data[:rows, pad:] == 0xab).all()) and bool((data[rows] == 0xab).all()), (b, blocks)


@pytest.mark.parametrize("kind", [torch.uint8, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("cols", [30, 128, 1000])
def test_activation_gradient_from_payloads_in_another_layout(cols, kind):
    """Kept payloads that come back as float8, and as a slice of a wider tensor: the same gradients."""
    gate, up, dy = torch.randn(3, 40, cols, device="cuda")
    _, saved = c8.swiglu8_forward(gate, up)
    want = c8.swiglu8_backward(saved, dy, act=True)
    alone = c8.silu8_backward(saved[0], dy, act=True)

    def moved(k, left):
        wide = torch.full((40, 2048), 0x55, device="cuda", dtype=torch.uint8)
        wide[:, left:left + cols] = k.data
        return k._replace(data=wide.view(kind)[:, left:left + cols])

    for left in (0, 16, 7):
        other = tuple(moved(k, left) for k in saved)
        for a, b in zip(c8.swiglu8_backward(other, dy, act=True), want):
            assert torch.equal(a, b)
        for a, b in zip(c8.silu8_backward(other[0], dy, act=True), alone):
            assert torch.equal(a, b)
        assert torch.equal(other[0].restore(), saved[0].restore())


@pytest.mark.parametrize("form", ["fwd", "dgrad", "wgrad"])
@pytest.mark.parametrize("size", [(2304, 2048, 4100), (700, 300, 5000), (64, 256, 8192)], ids=["pairs", "single", "shared"])
def test_every_block_takes_its_own_scales(size, form):
    """Neighbouring blocks' scales are powers of two far apart and every call has others in their places: a block that met
    another block's, another row's or the last call's would be off by a factor.  The calls follow one another unwatched."""
    a, b, *_ = operands(form, *size)
    M, Nn, K = size
    sets = []
    for i in range(6):
        at = lambda n, step: torch.arange(n, device="cuda").mul(step).add(5 * i).remainder(23).sub(11)               # noqa: E731
        # [M, blocks of K] and [blocks of N, blocks of K]
        sa = torch.exp2((at(M, 7)[:, None] + at(-(-K // 128), 9)[None]).float())
        sb = torch.exp2((at(-(-Nn // 128), 5)[:, None] - at(-(-K // 128), 4)[None]).float())
        sets.append((a[1].new_empty(a[1].shape).copy_(sa.t() if form == "wgrad" else sa), sb if form == "fwd" else sb.t()))
    torch.cuda.synchronize()
    outs = [[product(form, (a[0], sa), (b[0], sb), dtype=torch.float32, power_of_two=pow2) for sa, sb in sets for _ in range(4)]
            for pow2 in (False, True)]
    for i, (sa, sb) in enumerate(sets):
        a64 = a[0].view(torch.float8_e4m3fn).double() * fp8._spread(sa, *a[0].shape, "col" if form == "wgrad" else "row").double()
        b64 = b[0].view(torch.float8_e4m3fn).double() * fp8._spread(sb, *b[0].shape, "tile").double()
        a64, b64 = a64.t() if form == "wgrad" else a64, b64.t() if form == "fwd" else b64
        for got, check in zip(outs, (check_product, check_product_pow2)):
            check(got[4 * i], a64, b64)
            assert all(torch.equal(got[4 * i + j], got[4 * i]) for j in range(1, 4))
    assert N.lib().mt_gemm_fp8_error() == 0


def test_a_wait_that_runs_out_is_reported_once():
    """A wait that nothing ends (1 ms), on a stream that the default one does not wait for."""
    fp8.check()
    s = torch.cuda.Stream()
    assert N.lib().mt_test_gemm_fp8_expire(s.cuda_stream) == 0
    with pytest.raises(RuntimeError, match="ran out"):
        fp8.check("cuda:0")
    fp8.check(0)
    a, b, a64, b64 = operands("fwd", 300, 200, 400)
    check_product(product("fwd", a, b), a64, b64)
    fp8.check()


def test_layer_with_a_weight_whose_scales_have_any_value():
    """A checkpoint's tiles, at a size where the products run on pairs (and would make NaN of them): any value has to be said."""
    T, K, Nn = 2304, 1200, 2050
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(T, K, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    dy = torch.randn(T, Nn, generator=g, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(Nn, K, generator=g, device="cuda").requires_grad_(True)
    data, scale = fp8.quantize_fp8(w, "tile")
    scale = scale * (torch.rand(scale.shape, generator=g, device="cuda") + 0.5)
    w64 = data.view(torch.float8_e4m3fn).double() * fp8._spread(scale, Nn, K, "tile").double()
    y = fp8.linear_fp8(x, w, (data, scale), power_of_two=False)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    check_product(y.detach(), trip(x, "row"), w64.t())
    check_product(dx, trip(dy, "row"), w64)
    check_product(dw, trip(dy, "col").t(), trip(x, "tile"))
    fp8.check()


def test_encoding_under_vmap_takes_the_torch_path():
    x = torch.randn(3, 40, 300, device="cuda")
    for block in fp8.BLOCKS:
        data, scale = torch.vmap(lambda t: fp8.quantize_fp8(t, block))(x)
        back = torch.vmap(lambda d, s: fp8.dequantize_fp8(d, s, block))(data, scale)
        for i in range(3):
            same_encoding((data[i], scale[i]), x[i], block)
            assert torch.equal(back[i], fp8.dequantize_fp8(data[i], scale[i], block))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("given", [False, True], ids=["weight", "encoded_weight"])
def test_large_layer_and_its_gradients(given, dtype):
    """All three products on pairs, with scales that the tensor core applies; ragged sizes, rows of a wider tensor."""
    T, K, Nn = 2050, 2300, 1930
    g = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(T, K + 4, generator=g, device="cuda").to(dtype)[:, 4:].requires_grad_(True)
    w = (torch.randn(Nn, K, generator=g, device="cuda") * 0.05 * torch.exp(torch.randn(K, generator=g, device="cuda"))).to(dtype).requires_grad_(True)
    dy = torch.randn(T, Nn, generator=g, device="cuda").to(dtype)
    y = fp8.linear_fp8(x, w, fp8.quantize_fp8(w, "tile") if given else None)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    check_product_pow2(y.detach(), trip(x, "row"), trip(w, "tile").t())
    check_product_pow2(dx, trip(dy, "row"), trip(w, "tile"))
    check_product_pow2(dw, trip(dy, "col").t(), trip(x, "tile"))
    fp8.check()


@pytest.mark.parametrize("shape", [(33, 300, 130), (2050, 1500, 1600)], ids=["small", "pairs"])
def test_layer_takes_gradients_of_any_layout(shape):
    """Expanded along either dimension or both, turned, and every other one of a wider tensor: as contiguous ones."""
    T, K, Nn = shape
    g = torch.Generator(device="cuda").manual_seed(13)
    x = torch.randn(T, K, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    w = torch.randn(Nn, K, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    y = fp8.linear_fp8(x, w)
    wide = torch.randn(T + Nn, 2 * (T + Nn), generator=g, device="cuda", dtype=torch.bfloat16)
    for dy in (wide[:1, :1].expand(T, Nn), wide[:1, :Nn].expand(T, Nn), wide[:T, :1].expand(T, Nn), wide[:Nn, :T].t(),
               wide[:T, :2 * Nn:2], wide[1:T + 1, 3:Nn + 3]):
        got = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
        want = torch.autograd.grad(y, (x, w), dy.contiguous().clone(), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    want = torch.autograd.grad(y, (x, w), torch.ones_like(y), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="plain CUDA tensor"):
        torch.autograd.grad(y, (x, w), torch.ones(3, T, Nn, device="cuda", dtype=torch.bfloat16), is_grads_batched=True)
    fp8.check()
