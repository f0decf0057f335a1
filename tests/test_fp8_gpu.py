"""8-bit operands: quantisation, bit for bit against the same float32 operations,
and products against 64-bit ones of the values that the codes stand for.

Tolerances of a product, in terms of S = sum |x| |w| of an output's values.  Sums
of float32 outputs: 128 additions a group and one a group and split, each below
2^-24 of S, and two roundings of every group's scale.  bfloat16 outputs: the 8-bit
matrix cores add products in eights of consecutive k and cut each of them at 2^-13 of
the largest one's power of two.  (One product of 2^16 and another of 2^a at the
place q of a row: the sum is exact for a >= 3 and lacks the second for a <= 2
exactly where q is in the first one's eight.)  The largest loses nothing, so an eight
is off by less than 7 2^-13 of its largest product; its sum joins the other 15 in
float32 (counted as cut, 2 2^-24 each), and the output's rounding is 2^-8 of itself.
"""

import pytest
import torch

import tilec

E32 = 2.0 ** -24
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
WIDE = {"f32": torch.float32, "bf16": torch.bfloat16}


def plain_quantize(x, block, to):
    """On the CPU, in float32, one operation at a time."""
    R, C = x.shape
    padded = torch.nn.functional.pad(x.float().cpu(), (0, -C % 128, 0, -R % block))
    b = padded.view(padded.shape[0] // block, block, -1, 128)
    top = b.abs().amax(dim=(1, 3), keepdim=True)
    top = torch.where(top < float("inf"), top.clamp(min=2.0 ** -100), float("nan"))
    largest = torch.full_like(top, LARGEST[to])
    codes = (b * (largest / top)).to(F8[to]).view(torch.uint8).reshape(padded.shape)[:R, :C]
    return codes, (top / largest)[:, 0, :, 0]


def bits(codes):
    return codes.contiguous().view(torch.uint8).cpu()


def same(q, want):
    codes, scales = bits(q[0]), q[1].cpu()
    nan = torch.isnan(want[1])
    assert torch.equal(scales[~nan], want[1][~nan]) and torch.isnan(scales[nan]).all()
    # A NaN's sign and payload are the conversion's own.
    is_nan = torch.isnan(want[0].view(q[0].dtype).float())
    assert torch.equal(torch.isnan(codes.view(q[0].dtype).float()), is_nan)
    assert torch.equal(codes[~is_nan], want[0][~is_nan])


def normal(R, C, dtype, seed=0, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, C, generator=g)
    if spread:
        x = x * torch.exp2(torch.randn(R, 1, generator=g) * 3) * torch.exp2(torch.randn(1, C, generator=g) * 3)
    return x.to(WIDE[dtype]).cuda()


SHAPES = [(1, 1), (1, 128), (3, 7), (5, 129), (130, 16), (128, 128), (129, 257), (300, 1009), (1, 20000), (4099, 33),
          (257, 2048), (1000, 640)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,to", [("f32", "e4m3"), ("bf16", "e4m3"), ("f32", "e5m2"), ("bf16", "e5m2")])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("R,C", SHAPES)
def test_quantize(R, C, block, dtype, to):
    x = normal(R, C, dtype, seed=R + C)
    q = tilec.ext.quantize_fp8(x, (block, 128), F8[to])
    assert q[0].shape == (R, C) and q[0].dtype == F8[to] and q[1].shape == (-(-R // block), -(-C // 128))
    assert q[0].stride(1) == 1 and (R == 1 or q[0].stride(0) % 16 == 0)
    same(q, plain_quantize(x, block, to))
    # The transpose, read in place.
    same(tilec.ext.quantize_fp8(x.t(), (block, 128), F8[to]), plain_quantize(x.t(), block, to))
    # And back.
    each = q[1].repeat_interleave(block, 0)[:R].repeat_interleave(128, 1)[:, :C]
    for wide in (torch.float32, torch.bfloat16):
        assert torch.equal(tilec.ext.dequantize_fp8(q, wide), (q[0].float() * each).to(wide))


@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_views(block):
    x = normal(300, 700, "bf16")
    for v in (x[:, 5:300], x[3:, 1:2], x.t()[7:400, 3:290], x[::2, ::3], x[:1].expand(40, 700), x.t()[5:6]):
        same(tilec.ext.quantize_fp8(v, (block, 128)), plain_quantize(v, block, "e4m3"))
    # Codes of any stride and alignment go back.
    codes, scales = tilec.ext.quantize_fp8(x[:, :129], (block, 128))
    wide = torch.full((300, 141), 0x7f, dtype=torch.uint8, device="cuda")
    wide[:, 3:132] = codes.view(torch.uint8)
    v = wide.view(torch.float8_e4m3fn)[:, 3:132]
    want = tilec.ext.dequantize_fp8((codes, scales))
    assert torch.equal(tilec.ext.dequantize_fp8((v, scales)), want)
    spaced = torch.empty((scales.shape[0], 2 * scales.shape[1]), device="cuda")[:, ::2]
    spaced.copy_(scales)
    assert torch.equal(tilec.ext.dequantize_fp8([v.t().contiguous().t(), spaced]), want)


@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("transposed", [False, True])
def test_quantize_special_values(block, transposed):
    x = normal(300, 400, "f32")
    x[0] = 0
    x[1] *= 1e-38
    x[2] = 1e-30
    x[3, 7] = float("inf")
    x[150, 200] = float("nan")
    x[299] = torch.finfo(torch.float32).max
    x = x.t() if transposed else x
    for to in F8:
        same(tilec.ext.quantize_fp8(x, (block, 128), F8[to]), plain_quantize(x, block, to))


@pytest.mark.gpu
def test_quantize_past_32_bits():
    R, C = (1 << 19) + 130, 4096  # over 2^31 values
    x = torch.ones((R, C), dtype=torch.bfloat16, device="cuda")
    x[-70:] = normal(70, C, "bf16")
    first = R // 128 * 128 - 128  # where a tile begins
    for block in (1, 128):
        q = tilec.ext.quantize_fp8(x, (block, 128))
        same((q[0][first:], q[1][first // block:]), plain_quantize(x[first:], block, "e4m3"))
        back = tilec.ext.dequantize_fp8(q, torch.bfloat16)
        assert torch.equal(back[first:], tilec.ext.dequantize_fp8((q[0][first:], q[1][first // block:]), torch.bfloat16))
        del q, back
    x = x.view(C, R)  # the transpose [R, C], a column of which is a row of x
    q = tilec.ext.quantize_fp8(x.t()[-200:])
    same(q, plain_quantize(x.t()[-200:], 1, "e4m3"))


# ---------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------

def operand(R, C, to, block, seed, spread=1.0):
    """Codes over the whole range and scales that differ from block to block."""
    g = torch.Generator().manual_seed(seed)
    v = (torch.randn(R, C, generator=g) * LARGEST[to] / 4).clamp(-LARGEST[to], LARGEST[to])
    v = v * torch.exp2(-torch.rand(R, C, generator=g) * 8 * spread)
    scales = torch.exp2(torch.randn(-(-R // block), -(-C // 128), generator=g) * spread) / LARGEST[to]
    room = -(-C // 16) * 16
    codes = torch.full((R, room), 0x7f, dtype=torch.uint8)  # NaNs past the end of a row
    codes[:, :C] = v.to(F8[to]).view(torch.uint8)
    return codes.cuda().view(F8[to])[:, :C], scales.cuda()


def values(q, block):
    R, C = q[0].shape
    return q[0].double() * q[1].double().repeat_interleave(block, 0)[:R].repeat_interleave(128, 1)[:, :C]


def largest_of_eights(xv, wv):
    """sum over eights of k of the largest |x w| (by rows of x, to save memory)."""
    pad = -xv.shape[1] % 8
    xv, wv = (torch.nn.functional.pad(v.abs(), (0, pad)).float() for v in (xv, wv))
    rows = max(1, (1 << 26) // max(1, wv.numel()))
    parts = [(c[:, None] * wv[None]).view(len(c), len(wv), -1, 8).amax(dim=3).double().sum(dim=2) for c in xv.split(rows)]
    return torch.cat(parts)


def check_product(out, x, w, xb, wb):
    M, K = x[0].shape
    xv, wv = values(x, xb), values(w, wb)
    ref, S = torch.mm(xv, wv.t().contiguous()), torch.mm(xv.abs(), wv.t().contiguous().abs())
    G = -(-K // 128)
    if out.dtype == torch.float32:
        tol = (128 + G + 16) * E32 * S + 2 * E32 * ref.abs()
    else:
        tol = 7 * 2.0 ** -13 * 1.0001 * largest_of_eights(xv, wv) + (32 + G + 16) * E32 * S + 2.0 ** -8 * ref.abs()
    err = (out.double() - ref).abs()
    assert out.shape == ref.shape and (err <= tol + 1e-44).all(), (err / (tol + 1e-44)).max()


PRODUCTS = [(1, 1, 1), (1, 16, 128), (1, 4096, 4096), (5, 7, 130), (16, 33, 1000), (17, 64, 4097), (33, 20, 16),
            (64, 200, 129), (65, 130, 257), (100, 300, 64), (129, 257, 1025), (300, 500, 2048), (256, 256, 128),
            (700, 513, 640), (80, 128, 8192), (2000, 2100, 272), (72, 5000, 17),
            (3, 13001, 300), (16, 20000, 1290)]


@pytest.mark.gpu
@pytest.mark.parametrize("xt,wt", [("e4m3", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_products(M, N, K, out, xt, wt):
    for xb, wb in ((1, 128), (1, 1), (128, 128), (128, 1)):
        x, w = operand(M, K, xt, xb, M + K), operand(N, K, wt, wb, N + K + 1)
        got = tilec.ext.linear_fp8(x, w, dtype=WIDE[out])
        assert got.dtype == WIDE[out]
        check_product(got, x, w, xb, wb)
        assert torch.equal(got, tilec.ext.linear_fp8(x, w, dtype=WIDE[out]))  # the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("xt,wt,wb", [("e4m3", "e4m3", 128), ("e5m2", "e4m3", 1)])
@pytest.mark.parametrize("M,N,K", [(512, 4096, 1030), (1000, 3001, 4097), (1030, 2050, 1000), (2900, 5000, 201),
                                   (4000, 4100, 901), (520, 1030, 40003), (2048, 2048, 32768)])
def test_larger_products(M, N, K, xt, wt, wb, out):
    # Every tile, whole and ragged, with and without splits of K.  (An eight's largest
    # product is at most the eight's sum of magnitudes.)
    x, w = operand(M, K, xt, 1, M + K), operand(N, K, wt, wb, N + K + 1)
    got = tilec.ext.linear_fp8(x, w, dtype=WIDE[out])
    xv, wv = values(x, 1), values(w, wb).t().contiguous()
    ref, S = torch.mm(xv, wv), torch.mm(xv.abs_(), wv.abs_())
    G = -(-K // 128)
    err = (got.double() - ref).abs()
    if out == "f32":
        assert (err <= (128 + G + 16) * E32 * S + 2 * E32 * ref.abs()).all()
        assert err.norm() <= 8 * E32 * ref.norm()
    else:
        assert (err <= (7 * 2.0 ** -13 + (32 + G + 16) * E32) * S + 2.0 ** -8 * ref.abs()).all()
        assert err.norm() <= 2.0 ** -8 * ref.norm()
    assert torch.equal(got, tilec.ext.linear_fp8(x, w, dtype=WIDE[out]))


@pytest.mark.gpu
def test_integers_are_exact():
    # Small whole numbers, scales of powers of two: every sum is exact, in either type's reach.
    g = torch.Generator().manual_seed(0)
    for M, N, K in ((3, 40, 700), (40, 100, 1300), (200, 150, 515), (600, 700, 384)):
        x = torch.randint(-2, 3, (M, K), generator=g).float().cuda().to(torch.float8_e4m3fn)
        w = torch.randint(-1, 2, (N, K), generator=g).float().cuda().to(torch.float8_e5m2)
        G = -(-K // 128)
        sx = torch.exp2(torch.randint(0, 2, (M, G), generator=g).float()).cuda()
        sw = torch.exp2(torch.randint(0, 2, (N, G), generator=g).float()).cuda()
        want = (values((x, sx), 1) @ values((w, sw), 1).t()).float()
        assert torch.equal(tilec.ext.linear_fp8((x, sx), (w, sw)), want)
        assert torch.equal(tilec.ext.linear_fp8((x, sx), (w, sw), dtype=torch.bfloat16), want.bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_product_views(M):
    # Rows that begin anywhere, and codes that have to be copied.
    K, N = 300, 200
    x, w = operand(M, K, "e4m3", 1, 1), operand(N, K, "e4m3", 128, 2)
    want = tilec.ext.linear_fp8(x, w)
    for shift, room in ((1, 307), (16, 336), (5, 320), (0, 305)):
        wide = torch.full((max(M, N), room), 0x7f, dtype=torch.uint8, device="cuda")
        wide[:M, shift:shift + K] = x[0].view(torch.uint8)
        xv = wide.view(torch.float8_e4m3fn)[:M, shift:shift + K]
        assert torch.equal(tilec.ext.linear_fp8((xv, x[1]), w), want)
        wide = torch.full((N, room), 0x7f, dtype=torch.uint8, device="cuda")
        wide[:, shift:shift + K] = w[0].view(torch.uint8)
        wv = wide.view(torch.float8_e4m3fn)[:, shift:shift + K]
        assert torch.equal(tilec.ext.linear_fp8(x, (wv, w[1])), want)
        assert torch.equal(tilec.ext.linear_fp8((xv, x[1]), [wv, w[1]]), want)
    columns = x[0].contiguous().t().contiguous().t()
    spaced = torch.empty((M, 2 * x[1].shape[1]), device="cuda")[:, ::2]
    spaced.copy_(x[1])
    assert torch.equal(tilec.ext.linear_fp8((columns, spaced), w), want)
    one = x[0][:1].expand(M, K)  # stride 0
    assert torch.equal(tilec.ext.linear_fp8((one, x[1][:1].expand(M, -1)), w), want[:1].expand(M, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 50, 200])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_special_values_stay_in_their_rows(M, out):
    x, w = operand(M, 500, "e5m2", 1, 1), operand(140, 500, "e4m3", 1, 2)
    want = tilec.ext.linear_fp8(x, w, dtype=out)
    x[0].view(torch.uint8)[1, 499] = 0x7e  # NaN
    w[1][130, 3] = float("nan")
    w[0].view(torch.uint8)[7, 0] = 0x7f
    got = tilec.ext.linear_fp8(x, w, dtype=out)
    rows, cols = [r for r in range(M) if r != 1], [c for c in range(140) if c not in (7, 130)]
    assert got[1].isnan().all() and got[:, 7].isnan().all() and got[:, 130].isnan().all()
    assert torch.equal(got[rows][:, cols], want[rows][:, cols])
    x, w = operand(M, 500, "e5m2", 1, 1), operand(140, 500, "e5m2", 1, 2)
    x[0].view(torch.uint8)[2, 300] = 0x7c  # infinity
    w[0].view(torch.uint8)[:, 300] = 0x3c  # one
    assert (tilec.ext.linear_fp8(x, w, dtype=out)[2] == float("inf")).all()


@pytest.mark.gpu
def test_empty_products():
    for M, N, K in ((0, 5, 300), (5, 0, 300), (5, 6, 0), (0, 0, 0), (200, 300, 0)):
        x = torch.empty((M, K), dtype=torch.float8_e4m3fn, device="cuda")
        w = torch.empty((N, K), dtype=torch.float8_e4m3fn, device="cuda")
        G = -(-K // 128)
        for out in (torch.float32, torch.bfloat16):
            got = tilec.ext.linear_fp8((x, torch.empty((M, G), device="cuda")), (w, torch.empty((-(-N // 128), G), device="cuda")),
                                       dtype=out)
            assert torch.equal(got, torch.zeros((M, N), dtype=out, device="cuda"))
    for shape in ((0, 300), (300, 0), (0, 0)):
        for block in (1, 128):
            q = tilec.ext.quantize_fp8(torch.empty(shape, device="cuda"), (block, 128))
            assert q[0].shape == shape and q[1].shape == (-(-shape[0] // block), -(-shape[1] // 128))
            assert tilec.ext.dequantize_fp8(q).shape == shape


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_product_offsets_past_32_bits(out):
    # Operands of more than 2^31 codes and an output of more than 2^31 values.
    K = 4096
    R = (1 << 19) + 77
    big = torch.zeros((R, K), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.ones((R, K // 128), device="cuda")
    tail = operand(300, K, "e4m3", 1, 4)
    big[-300:], scales[-300:] = tail[0], tail[1]
    small = operand(70, K, "e4m3", 1, 5)
    got = tilec.ext.linear_fp8((big, scales), small, dtype=out)
    check_product(got[-300:], tail, small, 1, 1)
    assert (got[:1000] == 0).all()
    for few in (70, 9):
        q = (small[0][:few], small[1][:few])
        got = tilec.ext.linear_fp8(q, (big, scales), dtype=out)
        check_product(got[:, -300:], q, tail, 1, 1)
    x = operand(R, 32, "e4m3", 1, 6)
    w = operand(4200, 32, "e4m3", 128, 7)
    got = tilec.ext.linear_fp8(x, w, dtype=out)  # 2.2e9 values
    check_product(got[-200:], (x[0][-200:], x[1][-200:]), w, 1, 128)


@pytest.mark.gpu
def test_another_stream():
    x, w = operand(300, 1000, "e4m3", 1, 1), operand(500, 1000, "e4m3", 128, 2)
    wide = normal(300, 1000, "bf16")
    want = (tilec.ext.linear_fp8(x, w), *tilec.ext.quantize_fp8(wide))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = (tilec.ext.linear_fp8(x, w), *tilec.ext.quantize_fp8(wide))
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(bits(got[1]), bits(want[1])) and torch.equal(got[2], want[2])


@pytest.mark.gpu
def test_refusals():
    f = tilec.ext.linear_fp8
    x, w = operand(4, 200, "e4m3", 1, 1), operand(5, 200, "e4m3", 1, 2)
    for a, b, error in ((x[0], w, TypeError), (x, w[0], TypeError), ((x[0],), w, ValueError),
                        ((x[0], x[1], x[1]), w, ValueError), ((x[0][:, :199], x[1]), w, ValueError),
                        ((x[0], x[1][:3]), w, ValueError), ((x[0], x[1][:, :1]), w, ValueError),
                        ((x[0].float(), x[1]), w, TypeError), ((x[0], x[1].double()), w, TypeError),
                        ((x[0].cpu(), x[1]), w, TypeError), ((x[0], x[1].cpu()), w, TypeError),
                        ((x[0][0], x[1]), w, ValueError), ((3, 4), w, TypeError), (None, w, TypeError)):
        with pytest.raises(error):
            f(a, b)
    for dtype in (torch.float16, torch.float8_e4m3fn, "f32"):
        with pytest.raises(TypeError):
            f(x, w, dtype=dtype)
    g = tilec.ext.quantize_fp8
    y = torch.zeros((4, 8), device="cuda")
    for bad, error in (((y[None],), ValueError), ((y[0],), ValueError), ((y.half(),), TypeError),
                       ((y, (2, 128)), ValueError), ((y, (1, 64)), ValueError), ((y, (1, 128), torch.int8), TypeError),
                       ((y, (1,)), ValueError)):
        with pytest.raises(error):
            g(*bad)
    with pytest.raises(TypeError):
        tilec.ext.dequantize_fp8(x, torch.float16)
    with pytest.raises(TypeError):
        tilec.ext.dequantize_fp8(y)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 300)
    q = (x.to(torch.float8_e4m3fn), torch.ones(2, 3))
    for call in (lambda: tilec.ext.quantize_fp8(x), lambda: tilec.ext.dequantize_fp8(q), lambda: tilec.ext.linear_fp8(q, q)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 100])
def test_scales_far_apart(rows):
    # One row's scales, or one tile row's, have no row stride, whatever their view says;
    # several rows' may lie farther apart than the kernels index.
    x, w = (tilec.ext.quantize_fp8(normal(r, 256, "f32", seed=r)) for r in (rows, 40))
    far = (1 << 21) + 7
    store = torch.zeros(rows * far + 2, device="cuda")
    scales = store.as_strided(x[1].shape, (far, 1))
    scales.copy_(x[1])
    want = tilec.ext.linear_fp8(x, w), tilec.ext.dequantize_fp8(x)
    assert torch.equal(tilec.ext.linear_fp8((x[0], scales), w), want[0])
    assert torch.equal(tilec.ext.linear_fp8(w, (x[0], scales)), tilec.ext.linear_fp8(w, x))
    assert torch.equal(tilec.ext.dequantize_fp8((x[0], scales)), want[1])


@pytest.mark.gpu
def test_more_rows_than_small_tiles_have_grids_for():
    M = (1 << 30) + 5  # 2^24 tiles of 64 rows
    codes = torch.zeros(M, 16, dtype=torch.uint8, device="cuda")
    codes[0], codes[1 << 29], codes[M - 1] = 0x38, 0x40, 0x48  # 1, 2 and 4
    one = torch.ones(1, 1, device="cuda")
    x = codes.view(torch.float8_e4m3fn), one.expand(M, 1)
    w = codes[:1].view(torch.float8_e4m3fn), one
    out = tilec.ext.linear_fp8(x, w, dtype=torch.bfloat16)
    assert out[0].item() == 16 and out[1 << 29].item() == 32 and out[M - 1].item() == 64
    assert out.count_nonzero().item() == 3
