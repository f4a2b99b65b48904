"""trspmm.quant_mx4, dequant_mx4, rms_norm_mx4 and matmul_mx4 against their definitions in 64 bits.

Quantisation is exact: a power of two divides without rounding, so codes and scales have to be those of the definition.
Products are compared in two ways.  With scales of 0.5, 1 and 2 every product is a multiple of 1/16 of at most 144, and sums of up to
4096 of them stay below 2^24 sixteenths: every partial sum is a 32-bit float, in any order, and the result has to be the exact one,
rounded once to its type.  With scales over a wide range, k additions in any order, each rounding (to nearest or towards zero) by
at most 2^-23 of a partial sum, are off by at most k 2^-23 of the sum of the products' sizes."""
import pytest
import torch

import trspmm
from trspmm import _native as nat

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ROUND = {t: torch.finfo(t).eps / 2 for t in TYPES}
E8M0 = torch.float8_e8m0fnu
EPS = 1e-5
SIZES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(dtype)


def blocks_of(width):
    return (width + 31) // 32


def power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def values(codes, scale):
    """float64 [rows, 32 * blocks]."""
    table = torch.tensor(SIZES + [-s for s in SIZES], dtype=torch.float64, device="cuda")
    q = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), 2).view(codes.shape[0], -1, 32)
    byte = scale.view(torch.uint8).int()
    unit = torch.where(byte == 255, float("nan"), power(byte - 127))
    return (q * unit[:, :, None]).view(codes.shape[0], -1)


def definition(x):
    """(codes, scale bytes) of x [rows, width] by distances."""
    rows, width = x.shape
    full = torch.zeros((rows, blocks_of(width) * 32), dtype=torch.float64, device="cuda")
    full[:, :width] = x.double()
    b = full.view(rows, -1, 32)
    whole = torch.isfinite(b).all(2)
    b = torch.where(whole[:, :, None], b, 0.0)
    peak = b.abs().amax(2)
    e = torch.where(peak > 0, torch.frexp(peak).exponent - 1, -1000)
    e = (e - 2).clamp(min=-126)
    t = b / power(e)[:, :, None]
    off = (t.abs()[..., None] - torch.tensor(SIZES, dtype=torch.float64, device="cuda")).abs()
    # ties go to the even code: it wins by a hair (distances are multiples of 2^-130 apart otherwise, far above it)
    even = torch.tensor([0.0, 1.0] * 4, dtype=torch.float64, device="cuda")
    least = off.amin(3, keepdim=True)
    code = torch.where(off == least, even, 2.0).argmin(3)
    code = torch.where(torch.signbit(t) & whole[:, :, None], code + 8, code)
    code = code.view(rows, -1, 2)
    byte = torch.where(whole, e + 127, 255)
    return (code[:, :, 0] | code[:, :, 1] << 4).to(torch.uint8), byte.to(torch.uint8)


def hard_rows(rows, width, dtype, seed):
    """Values on and next to the borders between codes, at many sizes, signed zeros, blocks of zeros and of tiny values."""
    g = gen(seed)
    top = torch.randint(-12, 12, (rows, blocks_of(width)), generator=g, device="cuda")
    top = top.repeat_interleave(32, 1)[:, :width]
    grid = torch.randint(-34, 35, (rows, width), generator=g, device="cuda").double() / 4
    near = torch.randint(-1, 2, (rows, width), generator=g, device="cuda").double() * torch.finfo(dtype).eps
    x = grid * (1 + near) * torch.pow(2.0, top.double())
    kind = torch.randint(0, 8, (rows, blocks_of(width)), generator=g, device="cuda").repeat_interleave(32, 1)[:, :width]
    x = torch.where(kind == 0, torch.zeros_like(x), x)
    x = torch.where(kind == 1, -x * 0.0, x)
    x = torch.where(kind == 2, torch.randn((rows, width), generator=g, device="cuda").double() * 3, x)
    x = torch.where(kind == 3, x * 2.0 ** (-20 if dtype == torch.float16 else -125), x)
    return x.to(dtype)


WIDTHS = [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 100, 128, 255, 256, 257, 511, 1000, 2047, 2048, 2049, 4096, 5000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_quant_is_the_definition(width, dtype):
    say("quant", width, dtype)
    for rows in (1, 5, 67):
        x = hard_rows(rows, width, dtype, width)
        codes, scale = trspmm.quant_mx4(x)
        assert codes.dtype is torch.uint8 and scale.dtype is E8M0
        assert codes.shape == (rows, 16 * blocks_of(width)) and scale.shape == (rows, blocks_of(width))
        want, byte = definition(x)
        assert torch.equal(scale.view(torch.uint8), byte)
        assert torch.equal(codes, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out", TYPES)
def test_values(dtype, out):
    say("values", dtype, out)
    for rows, width in [(1, 1), (9, 31), (70, 300), (3, 4100)]:
        x = hard_rows(rows, width, dtype, 3)
        codes, scale = trspmm.quant_mx4(x)
        got = trspmm.dequant_mx4(codes, scale, width, dtype=out)
        assert got.dtype is out and torch.equal(got.double(), values(codes, scale)[:, :width].to(out).double())


def test_every_scale_and_code():
    say("all scales")
    scale = torch.arange(256, dtype=torch.uint8, device="cuda").view(E8M0).repeat(1, 1)
    codes = torch.randint(0, 256, (1, 256 * 16), generator=gen(1), device="cuda", dtype=torch.uint8)
    want = values(codes, scale)
    for out in TYPES:
        got = trspmm.dequant_mx4(codes, scale, 256 * 32, dtype=out)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = ~torch.isnan(want)
        assert torch.equal(got[fine], want[fine].to(out))


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_that_are_not_finite(dtype):
    say("not finite", dtype)
    x = rand((6, 160), dtype, 1)
    x[0, 5], x[1, 40], x[2, 159], x[3, 64] = float("nan"), float("inf"), -float("inf"), float("nan")
    codes, scale = trspmm.quant_mx4(x)
    want, byte = definition(x)
    assert torch.equal(codes, want) and torch.equal(scale.view(torch.uint8), byte) and int((byte == 255).sum()) == 4
    got = trspmm.dequant_mx4(codes, scale, 160, dtype=dtype)
    bad = torch.isnan(got).view(6, 5, 32)
    assert bool((bad.all(2) == bad.any(2)).all()) and torch.equal(bad.any(2), byte == 255)


def test_largest_and_smallest_values():
    say("extremes")
    big = torch.finfo(torch.float32).max
    x = torch.zeros((4, 64), device="cuda")
    x[0, 0], x[0, 1], x[0, 32], x[1, 3], x[1, 40] = big, -big / 3, 2.0 ** -149, 2.0 ** -126, 2.0 ** -124
    x[2] = 2.0 ** -125 * torch.arange(64, device="cuda") / 64
    codes, scale = trspmm.quant_mx4(x)
    want, byte = definition(x)
    assert torch.equal(codes, want) and torch.equal(scale.view(torch.uint8), byte)
    assert torch.equal(trspmm.dequant_mx4(codes, scale, 64, dtype=torch.float32).double(), values(codes, scale))


def guarded(rows, width, ld, dtype, fill):
    """A matrix of row stride ld in a buffer filled with `fill`, 4 spare rows on each side."""
    buf = torch.full(((rows + 8) * ld,), fill, dtype=torch.uint8 if dtype is E8M0 else dtype, device="cuda")
    view = buf[4 * ld:].as_strided((rows, width), (ld, 1))
    return buf, view.view(E8M0) if dtype is E8M0 else view


def untouched(buf, rows, width, ld, fill):
    rest = buf.clone()
    rest[4 * ld:].as_strided((rows, width), (ld, 1)).fill_(fill)
    return bool((rest == fill).all())


@pytest.mark.parametrize("rows,width", [(1, 33), (37, 95), (6, 2100)])
def test_strides_and_given_outputs(rows, width):
    say("strides", rows, width)
    b = blocks_of(width)
    x = rand((rows, width + 5), torch.float16, 1)[:, 3:width + 3]      # off every boundary
    cbuf, codes = guarded(rows, 16 * b, 16 * b + 32, torch.uint8, 7)
    sbuf, scale = guarded(rows, b, b + 3, E8M0, 7)
    got = trspmm.quant_mx4(x, out=codes, scale=scale)
    assert got[0].data_ptr() == codes.data_ptr() and got[1].data_ptr() == scale.data_ptr()
    want, byte = definition(x)
    assert torch.equal(codes, want) and torch.equal(scale.view(torch.uint8), byte)
    assert untouched(cbuf, rows, 16 * b, 16 * b + 32, 7) and untouched(sbuf, rows, b, b + 3, 7)
    obuf, out = guarded(rows, width, width + 1, torch.float32, 7.0)
    trspmm.dequant_mx4(codes, scale, width, out=out)
    assert torch.equal(out.double(), values(want, byte)[:, :width]) and untouched(obuf, rows, width, width + 1, 7.0)
    # columns that do not follow one another, codes off their boundary: copied
    t = rand((width, rows), torch.float32, 2).t()
    assert torch.equal(trspmm.quant_mx4(t)[0], definition(t)[0])
    odd = torch.zeros(rows * 16 * b + 1, dtype=torch.uint8, device="cuda")[1:].view(rows, 16 * b)
    odd.copy_(codes)
    assert torch.equal(trspmm.dequant_mx4(odd, scale.view(torch.uint8), width, dtype=torch.float32), out)


def test_nothing_to_do():
    say("empty")
    for rows, width in [(0, 64), (4, 0), (0, 0)]:
        codes, scale = trspmm.quant_mx4(torch.empty((rows, width), device="cuda"))
        assert codes.shape == (rows, 16 * blocks_of(width)) and scale.shape == (rows, blocks_of(width))
        assert trspmm.dequant_mx4(codes, scale, width).shape == (rows, width)
        w = torch.ones(width, device="cuda")
        assert trspmm.rms_norm_mx4(torch.empty((rows, width), device="cuda"), w)[0].shape == codes.shape
    empty = torch.empty((5, 0), dtype=torch.uint8, device="cuda")
    bias = rand((3,), torch.float32, 1)
    got = trspmm.matmul_mx4(empty, empty, empty[:3], empty[:3], bias=bias, dtype=torch.float32)   # no k: the bias
    assert torch.equal(got, bias.expand(5, 3))
    codes, scale = trspmm.quant_mx4(rand((4, 64), torch.float32, 1))
    assert trspmm.matmul_mx4(codes[:0], scale[:0], codes, scale).shape == (0, 4)
    assert trspmm.matmul_mx4(codes, scale, codes[:0], scale[:0]).shape == (4, 0)


# ------------------------------------------------------------------------------------------------
# The norm.  Its y is off by `far` of itself (the bound of tests/test_gpu_norm.py), so a code may be the neighbour where y lies
# that close to a border, and a scale that of the next power of two where the largest |y| does.

def far(width):
    return (60 + width / 1024) * 2.0 ** -24


def check_norm(x, w, res, codes, scale, r, eps=EPS):
    width = x.shape[1]
    h = x.double() + (0 if res is None else res.double())
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()
    pad = torch.zeros((x.shape[0], blocks_of(width) * 32), dtype=torch.float64, device="cuda")
    pad[:, :width] = y
    size, peak = far(width) + 2.0 ** -22, pad.view(x.shape[0], -1, 32).abs().amax(2)
    byte = scale.view(torch.uint8).int()

    def of(v):
        return (torch.where(v > 0, torch.frexp(v).exponent - 1, -1000) - 2).clamp(min=-126) + 127
    assert bool(((byte == of(peak * (1 - size))) | (byte == of(peak * (1 + size)))).all())
    got = values(codes, scale)
    unit = power(byte - 127).repeat_interleave(32, 1)
    best = (pad.abs()[..., None] - torch.tensor(SIZES, dtype=torch.float64, device="cuda") * unit[..., None]).abs().amin(2)
    assert bool(((got - pad).abs() <= best + 2 * size * pad.abs()).all())
    assert bool((got[:, width:] == 0).all())
    if res is None:
        assert r is None
    else:
        assert bool(((r.double() - h).abs() <= h.abs() * (2.0 ** -24 + ROUND[r.dtype] * 1.01) + 2.0 ** -25).all())


MIXES = [(x, r) for x in TYPES for r in [None, *TYPES] if r is None or r is x or torch.float32 in (x, r)]


@pytest.mark.parametrize("x_type,r_type", MIXES)
@pytest.mark.parametrize("w_type", TYPES)
def test_norm_types(x_type, r_type, w_type):
    say("norm types", x_type, r_type, w_type)
    for rows, width in [(37, 96), (9, 1000), (5, 1800), (6, 2300), (5, 4500)]:
        x, w = rand((rows, width), x_type, 1), (1 + 0.2 * rand((width,), torch.float32, 2)).to(w_type)
        res = None if r_type is None else rand((rows, width), r_type, 3, 2.0)
        check_norm(x, w, res, *trspmm.rms_norm_mx4(x, w, res, EPS))


@pytest.mark.parametrize("width", [*WIDTHS, 127, 512, 513, 1023, 1024, 1025, 1374, 1536, 1537, 2100, 2560, 2561, 2900, 3060, 3100, 4097, 6144, 6145, 8191, 8192, 8193, 12_001, 20_000])
def test_norm_widths(width):
    say("norm width", width)
    for rows in (1, 33, 1025):
        if rows * width > 3_000_000:
            continue
        x, w, res = rand((rows, width), torch.float16, 1), 1 + 0.2 * rand((width,), torch.float32, 2), rand((rows, width), torch.float16, 3)
        check_norm(x, w, res, *trspmm.rms_norm_mx4(x, w, res, EPS))
        check_norm(x, w, None, *trspmm.rms_norm_mx4(x, w, eps=EPS))
        # the residual's sum in the residual's place
        r = res.clone()
        codes, scale, got = trspmm.rms_norm_mx4(x, w, r, EPS, r_out=r)
        assert got.data_ptr() == r.data_ptr()
        check_norm(x, w, res, codes, scale, r)


@pytest.mark.parametrize("width", [40, 300, 1400, 2000, 2400, 5000, 7000, 9000])
def test_norm_of_large_values_and_of_none(width):
    say("norm extremes", width)
    w = torch.ones(width, device="cuda")
    for std in (1e30, 1e-30, 0.0):
        x = rand((5, width), torch.float32, 1, std)
        check_norm(x, w, None, *trspmm.rms_norm_mx4(x, w, eps=EPS))
    x = rand((5, width), torch.float32, 1)
    x[1, width - 1], x[3, 0] = float("nan"), float("inf")
    codes, scale, _ = trspmm.rms_norm_mx4(x, w, eps=EPS)
    byte = scale.view(torch.uint8)
    assert bool((byte[1] == 255).all()) and int(byte[3, 0]) == 255 and bool((byte[3, 1:] != 255).all())
    assert bool((codes[3] & 0x77 == 0).all()) and bool((codes[1] == 0).all())      # finite / infinity: zeros with their signs
    for row in (0, 2, 4):
        check_norm(x[row:row + 1], w, None, codes[row:row + 1], scale[row:row + 1], None)


# ------------------------------------------------------------------------------------------------
# The product.

def operand(rows, k, seed, low=126, high=129):
    """Codes and scales (bytes low .. high - 1) of rows of k numbers; what pads the last block is zeros."""
    b = blocks_of(k)
    codes = torch.randint(0, 256, (rows, 16 * b), generator=gen(seed), device="cuda", dtype=torch.uint8)
    half = torch.stack((codes & 15, codes >> 4), 2).view(rows, -1)
    half[:, k:] = 0
    half = half.view(rows, -1, 2)
    scale = torch.randint(low, high, (rows, b), generator=gen(seed + 1), device="cuda", dtype=torch.uint8)
    return half[:, :, 0] | half[:, :, 1] << 4, scale.view(E8M0)


def product(a, sa, w, sw, bias=None):
    out = torch.mm(values(a, sa), values(w, sw).t().contiguous())
    return out if bias is None else out + bias.double()


SHAPES = [(1, 1, 1), (1, 1, 32), (1, 16, 33), (2, 17, 64), (1, 4096, 4096), (3, 1000, 545), (16, 16, 512), (17, 33, 511),
          (5, 300, 1000), (31, 64, 513), (32, 2048, 1024), (33, 65, 2010), (64, 64, 64), (64, 100, 4096), (65, 129, 96),
          (100, 100, 100), (127, 255, 257), (128, 128, 256), (129, 257, 288), (200, 1000, 2016), (256, 256, 1056), (257, 300, 3000),
          (500, 1000, 2010), (512, 512, 4096), (700, 130, 256), (1000, 64, 128), (1023, 513, 1600), (4099, 256, 128), (5000, 100, 300),
          (20_001, 256, 128), (9000, 500, 64), (2049, 2050, 640), (4096, 4096, 512), (3000, 3100, 1000),
          (5000, 3000, 300), (2500, 2500, 1000), (600, 520, 4096),
          (9000, 47, 128), (9001, 64, 30), (9001, 128, 33), (40_001, 192, 90), (9000, 320, 160), (20_000, 256, 190), (20_000, 64, 225),
          (9999, 256, 256), (3001, 33, 100), (40_000, 1, 64),
          (50_001, 100, 128), (50_001, 172, 90), (40_000, 300, 128), (40_001, 301, 60), (30_000, 500, 64), (30_003, 255, 190),
          (20_000, 257, 250), (20_000, 443, 33)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products_are_exact(m, n, k):
    say("product", m, n, k)
    (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 3)
    want = product(a, sa, w, sw)
    for out in TYPES:
        got = trspmm.matmul_mx4(a, sa, w, sw, dtype=out)
        assert got.dtype is out and torch.equal(got, want.to(out)), (out, int((got != want.to(out)).sum()))
    bias = rand((n,), torch.float32, 5).half().float()      # the sum with it is rounded once, to 32 bits
    got = trspmm.matmul_mx4(a, sa, w, sw, bias=bias, dtype=torch.float32)
    assert torch.equal(got, (want + bias.double()).float())


@pytest.mark.parametrize("m,n,k", [(1, 300, 5000), (40, 70, 8192), (300, 400, 8192), (600, 1100, 1000), (2050, 300, 224)])
def test_products_of_wide_scales(m, n, k):
    say("wide scales", m, n, k)
    (a, sa), (w, sw) = operand(m, k, 1, 100, 140), operand(n, k, 3, 110, 150)
    want = product(a, sa, w, sw)
    size = torch.mm(values(a, sa).abs(), values(w, sw).abs().t().contiguous())
    got = trspmm.matmul_mx4(a, sa, w, sw, dtype=torch.float32)
    assert bool(((got.double() - want).abs() <= k * 2.0 ** -23 * size).all())
    # the same of the largest term alone: what is far below it is lost to rounding, what is near is not
    assert torch.equal(got, trspmm.matmul_mx4(a, sa, w, sw, dtype=torch.float32))


@pytest.mark.parametrize("m,n,k", [(1, 40, 100), (20, 70, 1100), (130, 140, 520), (600, 700, 290), (3000, 300, 100), (1500, 1900, 1000),
                                   (500, 400, 3000), (9000, 128, 120), (9000, 30, 250), (30_000, 172, 100), (20_000, 400, 64)])
def test_product_strides(m, n, k):
    say("product strides", m, n, k)
    b = blocks_of(k)
    (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 3)
    want = product(a, sa, w, sw)
    wide = torch.full((m, 16 * b + 48), 0x77, dtype=torch.uint8, device="cuda")
    wide[:, :16 * b] = a
    for extra in (1, 2, 3, 4, 16):      # scales' rows on every boundary, NaN bytes between them
        scale = torch.full((m + 1, b + extra), 255, dtype=torch.uint8, device="cuda")
        scale[:m, :b] = sa.view(torch.uint8)
        scale_w = torch.full((n + 1, b + extra), 255, dtype=torch.uint8, device="cuda")
        scale_w[:n, :b] = sw.view(torch.uint8)
        obuf, out = guarded(m, n, n + extra, torch.float32, 7.0)
        trspmm.matmul_mx4(wide[:, :16 * b], scale[:m, :b], w, scale_w[:n, :b].view(E8M0), out=out)
        assert torch.equal(out, want.float()) and untouched(obuf, m, n, n + extra, 7.0), extra
        skewed = scale.view(-1)[extra:][:m * b].view(m, b)       # starts off the boundary too
        skewed.copy_(sa.view(torch.uint8))
        assert torch.equal(trspmm.matmul_mx4(a, skewed, w, sw, dtype=torch.float32), want.float())
    odd = torch.zeros(m * 16 * b + 3, dtype=torch.uint8, device="cuda")[3:].view(m, 16 * b)
    odd.copy_(a)
    assert torch.equal(trspmm.matmul_mx4(odd, sa, w, sw, dtype=torch.float32), want.float())


@pytest.mark.parametrize("m,n,k", [(1, 40, 100), (40, 50, 1100), (300, 400, 1000), (3000, 256, 128), (9000, 256, 224), (9000, 64, 30), (40_000, 300, 90)])
def test_blocks_of_nan_reach_their_row_and_channel_alone(m, n, k):
    say("nan blocks", m, n, k)
    (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 3)
    sa.view(torch.uint8)[m - 1, -1] = 255
    sw.view(torch.uint8)[n // 2, 0] = 255
    got = trspmm.matmul_mx4(a, sa, w, sw, dtype=torch.float32)
    bad = torch.zeros((m, n), dtype=torch.bool, device="cuda")
    bad[m - 1], bad[:, n // 2] = True, True
    assert torch.equal(torch.isnan(got), bad)
    assert torch.equal(got[~bad], product(a, sa, w, sw).float()[~bad])


def test_another_stream_and_a_graph():
    say("stream, graph")
    x, w = rand((50, 300), torch.float16, 1), rand((70, 300), torch.float16, 2)
    weight = 1 + 0.1 * rand((300,), torch.float32, 3)
    codes, scale = trspmm.quant_mx4(w)

    def run():
        q, s, r = trspmm.rms_norm_mx4(x, weight, x, EPS)
        return trspmm.matmul_mx4(q, s, codes, scale), r, trspmm.dequant_mx4(q, s, 300)

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, s, r = trspmm.rms_norm_mx4(x, weight, x, EPS, stream=side)
    got = trspmm.matmul_mx4(q, s, codes, scale, stream=side)
    side.synchronize()
    assert torch.equal(got, want[0]) and torch.equal(r, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for turn in range(4):
        x.copy_(rand((50, 300), torch.float16, 10 + turn))
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), turn


def test_more_channels_than_a_walk_can_have():
    """600,000,001 channels of one block: weights of 9.6 GB, addresses past 32 bits, more strips than a grid of panels holds."""
    say("many channels")
    n = 600_000_001
    if torch.cuda.mem_get_info()[0] < 24e9:
        pytest.skip("not enough memory")
    w, sw = torch.zeros((n, 16), dtype=torch.uint8, device="cuda"), torch.full((n, 1), 127, dtype=torch.uint8, device="cuda")
    a, sa = operand(2, 32, 1)
    ends, scale = operand(300, 32, 3)
    for at in (0, 268_435_300, n - 300):
        w[at:at + 300], sw[at:at + 300] = ends, scale.view(torch.uint8)
    got = trspmm.matmul_mx4(a, sa, w, sw, dtype=torch.float32)
    want = product(a, sa, ends, scale).float()
    for at in (0, 268_435_300, n - 300):
        assert torch.equal(got[:, at:at + 300], want), at
        got[:, at:at + 300] = 0
    assert not bool(got.any())


def test_offsets_past_32_bits():
    """2.2 million rows of 1000: elements of x, of the residual's sum and of the product past 2^31; the last rows are those of a call of their own."""
    say("long offsets")
    rows, width = 2_200_001, 1000
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("not enough memory")
    x = torch.ones((rows, width), dtype=torch.float16, device="cuda")
    last = slice(rows - 301, rows)
    x[last] = rand((301, width), torch.float16, 1)
    weight = 1 + 0.1 * rand((width,), torch.float32, 2)

    def same(got, want):
        assert all(torch.equal(a[last].view(torch.uint8) if a.dtype == E8M0 else a[last], b.view(torch.uint8) if b.dtype == E8M0 else b)
                   for a, b in zip(got, want))
    codes, scale = trspmm.quant_mx4(x)
    same((codes, scale), trspmm.quant_mx4(x[last].clone()))
    same((trspmm.dequant_mx4(codes, scale, width),), (trspmm.dequant_mx4(codes[last].clone(), scale[last].clone(), width),))
    same(trspmm.rms_norm_mx4(x, weight, x, EPS), trspmm.rms_norm_mx4(x[last].clone(), weight, x[last].clone(), EPS))
    del x
    w, sw = operand(width, width, 3)
    a, sa = operand(301, width, 5)
    codes[last], scale.view(torch.uint8)[last] = a, sa.view(torch.uint8)
    same((trspmm.matmul_mx4(codes, scale, w, sw, dtype=torch.bfloat16),), (product(a, sa, w, sw).to(torch.bfloat16),))


def test_equal_inputs_give_equal_bits():
    say("again")
    for m, n, k in [(1, 500, 4000), (50, 500, 4000), (900, 800, 700), (5000, 256, 128)]:
        (a, sa), (w, sw) = operand(m, k, 1, 100, 150), operand(n, k, 3, 100, 150)
        first = trspmm.matmul_mx4(a, sa, w, sw, dtype=torch.float32)
        assert all(torch.equal(first, trspmm.matmul_mx4(a, sa, w, sw, dtype=torch.float32)) for _ in range(3))


def test_refusals():
    say("refusals")
    x = rand((4, 64), torch.float16, 1)
    codes, scale = trspmm.quant_mx4(x)
    w = torch.ones(64, device="cuda")
    for call in [lambda: trspmm.quant_mx4(x.cpu()), lambda: trspmm.quant_mx4(x[0]), lambda: trspmm.quant_mx4(x.int()),
                 lambda: trspmm.quant_mx4(x, out=codes[:, :16]), lambda: trspmm.quant_mx4(x, out=codes.view(torch.int8)),
                 lambda: trspmm.quant_mx4(x, scale=scale.float()), lambda: trspmm.quant_mx4(x, scale=scale[:3]),
                 lambda: trspmm.quant_mx4(x, out=torch.empty(4 * 32 + 1, dtype=torch.uint8, device="cuda")[1:].view(4, 32)),
                 lambda: trspmm.dequant_mx4(codes, scale, 65), lambda: trspmm.dequant_mx4(codes, scale, 32),
                 lambda: trspmm.dequant_mx4(codes, scale, -1), lambda: trspmm.dequant_mx4(codes, scale[:3], 64),
                 lambda: trspmm.dequant_mx4(codes[:, :24], scale, 64), lambda: trspmm.dequant_mx4(codes, scale.float(), 64),
                 lambda: trspmm.dequant_mx4(codes, scale, 64, dtype=torch.int8), lambda: trspmm.dequant_mx4(codes.int(), scale, 64),
                 lambda: trspmm.rms_norm_mx4(x, w[:63]), lambda: trspmm.rms_norm_mx4(x, w, r_out=x),
                 lambda: trspmm.rms_norm_mx4(x, w, x[:3]), lambda: trspmm.rms_norm_mx4(x, w, out=codes[:3]),
                 lambda: trspmm.matmul_mx4(codes, scale, codes[:, :16], scale[:, :1]), lambda: trspmm.matmul_mx4(codes, scale[:3], codes, scale),
                 lambda: trspmm.matmul_mx4(codes, scale, codes, scale[:, :1]), lambda: trspmm.matmul_mx4(codes, scale, codes, scale, bias=w),
                 lambda: trspmm.matmul_mx4(codes, scale, codes, scale, bias=torch.ones(4, dtype=torch.float16, device="cuda")),
                 lambda: trspmm.matmul_mx4(codes, scale, codes, scale, dtype=torch.float64),
                 lambda: trspmm.matmul_mx4(codes, scale, codes, scale, out=torch.empty((4, 5), dtype=torch.float16, device="cuda"))]:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(nat.TrsError):
        trspmm.rms_norm_mx4(x, w, eps=0.0)
    with pytest.raises(nat.TrsError):
        trspmm.rms_norm_mx4(x, w, x.bfloat16())


@pytest.mark.parametrize("blocks", [1, 3, 16, 33])
def test_a_single_rows_stride_says_nothing(blocks):
    """One row of codes with its scales behind it, 17 bytes a block: it starts on a 16-byte boundary, whatever follows it."""
    say("one row", blocks)
    k = 32 * blocks
    x, weight = rand((1, k), torch.float16, 1), 1 + 0.1 * rand((k,), torch.float32, 2)

    def packed():
        row = torch.full((1, 17 * blocks + 5), 9, dtype=torch.uint8, device="cuda")
        assert row[:, :16 * blocks].stride(0) % 16 != 0
        return row, row[:, :16 * blocks], row[:, 16 * blocks:17 * blocks]

    for quantise in (lambda **out: trspmm.quant_mx4(x, **out), lambda **out: trspmm.rms_norm_mx4(x, weight, eps=EPS, **out)):
        want, byte = (t.view(torch.uint8) for t in quantise()[:2])
        row, codes, scale = packed()
        got = quantise(out=codes, scale=scale)
        assert got[0].data_ptr() == codes.data_ptr() and got[1].data_ptr() == scale.data_ptr()
        assert torch.equal(codes, want) and torch.equal(scale, byte) and bool((row[:, 17 * blocks:] == 9).all())
    assert torch.equal(trspmm.dequant_mx4(codes, scale, k), trspmm.dequant_mx4(want, byte, k))
    for rows in (1, 40, 3000):
        b, sb = operand(rows, k, 3)
        # the packed row as the rows and as the channels
        assert torch.equal(trspmm.matmul_mx4(codes, scale, b, sb), trspmm.matmul_mx4(want, byte, b, sb))
        assert torch.equal(trspmm.matmul_mx4(b, sb, codes, scale), trspmm.matmul_mx4(b, sb, want, byte))


def test_the_terms_of_wide_scales_are_all_there():
    """One block of a row far above the others, by 2^13: what rounds is the largest term's share, so the sum has to be within
    k 2^-23 of the sum of the products' sizes, and without its largest block within that of the rest."""
    say("largest term")
    for m, n, k in [(1, 300, 5000), (300, 400, 4096), (9000, 64, 250)]:
        (a, sa), (w, sw) = operand(m, k, 1), operand(n, k, 3)
        high = sa.view(torch.uint8).clone()
        high[:, 0] += 13
        got = trspmm.matmul_mx4(a, high, w, sw, dtype=torch.float32).double()
        rest = a.clone()
        rest[:, :16] = 0
        less = trspmm.matmul_mx4(rest, high, w, sw, dtype=torch.float32).double()
        for value, codes in ((got, a), (less, rest)):
            size = torch.mm(values(codes, high).abs(), values(w, sw).abs().t().contiguous())
            assert bool(((value - product(codes, high, w, sw)).abs() <= k * 2.0 ** -23 * size).all())


def test_every_pair_of_scales():
    """One product of codes for each pair of scale bytes, from 2^-254 on, 255 among them: a 32-bit float as the product rounds to
    it, zeros and infinities too."""
    say("pairs of scales")
    byte = torch.arange(256, dtype=torch.int64, device="cuda")
    exponent = byte[:, None] + byte[None, :] - 254
    bad = (byte == 255)[:, None] | (byte == 255)[None, :]
    for rows, blocks in ((256, 1), (256, 16), (10_240, 1), (4096, 16)):
        times = rows // 256
        a, w = (torch.zeros((r, 16 * blocks), dtype=torch.uint8, device="cuda") for r in (rows, 256))
        sa, sw = (torch.full((r, blocks), 127, dtype=torch.uint8, device="cuda") for r in (rows, 256))
        sa[:, 0], sw[:, 0] = byte.repeat(times).to(torch.uint8), byte.to(torch.uint8)
        w[:, 0] = 2
        for code, size in ((0, 0.0), (2, 1.0), (10, -1.0)):
            a[:, 0] = code
            got = trspmm.matmul_mx4(a, sa, w, sw, dtype=torch.float32).view(times, 256, 256)
            want = torch.where(bad, float("nan"), power(exponent) * size).float()
            assert bool(((got == want) | (torch.isnan(got) & torch.isnan(want))).all()), (rows, blocks, code)
