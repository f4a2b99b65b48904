"""trspmm.matmul_i8 against integer products in 64 bits.

The integer sums are exact.  Taken to 32-bit floats (one rounding), times two scales (two more) and with the bias
added (one more), an output is off by at most 4 x 2^-24 of the product and of the bias, and its type's rounding."""
import pytest
import torch

import trspmm
from trspmm import _native as nat

pytestmark = pytest.mark.gpu

ROUND = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
TYPES = list(ROUND)


def say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def codes(rows, k, seed, low=-128):
    return torch.randint(low, 128, (rows, k), generator=gen(seed), device="cuda", dtype=torch.int8)


def scales(n, seed, width=64):
    return (0.5 + torch.rand(n, generator=gen(seed), device="cuda")) / (73 * width ** 0.25)


def sums(a, w):
    return torch.mm(a.double(), w.double().t().contiguous())


def check(out, a, sa, w, sw, bias):
    prod = sums(a, w) * sa.double()[:, None] * sw.double()
    ref = prod if bias is None else prod + bias.double()
    size = prod.abs() + (0 if bias is None else bias.double().abs())
    bound = size * 4 * 2.0 ** -24 + ref.abs() * ROUND[out.dtype] * 1.01 + TINY[out.dtype]
    off = (out.double() - ref).abs() - bound
    assert out.shape == ref.shape and bool((off <= 0).all()), float(off.max())


def run(m, n, k, dtype=torch.float16, bias=True, seed=1):
    a, w = codes(m, k, seed), codes(n, k, seed + 1)
    sa, sw = scales(m, seed + 2, max(k, 1)), scales(n, seed + 3, max(k, 1))
    b = torch.randn(n, generator=gen(seed + 4), device="cuda") if bias else None
    check(trspmm.matmul_i8(a, sa, w, sw, b, dtype), a, sa, w, sw, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 2, 5, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300, 513])
def test_rows(m, dtype):
    say("rows", m, dtype)
    run(m, 200, 320, dtype, bias=m % 2 == 0)
    run(m, 37, 67, dtype)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 79, 100, 127, 128, 129, 160, 192, 250, 256, 257,
                               384, 500, 512, 640, 1000, 1024, 1030, 2047, 4096, 4100, 8192, 10_000])
def test_inner_lengths(k):
    say("inner", k)
    run(3, 130, k)
    run(20, 70, k)
    run(200, 140, k)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 41, 63, 64, 65, 127, 128, 129, 250, 256, 257, 515])
def test_channels(n):
    say("channels", n)
    for m in (1, 40, 150, 700):
        run(m, n, 128, TYPES[n % 3])
        run(m, n, 131, TYPES[n % 3])


@pytest.mark.parametrize("m,n,k", [(2048, 2048, 512), (2000, 2100, 1000), (2049, 1030, 256), (513, 4097, 2049), (70_000, 96, 64),
                                   (33_000, 256, 128), (66_001, 200, 100), (70_000, 41, 128), (40_001, 100, 77), (4096, 8192, 256),
                                   (5000, 3000, 600), (5000, 3001, 601), (1500, 1500, 1031), (200, 4096, 4096), (500, 4096, 4095),
                                   (250, 4000, 2049), (60_000, 256, 200),
                                   (800_001, 200, 120), (790_000, 300, 127), (740_000, 1000, 128), (5_900_001, 136, 16), (1, 16_000, 8192), (8, 8192, 16_384), (64, 4096, 4096)])
def test_large(m, n, k):
    say("large", m, n, k)
    run(m, n, k, torch.bfloat16)


@pytest.mark.parametrize("m", [1, 16, 64, 130, 600])
@pytest.mark.parametrize("k", [1024, 131_071])
def test_exact_sums(m, k):
    """Scales of 1 and sums below 2^24 times 32: the float32 output is the integer; the largest sums do not wrap."""
    say("exact", m, k)
    one = torch.ones(max(m, 600), device="cuda")
    a, w = codes(m, 1024, 1, -127), codes(600, 1024, 2, -127)
    out = trspmm.matmul_i8(a, one[:m], w, one[:600], dtype=torch.float32)
    assert torch.equal(out.double(), sums(a, w))
    low = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    out = trspmm.matmul_i8(low, one[:m], low[:1], one[:1], dtype=torch.float32)
    assert bool((out == float(16384 * k)).all())


def test_no_rows_channels_or_inner_length():
    say("empty")
    a, w, one = codes(6, 64, 1), codes(10, 64, 2), torch.ones(10, device="cuda")
    assert trspmm.matmul_i8(a[:0], one[:0], w, one).shape == (0, 10)
    assert trspmm.matmul_i8(a, one[:6], w[:0], one[:0]).shape == (6, 0)
    bias = torch.randn(10, device="cuda")
    out = trspmm.matmul_i8(a[:, :0], one[:6], w[:, :0], one, bias, torch.float32)
    assert torch.equal(out, bias.expand(6, 10))                            # an empty sum is 0


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("k", [64, 75, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_offsets(m, k, dtype):
    say("strides", m, k, dtype)
    n = 150
    for lead in (1, 4, 16):
        a, w = codes(m, k + 2 * lead, 1)[:, lead:lead + k], codes(n, k + 3 * lead, 2)[:, lead:lead + k]
        sa, sw, b = scales(m + 1, 3)[1:], scales(n + 3, 4)[3:], torch.randn(n + 1, device="cuda")[1:]
        buf = torch.full((m, n + 9), 9.0, dtype=dtype, device="cuda")
        check(trspmm.matmul_i8(a, sa, w, sw, b, out=buf[:, 5:5 + n]), a, sa, w, sw, b)
        assert bool((buf[:, :5] == 9).all()) and bool((buf[:, 5 + n:] == 9).all())
    t = codes(k, m, 5).t()
    check(trspmm.matmul_i8(t, sa, w, sw), t, sa, w, sw, None)
    one = codes(1, k, 6).expand(m, k)
    check(trspmm.matmul_i8(one, sa, w, sw), one, sa, w, sw, None)


@pytest.mark.parametrize("m", [3, 200])
def test_offsets_past_32_bits(m):
    say("far rows", m)
    far = torch.empty((300, 1 << 24), dtype=torch.int8, device="cuda")
    a, w = far[:, 16:272], far[:, 4096:4096 + 256]
    a.copy_(codes(300, 256, 1))
    w.copy_(codes(300, 256, 2))
    sa, sw = scales(300, 3), scales(300, 4)
    check(trspmm.matmul_i8(a[300 - m:], sa[:m], w, sw), a[300 - m:], sa[:m], w, sw, None)
    out = torch.empty((300, 1 << 24), dtype=torch.float16, device="cuda")[:, 3:303]
    check(trspmm.matmul_i8(a, sa, w, sw, out=out), a, sa, w, sw, None)


def test_scales_that_are_zero_or_not_finite():
    say("scales")
    for m in (5, 100):
        a, w = codes(m, 96, 1), codes(70, 96, 2)
        sa, sw = scales(m, 3), scales(70, 4)
        sa[1], sa[2], sw[3] = 0.0, float("nan"), 0.0
        out = trspmm.matmul_i8(a, sa, w, sw)
        keep = [k for k in range(m) if k != 2]
        check(out[keep], a[keep], sa[keep], w, sw, None)
        assert bool(torch.isnan(out[2]).all()) and not out[1].any()


@pytest.mark.parametrize("m,n,k", [(4, 512, 2048), (700, 300, 500)])
def test_graph_replays_and_streams(m, n, k):
    say("graph", m, n, k)
    a, w, sa, sw = codes(m, k, 1), codes(n, k, 2), scales(m, 3), scales(n, 4)
    out = torch.empty((m, n), dtype=torch.float16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other = trspmm.matmul_i8(a, sa, w, sw, stream=s)
    s.synchronize()
    assert torch.equal(other, trspmm.matmul_i8(a, sa, w, sw, out=out))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        trspmm.matmul_i8(a, sa, w, sw, out=out)
    for i in range(4):
        a.copy_(codes(m, k, 30 + i))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, trspmm.matmul_i8(a, sa, w, sw)), f"replay {i}"


def test_refusals():
    say("refusals")
    a, w, sa, sw = codes(4, 32, 1), codes(6, 32, 2), scales(4, 3), scales(6, 4)
    for kw in [dict(a=a.cpu()), dict(a=a.short()), dict(w=w[:, :16]), dict(w=w.float()), dict(a_scale=sa[:3]), dict(a_scale=sa.half()),
               dict(w_scale=sw[:, None]), dict(bias=sa), dict(dtype=torch.int8), dict(out=torch.empty((4, 7), device="cuda")),
               dict(a=a[0])]:
        with pytest.raises(ValueError):
            trspmm.matmul_i8(**{"a": a, "a_scale": sa, "w": w, "w_scale": sw, **kw})
    long = torch.zeros((1, 131_072), dtype=torch.int8, device="cuda")
    with pytest.raises(nat.TrsError) as e:
        trspmm.matmul_i8(long, sa[:1], long, sw[:1])
    assert e.value.code == 5
    lib, out = nat.lib(), torch.empty((4, 6), device="cuda")
    good = (a.data_ptr(), 32, sa.data_ptr(), w.data_ptr(), 32, sw.data_ptr(), None, 4, 6, 32, out.data_ptr(), 0, 6, None)
    for k, v in [(0, None), (1, 31), (2, None), (3, None), (4, 31), (5, None), (7, -1), (8, -1), (9, -1), (10, None), (11, 5), (12, 5)]:
        call = list(good)
        call[k] = v
        assert lib.trs_matmul_i8(*call) == 1, k


def test_an_output_of_another_type_than_asked_for_is_refused():
    """Every operator that takes both; where no type is asked for, the output's is the one."""
    say("dtype and out")
    a, w, sa, sw = codes(4, 32, 1), codes(6, 32, 2), scales(4, 3), scales(6, 4)
    x, ids, one = torch.randn((6, 32), device="cuda"), torch.tensor([0, 5, 1, 1], device="cuda"), torch.ones(32, device="cuda")
    calls = [((4, 6), lambda **kw: trspmm.matmul_i8(a, sa, w, sw, **kw)), ((4, 32), lambda **kw: trspmm.embed(x, ids, **kw)),
             ((9, 32), lambda **kw: trspmm.embed_grad(x[:4], ids, 9, **kw)), ((6, 32), lambda **kw: trspmm.rms_norm(x, one, **kw)[0])]
    for shape, call in calls:
        for asked in TYPES:
            for given in TYPES:
                out = torch.full(shape, 7.0, dtype=given, device="cuda")
                if given is not asked:
                    with pytest.raises(ValueError):
                        call(out=out, dtype=asked)
                    assert bool((out == 7).all())
                kw = {"dtype": asked} if given is asked else {}
                assert call(out=out, **kw).dtype is given and not bool((out == 7).all())
