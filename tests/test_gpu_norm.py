"""trspmm.rms_norm, rms_norm_i8 and rms_norm_grad against the definitions in 64 bits.

Bounds (u = 2^-24, one rounding in 32 bits): a row's sum of squares adds at most 32 products in a lane and then
halves (long rows: up to width / 2048 products), so it is off by (40 + width / 2048) u of itself and the factor
1 / sqrt by half of that; a normed value takes four more roundings.  FAR covers that, doubled."""
import pytest
import torch

import trspmm
from trspmm import _native as nat
from trspmm import dense

pytestmark = pytest.mark.gpu

ROUND = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
TYPES = list(ROUND)
EPS = 1e-5


def far(width):
    return (60 + width / 1024) * 2.0 ** -24


def say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(dtype)


def weights(width, dtype, seed):
    return (1 + 0.2 * torch.randn(width, generator=gen(seed), device="cuda")).to(dtype)


def exact(x, w, res, eps=EPS):
    h = x.double() + (0 if res is None else res.double())
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()
    return h, y


def close(out, ref, rel):
    bound = ref.abs() * (rel + ROUND[out.dtype] * 1.01) + TINY[out.dtype]
    off = (out.double() - ref).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


def check_norm(x, w, res, y, r, eps=EPS):
    h, ref = exact(x, w, res, eps)
    close(y, ref, far(x.shape[1]))
    if res is None:
        assert r is None
    else:
        close(r, h, 2.0 ** -24)


def check_codes(x, w, res, q, scale, r, eps=EPS):
    h, ref = exact(x, w, res, eps)
    peak = ref.abs().amax(1)
    assert q.dtype is torch.int8 and scale.dtype is torch.float32
    assert bool(((scale.double() - peak / 127).abs() <= peak / 127 * (far(x.shape[1]) + 2.0 ** -22) + 2.0 ** -149).all())
    some = peak > 1e-30
    steps = ref[some] / (peak[some] / 127)[:, None]
    off = (q[some].double() - steps).abs()
    assert bool((off <= 0.5 + 127 * 2 * (far(x.shape[1]) + 2.0 ** -22)).all()), float(off.max())
    assert bool((q[~some] == 0).all()) and int(q.min()) >= -127
    if res is not None:
        close(r, h, 2.0 ** -24)


MIXES = [(x, r) for x in TYPES for r in [None, *TYPES] if r is None or r is x or torch.float32 in (x, r)]


@pytest.mark.parametrize("x_type,r_type", MIXES)
@pytest.mark.parametrize("w_type", TYPES)
def test_types(x_type, r_type, w_type):
    say("types", x_type, r_type, w_type)
    for rows, width in [(37, 96), (9, 1000)]:
        x, w = rand((rows, width), x_type, 1), weights(width, w_type, 2)
        res = None if r_type is None else rand((rows, width), r_type, 3, 2.0)
        for y_type in TYPES:
            check_norm(x, w, res, *trspmm.rms_norm(x, w, res, EPS, y_type))
        check_codes(x, w, res, *trspmm.rms_norm_i8(x, w, res, EPS))


@pytest.mark.parametrize("width", [1, 2, 5, 7, 8, 9, 16, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000,
                                   1023, 2047, 2048, 2049, 4095, 4096, 4097, 5000, 8191, 8192, 8193, 12_001, 20_000])
def test_widths(width):
    say("width", width)
    for rows in (1, 33):
        x, w, res = rand((rows, width), torch.float16, 1), weights(width, torch.float16, 2), rand((rows, width), torch.float16, 3)
        check_norm(x, w, res, *trspmm.rms_norm(x, w, res, EPS))
        check_codes(x, w, res, *trspmm.rms_norm_i8(x, w, res, EPS))
        check_norm(x, w, None, *trspmm.rms_norm(x, w, eps=EPS))
        f, r = x.float(), rand((rows, width), torch.bfloat16, 4)
        check_codes(f, w, r, *trspmm.rms_norm_i8(f, w, r, EPS))


def grad_reference(grad, r, w, grad_r, eps=EPS):
    r, dy = r.double(), grad.double()
    s = 1 / torch.sqrt((r * r).mean(1, keepdim=True) + eps)
    u, g = r * s, dy * w.double()
    mean, size = (g * u).mean(1, keepdim=True), (g * u).abs().mean(1, keepdim=True)
    more = 0 if grad_r is None else grad_r.double()
    dr = s * (g - u * mean) + more
    dr_size = s * (g.abs() + u.abs() * size) + (0 if grad_r is None else more.abs())
    return dr, dr_size, (dy * u).sum(0), (dy * u).abs().sum(0)


def check_grad(grad, r, w, grad_r, dr, dw, eps=EPS):
    rows, width = r.shape
    ref, size, wref, wsize = grad_reference(grad, r, w, grad_r, eps)
    off = (dr.double() - ref).abs() - (size * 2 * far(width) + ref.abs() * ROUND[dr.dtype] * 1.01 + TINY[dr.dtype])
    assert bool((off <= 0).all()), float(off.max())
    # the weight's sum: the rows of a workgroup, then shares of the workgroups
    off = (dw.double() - wref).abs() - wsize * (far(width) + (rows / 1024 + 100) * 2.0 ** -24)
    assert dw.dtype is torch.float32 and bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("d_type,r_type", [(d, r) for d, r in MIXES if r is not None])
@pytest.mark.parametrize("w_type", TYPES)
def test_grad_types(d_type, r_type, w_type):
    say("grad types", d_type, r_type, w_type)
    for rows, width in [(70, 96), (11, 1000)]:
        r, w, g, more = rand((rows, width), r_type, 1), weights(width, w_type, 2), rand((rows, width), d_type, 3), rand((rows, width), r_type, 4)
        check_grad(g, r, w, more, *trspmm.rms_norm_grad(g, r, w, more, EPS))
        check_grad(g, r, w, None, *trspmm.rms_norm_grad(g, r, w, eps=EPS))


@pytest.mark.parametrize("width", [1, 3, 8, 9, 64, 65, 100, 128, 250, 257, 512, 513, 1000, 2048, 2049, 4096, 5001, 8192, 8193, 12_001])
@pytest.mark.parametrize("rows", [1, 2, 300, 3001])
def test_grad_sizes(width, rows):
    say("grad", rows, width)
    r, w, g, more = rand((rows, width), torch.bfloat16, 1), weights(width, torch.float32, 2), rand((rows, width), torch.bfloat16, 3), rand((rows, width), torch.bfloat16, 4)
    check_grad(g, r, w, more, *trspmm.rms_norm_grad(g, r, w, more, EPS))


@pytest.mark.parametrize("rows,width", [(5, 40), (3, 700), (2, 9000)])
def test_grad_against_differences(rows, width):
    """<dr, v> and <dweight, z> against central differences of the definition in 64 bits (step 1e-4: their
    own error is some 1e-8 of the terms), within the gradient's bound summed over the elements."""
    say("differences", rows, width)
    r, w, g, more = (rand(s, torch.float32, k) for k, s in enumerate([(rows, width), (width,), (rows, width), (rows, width)]))
    v, z = rand((rows, width), torch.float64, 7), rand((width,), torch.float64, 8)
    dr, dw = trspmm.rms_norm_grad(g, r, w, more, EPS)

    def loss(r, w):
        return (r / torch.sqrt((r * r).mean(1, keepdim=True) + EPS) * w * g.double()).sum() + (r * more.double()).sum()

    r, w, h = r.double(), w.double(), 1e-4
    _, size, _, wsize = grad_reference(g, r, w, more)
    bound = float((size * v.abs()).sum()) * (2 * far(width) + 2.0 ** -24 + 1e-7)
    assert abs(float((loss(r + h * v, w) - loss(r - h * v, w)) / (2 * h) - (dr.double() * v).sum())) <= bound
    bound = float((wsize * z.abs()).sum()) * (far(width) + 100 * 2.0 ** -24 + 1e-7)
    assert abs(float((loss(r, w + h * z) - loss(r, w - h * z)) / (2 * h) - (dw.double() * z).sum())) <= bound


@pytest.mark.parametrize("width", [40, 127, 600, 5000, 9001])
def test_special_rows(width):
    """Rows of zeros, with a NaN or an infinity, too large for 32-bit squares, tiny; the rows beside them."""
    say("special", width)
    x, w = rand((12, width), torch.float32, 1), weights(width, torch.float32, 2)
    x[1] = 0
    x[2, width // 2] = float("nan")
    x[3, 0] = float("inf")
    x[4] *= 1e30
    x[5] *= 1e-30
    x[6, -1] = -float("inf")
    x[8] *= 3e37
    fine = [k for k in range(12) if k not in (2, 3, 6)]
    q, scale, _ = trspmm.rms_norm_i8(x, w, eps=EPS)
    y, _ = trspmm.rms_norm(x, w, eps=EPS)
    check_norm(x[fine], w, None, y[fine], None)
    check_codes(x[fine], w, None, q[fine], scale[fine], None)
    assert not q[1].any() and float(scale[1]) == 0
    assert bool(torch.isnan(scale[[2, 3, 6]]).all()) and not q[[2, 3, 6]].any()
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3, 0])) and bool(torch.isnan(y[6, -1]))
    w[1] = float("nan")                                                    # a weight that is not finite: every row
    q, scale, _ = trspmm.rms_norm_i8(x, w, eps=EPS)
    assert bool(torch.isnan(scale).all()) and not q.any()


@pytest.mark.parametrize("width", [40, 600, 9001])
def test_grad_of_special_rows(width):
    say("special grad", width)
    r, w, g = rand((9, width), torch.float32, 1), weights(width, torch.float32, 2), rand((9, width), torch.float32, 3)
    r[1] = 0
    r[4] *= 1e30
    r[6] *= 3e37
    check_grad(g, r, w, None, *trspmm.rms_norm_grad(g, r, w, eps=EPS))
    r[2, 3] = float("nan")
    dr, dw = trspmm.rms_norm_grad(g, r, w, eps=EPS)
    assert bool(torch.isnan(dr[2]).all()) and bool(torch.isfinite(dr[[0, 1, 3, 4, 5, 6, 7, 8]]).all())
    assert bool(torch.isnan(dw).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [5, 40, 127, 600, 2100, 5000, 9001])
def test_grad_where_products_pass_32_bits(width, dtype):
    """dr is ordinary where grad is as large as r, while their products are not: with squares in 32 bits and beyond, beside
    ordinary rows, and with a residual's own gradient."""
    say("large products", width, dtype)
    r, w, g, more = (rand((9, width), dtype, 1), weights(width, torch.float32, 2), rand((9, width), dtype, 3), rand((9, width), dtype, 4))
    for row, of_r, of_g in [(1, 1e17, 1e22), (2, 1e18, 1e24), (4, 3e37, 1e37), (5, 1e-3, 1e34), (7, 1e30, 1e30)]:
        r[row] *= of_r
        g[row] *= of_g
    dr, dw = trspmm.rms_norm_grad(g, r, w, more, EPS)
    assert bool(torch.isfinite(dr).all())
    check_grad(g, r, w, more, dr, dw)


@pytest.mark.parametrize("eps", [1e-5, 1e36, 1e38])
@pytest.mark.parametrize("width", [6, 40, 600, 4000, 9001])
def test_eps_beside_squares_beyond_32_bits(width, eps):
    """eps counts at every size of it and of the rows, also where squares pass 32 bits."""
    say("large eps", width, eps)
    x, w, g = rand((6, width), torch.float32, 1), weights(width, torch.float32, 2), rand((6, width), torch.float32, 3)
    for row, size in enumerate([1.0, 3e17, 1e19, 3e19, 1e21, 3e37]):
        x[row] *= size
    check_norm(x, w, None, *trspmm.rms_norm(x, w, eps=eps), eps=eps)
    check_codes(x, w, None, *trspmm.rms_norm_i8(x, w, eps=eps), eps=eps)
    check_grad(g, x, w, None, *trspmm.rms_norm_grad(g, x, w, eps=eps), eps=eps)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [13, 43, 130, 1001, 8199])
def test_strides_offsets_and_place(dtype, width):
    """Operands and outputs inside wider buffers at odd offsets; the new residual in the old one's place."""
    say("strides", dtype, width)
    rows, wide = 21, width + 18
    x, res = rand((rows, wide), dtype, 1)[:, 3:3 + width], rand((rows, wide), dtype, 2)[:, 5:5 + width]
    w = weights(width + 1, dtype, 3)[1:]
    old = res.clone()
    codes = torch.full((rows, wide), 99, dtype=torch.int8, device="cuda")
    q, scale, r = trspmm.rms_norm_i8(x, w, res, EPS, out=codes[:, 1:1 + width], r_out=res)
    assert r is res
    check_codes(x, w, old, q, scale, r)
    assert bool((codes[:, 0] == 99).all()) and bool((codes[:, 1 + width:] == 99).all())
    buf = torch.full((rows, wide), 9.0, dtype=dtype, device="cuda")
    res.copy_(old)
    y, r = trspmm.rms_norm(x, w, res, EPS, out=buf[:, 7:7 + width], r_out=res)
    check_norm(x, w, old, y, r)
    assert bool((buf[:, :7] == 9).all()) and bool((buf[:, 7 + width:] == 9).all())
    g, more = rand((rows, wide), dtype, 4)[:, 1:1 + width], rand((rows, wide), dtype, 5)[:, 2:2 + width]
    kept = more.clone()
    dr, dw = trspmm.rms_norm_grad(g, r, w, more, EPS, out=more)
    check_grad(g, r, w, kept, dr, dw)
    t = rand((width, rows), dtype, 6).t()
    check_norm(t, w, None, *trspmm.rms_norm(t, w, eps=EPS))
    one = rand((1, width), dtype, 7).expand(rows, width)                   # a broadcast residual
    check_norm(x, w, one, *trspmm.rms_norm(x, w, one, EPS))


def test_offsets_past_32_bits():
    say("far rows")
    x = torch.empty((300, 1 << 24), dtype=torch.float16, device="cuda")[:, 11:111]
    x.copy_(rand((300, 100), torch.float16, 1))
    w = weights(100, torch.float16, 2)
    check_norm(x, w, x, *trspmm.rms_norm(x, w, x, EPS))
    check_codes(x, w, x, *trspmm.rms_norm_i8(x, w, x, EPS))
    g = rand((300, 100), torch.float16, 3)
    check_grad(g, x, w, x, *trspmm.rms_norm_grad(g, x, w, x, EPS))


def test_many_rows():
    say("many rows")
    x, w, res = rand((70_001, 40), torch.float32, 1), weights(40, torch.float16, 2), rand((70_001, 40), torch.float16, 3)
    check_codes(x, w, res, *trspmm.rms_norm_i8(x, w, res, EPS))
    g = rand((70_001, 40), torch.float32, 4)
    check_grad(g, x, w, None, *trspmm.rms_norm_grad(g, x, w, eps=EPS))


@pytest.mark.parametrize("width", [512, 516])
def test_large_outputs(width):
    """Outputs of more than 128 MB, which leave past the caches where their rows allow it."""
    say("large", width)
    rows = 270_000
    x, w, res = rand((rows, width), torch.bfloat16, 1), weights(width, torch.float16, 2), rand((rows, width), torch.bfloat16, 3)
    check_codes(x, w, res, *trspmm.rms_norm_i8(x, w, res, EPS))
    check_norm(x, w, res, *trspmm.rms_norm(x, w, res, EPS))
    check_grad(x, res, w, x, *trspmm.rms_norm_grad(x, res, w, x, EPS))


def test_more_rows_than_a_launch():
    """2^24 + 1000 rows of 3: more than 2^32 threads at a workgroup a row; and at 32 rows a workgroup many."""
    say("rows past a launch")
    rows = (1 << 24) + 1000
    x, w, res = rand((rows, 3), torch.float16, 1), weights(3, torch.float16, 2), rand((rows, 3), torch.float16, 3)
    keep = torch.cat([torch.arange(50), torch.arange((1 << 24) - 50, rows)]).cuda()
    q, scale, r = trspmm.rms_norm_i8(x, w, res, EPS)
    check_codes(x[keep], w, res[keep], q[keep], scale[keep], r[keep])
    y, r = trspmm.rms_norm(x, w, res, EPS)
    check_norm(x[keep], w, res[keep], y[keep], r[keep])


def test_no_rows_no_width():
    say("empty")
    x, w = rand((4, 24), torch.float16, 1), weights(24, torch.float16, 2)
    y, r = trspmm.rms_norm(x[:0], w, x[:0])
    assert y.shape == (0, 24) and r.shape == (0, 24)
    assert trspmm.rms_norm_i8(x[:, :0], w[:0])[0].shape == (4, 0)
    dw = torch.full((24,), 5.0, device="cuda")
    dr, dw = trspmm.rms_norm_grad(x[:0], x[:0], w, dweight=dw)
    assert dr.shape == (0, 24) and not dw.any()


def test_codes_of_rows_without_width():
    """The scale of an empty row is a row of zeros' own, also in a scale that is given and holds something else; a product of
    such codes is the bias alone."""
    say("no width")
    x, w = rand((4, 24), torch.float16, 1)[:, :0], weights(24, torch.float16, 2)[:0]
    given = torch.full((4,), float("nan"), device="cuda")
    for kw in ({}, {"scale": given}):
        q, scale, _ = trspmm.rms_norm_i8(x, w, **kw)
        assert q.shape == (4, 0) and scale.tolist() == [0.0] * 4
    codes, bias = torch.empty((3, 0), dtype=torch.int8, device="cuda"), rand((3,), torch.float32, 3)
    out = trspmm.matmul_i8(q, scale, codes, torch.ones(3, device="cuda"), bias, torch.float32)
    assert torch.equal(out, bias.expand(4, 3))


def test_graph_replays_and_streams():
    say("graph")
    x, res, w = rand((500, 384), torch.float16, 1), rand((500, 384), torch.float16, 2), weights(384, torch.float16, 3)
    g, more = rand((500, 384), torch.float16, 4), rand((500, 384), torch.float16, 5)
    q, scale = torch.empty((500, 384), dtype=torch.int8, device="cuda"), torch.empty(500, device="cuda")
    r, dr, dw = torch.empty_like(x), torch.empty_like(x), torch.empty(384, device="cuda")
    ws = torch.empty(dense.rms_norm_grad_workspace_bytes(500, 384), dtype=torch.uint8, device="cuda")

    def step(stream=None):
        trspmm.rms_norm_i8(x, w, res, EPS, out=q, scale=scale, r_out=r, stream=stream)
        trspmm.rms_norm_grad(g, r, w, more, EPS, out=dr, dweight=dw, workspace=ws, stream=stream)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    step(s)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(rand((500, 384), torch.float16, 20 + i))
        for t in (scale, r, dr, dw):
            t.fill_(float("nan"))
        ws.fill_(255)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        q2, s2, r2 = trspmm.rms_norm_i8(x, w, res, EPS)
        dr2, dw2 = trspmm.rms_norm_grad(g, r2, w, more, EPS)
        for a, b in ((q, q2), (scale, s2), (r, r2), (dr, dr2), (dw, dw2)):
            assert torch.equal(a, b), f"replay {i}"


def test_refusals():
    say("refusals")
    x, w = rand((4, 24), torch.float16, 1), weights(24, torch.float16, 2)
    for kw in [dict(x=x.cpu()), dict(x=x[0]), dict(x=x.double()), dict(weight=w[:-1]), dict(weight=w.double()),
               dict(weight=torch.stack([w, w], 1)[:, 0]), dict(residual=x[:2]), dict(residual=x.long()), dict(r_out=x.clone()),
               dict(dtype=torch.int8), dict(out=x[:, :8])]:
        with pytest.raises(ValueError):
            trspmm.rms_norm(**{"x": x, "weight": w, **kw})
    for kw in [dict(out=x), dict(scale=torch.empty(3, device="cuda")), dict(scale=torch.empty(4, device="cuda").half())]:
        with pytest.raises(ValueError):
            trspmm.rms_norm_i8(x, w, **kw)
    for kw in [dict(grad=x[:2]), dict(grad_r=x.float()), dict(dweight=w)]:
        with pytest.raises(ValueError):
            trspmm.rms_norm_grad(**{"grad": x, "r": x, "weight": w, **kw})
    for call in [lambda: trspmm.rms_norm(x, w, eps=0.0), lambda: trspmm.rms_norm(x, w, eps=float("nan")),
                 lambda: trspmm.rms_norm_i8(x, w, x.bfloat16()), lambda: trspmm.rms_norm_grad(x, x.bfloat16(), w),
                 lambda: trspmm.rms_norm_grad(x, x.clone(), w, eps=-1.0), lambda: trspmm.rms_norm_grad(x, x.clone(), w, out=x)]:
        with pytest.raises(nat.TrsError) as e:
            call()
        assert e.value.code == 1
    lib, y = nat.lib(), torch.empty_like(x)
    good = (x.data_ptr(), 1, 24, None, 0, 0, w.data_ptr(), 1, EPS, 4, 24, y.data_ptr(), 1, 24, None, 0, None)
    for k, v in [(0, None), (1, 3), (2, 23), (3, x.data_ptr()), (6, None), (7, -1), (9, -1), (10, -1), (11, None), (12, 9), (13, 23)]:
        call = list(good)
        call[k] = v
        assert lib.trs_rms_norm(*call) == 1, k
    good = (x.data_ptr(), 1, 24, x.data_ptr(), 1, 24, w.data_ptr(), 1, None, 0, EPS, 4, 24, y.data_ptr(), 24,
            torch.empty(24, device="cuda").data_ptr(), 0, 0, None)
    assert lib.trs_rms_norm_grad(*good) == 1                               # no workspace
