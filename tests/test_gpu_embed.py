"""trspmm.embed and embed_grad against the definition in 64 bits: types, id widths, odd widths, strides and
offsets, padded ids, ids of one row, tables without rows, graphs and streams.

A looked-up element is one 32-bit product, rounded once: off by 2^-24 of itself and the output type's rounding.
A gradient is a sum of n terms in 32 bits, off by at most (n + 2) 2^-24 of the sum of their sizes, and the
rounding."""
import pytest
import torch

import trspmm
from trspmm import _native as nat
from trspmm import dense

pytestmark = pytest.mark.gpu

ROUND = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # half a subnormal step
TYPES = list(ROUND)


def say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(shape, dtype, seed):
    return torch.randn(shape, generator=gen(seed), device="cuda").to(dtype)


def some_ids(count, rows, dtype, seed, skew=1, pad=0.1):
    g = gen(seed)
    ids = (torch.rand(count, generator=g, device="cuda", dtype=torch.float64) ** skew * max(rows, 1)).long()
    ids = torch.where(torch.rand(count, generator=g, device="cuda") < pad, -1, ids.clamp(max=rows - 1))
    return ids.to(dtype)


def check_embed(out, table, ids, scale):
    ref = torch.zeros(out.shape, dtype=torch.float64, device="cuda")
    there = (ids >= 0) & (ids < table.shape[0])
    ref[there] = table[ids[there].long()].double() * scale
    bound = ref.abs() * (2.0 ** -24 + ROUND[out.dtype]) * 1.01 + TINY[out.dtype]
    assert bool(((out.double() - ref).abs() <= bound).all())


def grad_reference(grad, ids, rows, scale):
    there = (ids >= 0) & (ids < rows)
    at = ids[there].long()
    ref = torch.zeros((rows, grad.shape[1]), dtype=torch.float64, device="cuda")
    size, n = torch.zeros_like(ref), torch.zeros(rows, dtype=torch.float64, device="cuda")
    ref.index_add_(0, at, grad[there].double() * scale)
    size.index_add_(0, at, (grad[there].double() * scale).abs())
    n.index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    return ref, size, n


def check_grad(out, grad, ids, rows, scale):
    ref, size, n = grad_reference(grad, ids, rows, scale)
    bound = size * (n[:, None] + 2) * 2.0 ** -24 + ref.abs() * ROUND[out.dtype] * 1.01 + TINY[out.dtype]
    off = (out.double() - ref).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
    assert bool((out[n == 0] == 0).all())


@pytest.mark.parametrize("x", TYPES)
@pytest.mark.parametrize("o", TYPES)
@pytest.mark.parametrize("ids_type", [torch.int32, torch.int64])
def test_types(x, o, ids_type):
    say("types", x, o, ids_type)
    ids = some_ids(1500, 300, ids_type, 1)
    table, grad = rand((300, 72), x, 2), rand((1500, 72), x, 3)
    check_embed(trspmm.embed(table, ids, 1.7, o), table, ids, 1.7)
    check_grad(trspmm.embed_grad(grad, ids, 300, 1.7, o), grad, ids, 300, 1.7)


@pytest.mark.parametrize("width", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 64, 65, 100, 127, 250, 257, 511, 513, 1000, 1030, 2050])
@pytest.mark.parametrize("x", [torch.float16, torch.float32])
def test_widths(width, x):
    say("width", width, x)
    ids = some_ids(700, 90, torch.int64, width)
    table, grad = rand((90, width), x, 2), rand((700, width), x, 3)
    check_embed(trspmm.embed(table, ids, 0.5), table, ids, 0.5)
    check_grad(trspmm.embed_grad(grad, ids, 90, 0.5), grad, ids, 90, 0.5)


@pytest.mark.parametrize("count", [1, 2, 63, 64, 65, 255, 256, 257, 2047, 2048, 2049, 4097, 8191, 8192, 8193, 20_000, 70_001])
@pytest.mark.parametrize("rows", [1, 5, 1023, 2047, 2048, 65_536, 100_000])
def test_counts(count, rows):
    say("count", count, rows)
    ids = some_ids(count, rows, torch.int32, count + rows, skew=2)
    table, grad = rand((rows, 24), torch.float16, 2), rand((count, 24), torch.float16, 3)
    check_embed(trspmm.embed(table, ids), table, ids, 1.0)
    check_grad(trspmm.embed_grad(grad, ids, rows), grad, ids, rows, 1.0)


@pytest.mark.parametrize("rows", [4_194_303, 4_194_304, 5_000_001])
def test_three_digit_tables(rows):
    """Keys of 22, 23 and 23 bits: two and three sorting passes."""
    say("rows", rows)
    ids = some_ids(9000, rows, torch.int64, 5)
    ids[:3] = torch.tensor([rows - 1, 0, rows - 1], device="cuda")
    grad = rand((9000, 8), torch.float32, 3)
    check_grad(trspmm.embed_grad(grad, ids, rows), grad, ids, rows, 1.0)


@pytest.mark.parametrize("rows", [2000, 4_194_303, 4_194_304, 5_000_001])
@pytest.mark.parametrize("count", [20_000, 262_144, 262_145])
def test_sorted_tables(rows, count):
    """One to three sorting passes, with the blocks' counts added up where they are used (at most 64 blocks of 4096) and before."""
    say("sorted", rows, count)
    ids = some_ids(count, rows, torch.int64, 6, skew=2)
    ids[:3] = torch.tensor([rows - 1, 0, rows - 1], device="cuda")
    grad = rand((count, 8), torch.float32, 4)
    check_grad(trspmm.embed_grad(grad, ids, rows), grad, ids, rows, 1.0)


@pytest.mark.parametrize("count", [16_383, 16_384, 16_385])
@pytest.mark.parametrize("width", [3, 8, 120, 128, 129])
@pytest.mark.parametrize("rows", [1, 40, 3000, 300_000])
def test_most_ids_of_one_launch(count, width, rows):
    """Around the most ids and columns that one launch takes; few rows make each workgroup's list of ids long."""
    say("most", count, width, rows)
    grad = rand((count, width), torch.bfloat16, 1)
    for skew in (1, 4):
        ids = some_ids(count, rows, torch.int32, count + skew, skew=skew)
        check_grad(trspmm.embed_grad(grad, ids, rows, 0.25), grad, ids, rows, 0.25)


@pytest.mark.parametrize("found", [511, 512, 513, 1024, 1025, 2048, 2049, 4096, 5000, 8192, 8193])
def test_lists_of_one_workgroup(found):
    """Lists of ids around each size of the sort in LDS, all different runs and places: row 0's neighbours share its workgroup."""
    say("list", found)
    ids = torch.full((max(found, 9000),), -1, dtype=torch.int64, device="cuda")
    ids[:found] = torch.randint(0, 4, (found,), generator=gen(found), device="cuda")
    ids = ids[torch.randperm(ids.shape[0], generator=gen(1), device="cuda")]
    grad = rand((ids.shape[0], 16), torch.float16, 2)
    check_grad(trspmm.embed_grad(grad, ids, 10_000), grad, ids, 10_000, 1.0)
    assert torch.equal(trspmm.embed_grad(grad, ids, 10_000), trspmm.embed_grad(grad, ids, 10_000))


@pytest.mark.parametrize("count", [300, 5000, 300_001])
@pytest.mark.parametrize("width", [8, 128, 600])
def test_one_frequent_row(count, width):
    """Nearly all ids name one row; runs cross pieces, workgroups and, with width 600, column blocks."""
    say("frequent", count, width)
    ids = torch.full((count,), 7, dtype=torch.int32, device="cuda")
    ids[::97] = 3
    grad = rand((count, width), torch.float16, 1)
    out = trspmm.embed_grad(grad, ids, 20, 2.0)
    check_grad(out, grad, ids, 20, 2.0)
    ids.fill_(19)
    check_grad(trspmm.embed_grad(grad, ids, 20, 2.0), grad, ids, 20, 2.0)


def frequent_ids(count, rows, kind, dtype, seed):
    """Ids with frequent rows: all of one, half of one among spread ones, four and twelve rows with hardly any others, one row
    beside as many padded slots, one at the end of the call alone."""
    g = gen(seed)
    ids = torch.randint(0, rows, (count,), generator=g, device="cuda")
    coin = torch.rand(count, generator=g, device="cuda")
    few = torch.tensor([rows - 1, 0, rows // 2, rows // 3] if kind == "four" else [rows * k // 12 for k in range(12)], device="cuda")
    if kind == "all":
        ids[:] = rows - 1
    elif kind == "half":
        ids[coin < 0.5] = rows // 2
    elif kind in ("four", "twelve"):
        ids = torch.where(coin < 0.97, few[torch.randint(0, len(few), (count,), generator=g, device="cuda")], ids)
    elif kind == "padded":
        ids = torch.where(coin < 0.45, rows - 2, torch.where(coin < 0.9, -1, ids))
    else:
        ids[count - count // 3:] = 1
    return ids.to(dtype)


@pytest.mark.parametrize("kind", ["all", "half", "four", "twelve", "padded", "end"])
@pytest.mark.parametrize("count", [1024, 1025, 4099, 8192, 16_384])
@pytest.mark.parametrize("width", [1, 8, 13, 64, 100, 128, 300, 1030])
def test_frequent_rows_of_one_launch(kind, count, width):
    say("frequent", kind, count, width)
    if count > 8192 and width > 128:
        count = 8000
    dtype, out = TYPES[width % 3], TYPES[count % 3]
    for rows in (12, 5000):
        assert dense.embed_grad_workspace_bytes(count, rows, width) == 0
        ids = frequent_ids(count, rows, kind, torch.int32 if width % 2 else torch.int64, count + width)
        grad = rand((count, width + 3), dtype, 3)[:, 2:2 + width]
        got = trspmm.embed_grad(grad, ids, rows, 1.5, out)
        check_grad(got, grad, ids, rows, 1.5)
        assert torch.equal(got, trspmm.embed_grad(grad, ids, rows, 1.5, out))
        buf = torch.full((rows, width + 5), 9.0, dtype=out, device="cuda")
        assert torch.equal(trspmm.embed_grad(grad, ids, rows, 1.5, out=buf[:, 3:3 + width]), got)
        assert bool((buf[:, :3] == 9).all()) and bool((buf[:, 3 + width:] == 9).all())


@pytest.mark.parametrize("count,width,most", [(16_384, 64, 7), (8192, 1024, 4)])
def test_a_frequent_row_costs_little_more(count, width, most):
    """All ids naming one row against ids spread evenly: 3.9 and 1.6 times when this was written, 13.6 and 15 where one workgroup
    sorted and summed them alone."""
    say("frequent row's time", count, width)
    grad, times = rand((count, width), torch.float16, 1), []
    for ids in (torch.randint(0, 16_384, (count,), generator=gen(2), device="cuda"), torch.full((count,), 5, device="cuda")):
        out, best = torch.empty((16_384, width), device="cuda"), float("inf")
        for _ in range(6):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(30):
                trspmm.embed_grad(grad, ids, 16_384, out=out)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end))
        times.append(best)
    assert times[1] < most * times[0], times


def test_runs_at_every_boundary():
    """Run lengths around the sums' pieces (16) and workgroups (16 x 16 ids at this width)."""
    lengths = [1, 15, 16, 17, 1, 1, 14, 255, 256, 257, 2, 1000, 16, 16, 240, 31, 33, 512, 3]
    say("runs", sum(lengths))
    ids = torch.cat([torch.full((n,), 2 * i, device="cuda") for i, n in enumerate(lengths)] +
                    [torch.full((5,), -1, device="cuda")])
    ids = ids[torch.randperm(ids.shape[0], generator=gen(1), device="cuda")].repeat(4)
    grad = rand((ids.shape[0], 128), torch.float32, 1)
    check_grad(trspmm.embed_grad(grad, ids, 2 * len(lengths)), grad, ids, 2 * len(lengths), 1.0)


def sorts(count, rows, width):
    """That a call of this size sorts its ids, and does not run in one launch."""
    assert dense.embed_grad_workspace_bytes(count, rows, width) > 0


@pytest.mark.parametrize("x", TYPES)
@pytest.mark.parametrize("o", TYPES)
@pytest.mark.parametrize("ids_type", [torch.int32, torch.int64])
def test_types_of_sorted_ids(x, o, ids_type):
    say("sorted types", x, o, ids_type)
    sorts(17_003, 300, 72)
    ids, grad = some_ids(17_003, 300, ids_type, 1), rand((17_003, 72), x, 3)
    check_grad(trspmm.embed_grad(grad, ids, 300, 1.7, o), grad, ids, 300, 1.7)


@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 6, 7, 8, 9, 11, 12, 13, 15, 16, 17, 31, 33, 64, 65, 100, 127, 129, 250, 257, 511, 512, 513,
                                   520, 1000, 1023, 1030, 2050])
@pytest.mark.parametrize("x", [torch.float16, torch.float32])
def test_widths_of_sorted_ids(width, x):
    """Each size of a group of lanes, whole and cut last chunks, one and several blocks of columns."""
    say("sorted width", width, x)
    for rows in (90, 9001):
        sorts(17_003, rows, width)
        ids, grad = some_ids(17_003, rows, torch.int64, width, skew=2), rand((17_003, width), x, 3)
        check_grad(trspmm.embed_grad(grad, ids, rows, 0.5), grad, ids, rows, 0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [3, 13, 43, 517])
def test_strides_of_sorted_ids(dtype, width):
    say("sorted strides", dtype, width)
    wide, rows, count = width + 18, 700, 17_003
    sorts(count, rows, width)
    ids = some_ids(2 * count, rows, torch.int64, 4)[::2]
    grad = rand((count, wide), dtype, 2)[:, 5:5 + width]
    buf = torch.full((rows, wide), 9.0, dtype=dtype, device="cuda")
    out = trspmm.embed_grad(grad, ids, rows, 1.5, out=buf[:, 7:7 + width])
    check_grad(out, grad, ids, rows, 1.5)
    assert bool((buf[:, :7] == 9).all()) and bool((buf[:, 7 + width:] == 9).all())
    g = rand((1, width), dtype, 6).expand(count, width)                    # a broadcast gradient
    check_grad(trspmm.embed_grad(g, ids, rows, 1.5), g, ids, rows, 1.5)


@pytest.mark.parametrize("width", [4, 8, 16, 24, 50, 128, 200, 512, 600, 1030])
def test_sorted_runs_at_every_boundary(width):
    """Runs that end just before, at and just after the 16 ids of a piece and the ids of a workgroup (a piece for each of its
    groups of lanes), and runs over several workgroups, each begun at such a place."""
    lanes = 1
    while lanes < 64 and lanes * 8 < width:
        lanes *= 2
    piece, block = 16, 256 // lanes * 16
    lengths = []
    for unit in (piece, block, 2 * block, 3 * block):
        for off in (-1, 0, 1, 7):
            lengths += [unit + off, unit - off] if off else [unit, 1, unit - 1]   # the next one starts on a boundary again
    lengths += [1, 15, 1, block - 17, 1, block, block, 2, block - 2, piece, block - piece]
    while sum(lengths) <= 16_400:
        lengths += [1, 15, 16, 17, 5, 2 * block + 3, block - 1]
    say("sorted runs", width, sum(lengths))
    rows = 2 * len(lengths)
    sorts(sum(lengths), rows, width)
    ids = torch.cat([torch.full((n,), 2 * i, device="cuda") for i, n in enumerate(lengths)] + [torch.full((5,), -1, device="cuda")])
    for seed in (0, 1):                                                    # in their order, and not
        if seed:
            ids = ids[torch.randperm(ids.shape[0], generator=gen(seed), device="cuda")]
        grad = rand((ids.shape[0], width), torch.float32, 1)
        check_grad(trspmm.embed_grad(grad, ids, rows), grad, ids, rows, 1.0)


def test_ids_outside_the_table():
    say("outside")
    ids = torch.tensor([0, -1, 4, 5, 2 ** 31, 2 ** 32 + 1, -2 ** 40, 3], device="cuda")
    table, grad = rand((5, 40), torch.float32, 1), rand((8, 40), torch.float32, 2)
    check_embed(trspmm.embed(table, ids, 3.0), table, ids, 3.0)
    check_grad(trspmm.embed_grad(grad, ids, 5, 3.0), grad, ids, 5, 3.0)
    none = torch.full((4000,), -1, device="cuda")
    assert not trspmm.embed(table, none).any()
    assert not trspmm.embed_grad(rand((4000, 40), torch.float32, 2), none, 5).any()


def test_no_ids_no_rows_no_width():
    say("empty")
    empty = torch.empty(0, dtype=torch.int64, device="cuda")
    table = rand((5, 40), torch.float16, 1)
    assert trspmm.embed(table, empty).shape == (0, 40)
    out = torch.full((5, 40), 7.0, device="cuda")
    assert not trspmm.embed_grad(table[:0], empty, 5, out=out).any()      # every row is written
    ids = torch.tensor([0, 1], device="cuda")
    assert not trspmm.embed(table[:0], ids).any()                          # a table without rows
    assert trspmm.embed_grad(table[:2], ids, 0).shape == (0, 40)
    assert trspmm.embed(table[:, :0], ids).shape == (2, 0)
    assert trspmm.embed_grad(table[:2, :0], ids, 5).shape == (5, 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_offsets(dtype):
    """Operands and outputs inside wider buffers, at odd element offsets; what lies around is untouched."""
    say("strides", dtype)
    wide, rows, count, width = 61, 50, 3000, 43
    ids = some_ids(2 * count, rows, torch.int64, 4)[::2]
    table = rand((rows, wide), dtype, 1)[:, 3:3 + width]
    grad = rand((count, wide), dtype, 2)[:, 5:5 + width]
    buf = torch.full((count, wide), 9.0, dtype=dtype, device="cuda")
    out = trspmm.embed(table, ids, 1.5, out=buf[:, 1:1 + width])
    check_embed(out, table, ids, 1.5)
    assert bool((buf[:, 0] == 9).all()) and bool((buf[:, 1 + width:] == 9).all())
    buf = torch.full((rows, wide), 9.0, dtype=dtype, device="cuda")
    out = trspmm.embed_grad(grad, ids, rows, 1.5, out=buf[:, 7:7 + width])
    check_grad(out, grad, ids, rows, 1.5)
    assert bool((buf[:, :7] == 9).all()) and bool((buf[:, 7 + width:] == 9).all())
    t = rand((width, rows), dtype, 6).t()                                  # columns apart: copied
    check_embed(trspmm.embed(t, ids, 1.5), t, ids, 1.5)
    g = rand((1, width), dtype, 6).expand(count, width)                    # a broadcast gradient
    check_grad(trspmm.embed_grad(g, ids, rows, 1.5), g, ids, rows, 1.5)


def test_offsets_past_32_bits():
    """Row offsets beyond 2^32 elements on either side."""
    say("far rows")
    far = torch.empty((300, 1 << 24), dtype=torch.float16, device="cuda")[:, 11:59]
    far.copy_(rand((300, 48), torch.float16, 1))
    ids = some_ids(300, 300, torch.int32, 2, pad=0.0)
    check_embed(trspmm.embed(far, ids), far, ids, 1.0)
    check_grad(trspmm.embed_grad(far, ids, 300), far, ids, 300, 1.0)
    table = far.contiguous()
    trspmm.embed(table, ids, out=far)
    check_embed(far, table, ids, 1.0)
    trspmm.embed_grad(table, ids, 300, out=far)
    check_grad(far, table, ids, 300, 1.0)


def test_not_finite_values_stay_in_their_rows():
    say("not finite")
    ids = torch.tensor([0, 1, 2, 1, 3], device="cuda").repeat(40)
    grad = rand((200, 33), torch.float32, 1)
    grad[2, 5], grad[3, 7] = float("nan"), float("inf")
    out = trspmm.embed_grad(grad, ids, 6)
    finite = torch.isfinite(out)
    want = torch.ones_like(finite)
    want[2, 5] = want[1, 7] = False
    assert torch.equal(finite, want)
    assert bool((trspmm.embed(grad, torch.tensor([1, 0], device="cuda")) == grad[[1, 0]]).all())


def test_same_bits_every_time():
    """A fixed order of the sums, whatever the timing; another stream gives them too."""
    say("same bits")
    ids = some_ids(60_000, 3000, torch.int32, 1, skew=3)
    grad = rand((60_000, 96), torch.float16, 2)
    first = trspmm.embed_grad(grad, ids, 3000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        assert torch.equal(trspmm.embed_grad(grad, ids, 3000), first)
        other = trspmm.embed_grad(grad, ids, 3000, stream=s)
        s.synchronize()
        assert torch.equal(other, first)


@pytest.mark.parametrize("count", [500, 30_000])
def test_graph_replays(count):
    say("graph", count)
    ids, grad, table = some_ids(count, 999, torch.int64, 1), rand((count, 64), torch.float16, 2), rand((999, 64), torch.float16, 3)
    out, back = torch.empty((count, 64), dtype=torch.float16, device="cuda"), torch.empty((999, 64), device="cuda")
    ws = torch.empty(max(1, dense.embed_grad_workspace_bytes(count, 999, 64)), dtype=torch.uint8, device="cuda")

    def both():
        trspmm.embed(table, ids, 2.0, out=out)
        trspmm.embed_grad(grad, ids, 999, 2.0, out=back, workspace=ws)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for i in range(4):
        ids.copy_(some_ids(count, 999, torch.int64, 10 + i))
        out.fill_(float("nan"))
        back.fill_(float("nan"))
        ws.fill_(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, trspmm.embed(table, ids, 2.0)), f"replay {i}"
        assert torch.equal(back, trspmm.embed_grad(grad, ids, 999, 2.0)), f"replay {i}"


@pytest.mark.parametrize("o", TYPES)
def test_large_outputs(o):
    """Outputs of more than 16 MB, which leave past the caches where their rows allow it."""
    say("large", o)
    for width in (128, 132, 131):
        ids = some_ids(70_001, 90_000, torch.int32, 3, skew=2)
        table, grad = rand((90_000, width), torch.float16, 2), rand((70_001, width), torch.float16, 3)
        check_embed(trspmm.embed(table, ids, 0.7, o), table, ids, 0.7)
        check_grad(trspmm.embed_grad(grad, ids, 90_000, 0.7, o), grad, ids, 90_000, 0.7)
        check_grad(trspmm.embed_grad(grad[:900], ids[:900], 90_000, 0.7, o), grad[:900], ids[:900], 90_000, 0.7)


@pytest.mark.parametrize("off", [0, 1, 4, 8])
def test_workspaces_at_any_address(off):
    """One off the 8-byte boundary is left alone, and another used in its place."""
    say("workspace", off)
    ids, grad = some_ids(20_000, 700, torch.int64, 1), rand((20_000, 24), torch.float16, 2)
    need = dense.embed_grad_workspace_bytes(20_000, 700, 24)
    ws = torch.full((need + 16,), 171, dtype=torch.uint8, device="cuda")
    out = trspmm.embed_grad(grad, ids, 700, workspace=ws[off:off + need])
    check_grad(out, grad, ids, 700, 1.0)
    assert bool((ws == 171).all()) == (off % 8 != 0)


def test_gradient_against_differences():
    """The lookup is linear in the table: <embed(table + v) - embed(table), g> = <embed_grad(g), v>."""
    say("differences")
    ids = some_ids(2500, 60, torch.int64, 1, skew=2)
    table, v, g = (rand(s, torch.float32, k) for k, s in enumerate([(60, 50), (60, 50), (2500, 50)]))
    left = ((trspmm.embed(table + v, ids, 1.25).double() - trspmm.embed(table, ids, 1.25).double()) * g.double()).sum()
    terms = trspmm.embed_grad(g, ids, 60, 1.25).double() * v.double()
    # each of 125,000 differences of values below 16 is off by 2^-20 at most, times |g| below 6, at random
    assert abs(float(left - terms.sum())) <= 6 * 2.0 ** -20 * 6 * 125_000 ** 0.5
    assert float(terms.abs().sum()) > 1000


def refused(code, fn, *args, **kw):
    with pytest.raises(nat.TrsError) as e:
        fn(*args, **kw)
    assert e.value.code == code


def test_refusals():
    say("refusals")
    table, ids = rand((5, 16), torch.float16, 1), torch.tensor([0, 1], device="cuda")
    bad = [dict(table=table.cpu()), dict(table=table.double()), dict(table=table[0]), dict(ids=ids.cpu()),
           dict(ids=ids.float()), dict(ids=ids[None]), dict(dtype=torch.int8),
           dict(out=torch.empty((3, 16), dtype=torch.float16, device="cuda")),
           dict(out=torch.empty((2, 32), dtype=torch.float16, device="cuda")[:, ::2])]
    for kw in bad:
        with pytest.raises(ValueError):
            trspmm.embed(**{"table": table, "ids": ids, **kw})
    grad = rand((2, 16), torch.float16, 1)
    for kw in [dict(grad=grad[:1]), dict(rows=-1), dict(grad=grad.double()), dict(workspace=torch.empty(1 << 20, dtype=torch.uint8))]:
        with pytest.raises(ValueError):
            trspmm.embed_grad(**{"grad": grad, "ids": ids, "rows": 5, **kw})
    refused(1, trspmm.embed, table, ids, float("inf"))
    refused(1, trspmm.embed_grad, grad, ids, 5, float("nan"))
    lib, out = nat.lib(), torch.empty((5, 16), device="cuda")
    args = lambda ws, n: (grad.data_ptr(), 1, 16, ids.data_ptr(), 64, 2, 5, 16, 1.0, out.data_ptr(), 0, 16, ws, n, None)  # noqa: E731
    assert lib.trs_embed_grad_workspace_bytes(2, 5, 16) >= 0
    for k, v in [(4, 16), (1, 3), (10, 3), (2, 15), (11, 15), (5, -1), (6, -1), (7, -1), (0, None), (9, None), (3, None)]:
        call = list(args(0, 0))
        call[k] = v
        assert lib.trs_embed_grad(*call) == 1, k
    call = list(args(0, 0))
    call[6] = 2 ** 31
    assert lib.trs_embed_grad(*call) == 5
    need = lib.trs_embed_grad_workspace_bytes(100_000, 5, 16)
    call = list(args(out.data_ptr(), need - 1))
    call[5] = 100_000                                       # refused before anything is read
    assert need > 0 and lib.trs_embed_grad(*call) == 1
