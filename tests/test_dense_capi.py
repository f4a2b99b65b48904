"""The dense operators' C entry points without a GPU: every wrong argument is refused with its status and a
message before anything is launched or read, sizes of workspaces, and calls that have nothing to do."""
import numpy as np
import pytest

import trspmm._native as nat

X = np.zeros(4096, np.float32).ctypes.data      # an address that no refused call reads
INF, NAN = float("inf"), float("nan")

EMBED = dict(table=X, table_type=0, ldt=16, rows=5, ids=X, id_bits=64, count=3, width=16, scale=1.0, out=X, out_type=0,
             ldo=16, stream=None)
EMBED_GRAD = dict(grad=X, grad_type=0, ldg=16, ids=X, id_bits=64, count=3, rows=5, width=16, scale=1.0, out=X, out_type=0,
                  ldo=16, ws=None, ws_bytes=0, stream=None)
NORM = dict(x=X, x_type=0, ldx=16, res=X, r_type=0, ldr=16, weight=X, w_type=0, eps=1e-5, rows=3, width=16, y=X, y_type=0,
            ldy=16, r_out=X, ldro=16, stream=None)
NORM_I8 = dict(x=X, x_type=0, ldx=16, res=X, r_type=0, ldr=16, weight=X, w_type=0, eps=1e-5, rows=3, width=16, q=X, ldq=16,
               scale=X, r_out=X, ldro=16, stream=None)
NORM_GRAD = dict(grad=X, grad_type=0, ldg=16, r=X, r_type=0, ldr=16, weight=X, w_type=0, grad_r=None, ldgr=0, eps=1e-5, rows=3,
                 width=16, dr=X + 1024, lddr=16, dweight=X, ws=X, ws_bytes=1 << 20, stream=None)
MATMUL = dict(a=X, lda=16, a_scale=X, w=X, ldw=16, w_scale=X, bias=None, m=3, n=4, k=16, out=X, out_type=0, ldo=4, stream=None)

COMMON = [("width", -1, 1), ("rows", -1, 1)]
BAD = {
    "trs_embed": (EMBED, [*COMMON, ("count", -1, 1), ("table_type", 3, 1), ("out_type", -1, 1), ("id_bits", 16, 1), ("ids", None, 1),
                          ("table", None, 1), ("out", None, 1), ("ldt", 15, 1), ("ldo", 15, 1), ("scale", INF, 1), ("scale", NAN, 1),
                          ("count", 1 << 50, 5)]),
    "trs_embed_grad": (EMBED_GRAD, [*COMMON, ("count", -1, 1), ("grad_type", 3, 1), ("out_type", 9, 1), ("id_bits", 8, 1), ("ids", None, 1),
                                    ("grad", None, 1), ("out", None, 1), ("ldg", 15, 1), ("ldo", 15, 1), ("scale", -INF, 1),
                                    ("count", 2 ** 31 - 1, 5), ("rows", 2 ** 31 - 1, 5), ("count", 100_000, 1)]),
    "trs_rms_norm": (NORM, [*COMMON, ("x_type", 3, 1), ("r_type", 3, 1), ("w_type", -1, 1), ("y_type", 3, 1), ("eps", 0.0, 1), ("eps", -1.0, 1),
                            ("eps", NAN, 1), ("eps", INF, 1), ("x", None, 1), ("weight", None, 1), ("y", None, 1), ("r_out", None, 1),
                            ("res", None, 1), ("ldx", 15, 1), ("ldr", 15, 1), ("ldy", 15, 1), ("ldro", 15, 1), ("rows", 1 << 40, 5)]),
    "trs_rms_norm_i8": (NORM_I8, [*COMMON, ("x_type", 3, 1), ("w_type", 3, 1), ("eps", NAN, 1), ("q", None, 1), ("scale", None, 1), ("ldq", 15, 1),
                                  ("r_out", None, 1), ("rows", 1 << 40, 5)]),
    "trs_rms_norm_grad": (NORM_GRAD, [*COMMON, ("grad_type", 3, 1), ("r_type", 3, 1), ("w_type", 3, 1), ("eps", 0.0, 1), ("grad", None, 1),
                                      ("r", None, 1), ("weight", None, 1), ("dr", None, 1), ("dweight", None, 1), ("ldg", 15, 1), ("ldr", 15, 1),
                                      ("lddr", 15, 1), ("grad_r", X + 2048, 1), ("ws", None, 1), ("ws_bytes", 1, 1), ("dr", X, 1),
                                      ("rows", 1 << 40, 5)]),
    "trs_matmul_i8": (MATMUL, [("m", -1, 1), ("n", -1, 1), ("k", -1, 1), ("out_type", 3, 1), ("a", None, 1), ("w", None, 1), ("a_scale", None, 1),
                               ("w_scale", None, 1), ("out", None, 1), ("lda", 15, 1), ("ldw", 15, 1), ("ldo", 3, 1), ("k", 131_072, 5),
                               ("m", 1 << 50, 5)]),
}


REFUSED = [(n, *b) for n, (_, bad) in BAD.items() for b in bad]


# named by their place in the list: an address is another in each process
@pytest.mark.parametrize("name,arg,value,status", REFUSED, ids=[f"{n}-{arg}-{i}" for i, (n, arg, _, _) in enumerate(REFUSED)])
def test_refused(name, arg, value, status):
    lib = nat.lib()
    rc = getattr(lib, name)(*{**BAD[name][0], arg: value}.values())
    assert rc == status, lib.trs_last_error()
    assert lib.trs_last_error().startswith(name.encode() + b": ")


@pytest.mark.parametrize("m,n", [(1 << 62, 2 ** 31 - 1), (64, 2 ** 31 - 1), (1, 2 ** 27 + 1)])
def test_products_past_a_launch_are_refused(m, n):
    lib = nat.lib()
    assert lib.trs_matmul_i8(*{**MATMUL, "m": m, "n": n, "ldo": n}.values()) == 5, lib.trs_last_error()


@pytest.mark.parametrize("first,second", [(1, 2), (2, 1)])
def test_two_different_16_bit_types_are_refused(first, second):
    lib = nat.lib()
    assert lib.trs_rms_norm(*{**NORM, "x_type": first, "r_type": second}.values()) == 1
    assert lib.trs_rms_norm_i8(*{**NORM_I8, "x_type": first, "r_type": second}.values()) == 1
    assert lib.trs_rms_norm_grad(*{**NORM_GRAD, "grad_type": first, "r_type": second}.values()) == 1


def test_nothing_to_do_is_no_error():
    lib = nat.lib()
    for name, args in [("trs_embed", {**EMBED, "count": 0, "out": None}), ("trs_embed", {**EMBED, "width": 0}),
                       ("trs_embed_grad", {**EMBED_GRAD, "rows": 0}), ("trs_embed_grad", {**EMBED_GRAD, "width": 0}),
                       ("trs_rms_norm", {**NORM, "rows": 0, "x": None, "y": None}), ("trs_rms_norm_i8", {**NORM_I8, "width": 0}),
                       ("trs_rms_norm_grad", {**NORM_GRAD, "width": 0}), ("trs_matmul_i8", {**MATMUL, "m": 0, "out": None}),
                       ("trs_matmul_i8", {**MATMUL, "n": 0})]:
        assert getattr(lib, name)(*args.values()) == 0, name


def test_workspace_sizes():
    lib = nat.lib()
    grad, norm = lib.trs_embed_grad_workspace_bytes, lib.trs_rms_norm_grad_workspace_bytes
    assert grad(0, 5, 8) == grad(5, 0, 8) == grad(5, 5, 0) == grad(2 ** 31, 5, 8) == 0
    assert grad(8192, 1 << 20, 128) == 0                        # few ids: no workspace
    big = grad(1_000_000, 1 << 20, 128)
    assert 16_000_000 <= big < 64_000_000                       # two copies of the ids and places, parts, counts
    assert grad(2_000_000, 1 << 20, 128) > big
    assert grad(8192, 2 ** 30, 8) > 0                           # more rows than a few workgroups' marks hold
    assert norm(0, 8) == norm(8, 0) == 0
    assert norm(10_000, 4096) >= 256 * 4096 * 4
    assert norm(10, 10_000) >= 10 * 10_000 * 4 + 10 * 8         # long rows keep two numbers a row


WIDEST, FAR = 2 ** 31 - 65536, 1 << 31   # the most columns whose indexes, a step past the last among them, are 32-bit integers


@pytest.mark.parametrize("width", [WIDEST + 1, 2 ** 31 - 2048, 2 ** 31 - 7, 2 ** 31 - 1])
def test_columns_past_32_bit_indexes_are_refused(width):
    lib = nat.lib()
    for count in (3, 100_000):      # the one launch's sums and the sorted ones
        for name, args in [("trs_embed", {**EMBED, "ldt": FAR, "ldo": FAR}), ("trs_embed_grad", {**EMBED_GRAD, "ldg": FAR, "ldo": FAR})]:
            assert getattr(lib, name)(*{**args, "width": width, "count": count}.values()) == 5, (name, lib.trs_last_error())
    for name, args in [("trs_rms_norm", {**NORM, "ldx": FAR, "ldr": FAR, "ldy": FAR, "ldro": FAR}),
                       ("trs_rms_norm_i8", {**NORM_I8, "ldx": FAR, "ldr": FAR, "ldq": FAR, "ldro": FAR})]:
        assert getattr(lib, name)(*{**args, "width": width}.values()) == 5, (name, lib.trs_last_error())


@pytest.mark.parametrize("width", [65535 * 2048 + 1, WIDEST, 2 ** 31 - 1])
@pytest.mark.parametrize("rows", [0, 3])
def test_gradients_of_more_columns_than_a_grid_are_refused(width, rows):
    """Before the first of its launches, and where there are no rows and dweight alone is written."""
    lib = nat.lib()
    args = {**NORM_GRAD, "ldg": FAR, "ldr": FAR, "lddr": FAR, "width": width, "rows": rows, "ws_bytes": 1 << 60}
    assert lib.trs_rms_norm_grad(*args.values()) == 5, lib.trs_last_error()


@pytest.mark.parametrize("off", [1, 2, 4, 7])
def test_workspaces_off_8_byte_boundaries_are_refused(off):
    lib = nat.lib()
    assert X % 8 == 0
    args = {**EMBED_GRAD, "count": 100_000, "ws": X + off, "ws_bytes": 1 << 40}
    assert lib.trs_embed_grad(*args.values()) == 1, lib.trs_last_error()
    assert lib.trs_rms_norm_grad(*{**NORM_GRAD, "ws": X + off}.values()) == 1, lib.trs_last_error()
