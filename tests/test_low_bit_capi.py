"""The C entry points of 4-bit codes and of the AdamW step without a GPU: wrong arguments are refused with their status and a
message before anything is launched or read, and calls that have nothing to do succeed."""
import ctypes

import numpy as np
import pytest

import trspmm._native as nat

_buf = np.zeros(8192, np.float32)
X = (_buf.ctypes.data + 63) // 64 * 64      # an address that no refused call reads
INF, NAN = float("inf"), float("nan")
FAR = 1 << 31

QUANT = dict(x=X, x_type=0, ldx=40, rows=3, width=40, codes=X, ldc=32, scale=X, lds=2, stream=None)
DEQUANT = dict(codes=X, ldc=32, scale=X, lds=2, rows=3, width=40, out=X, out_type=0, ldo=40, stream=None)
NORM = dict(x=X, x_type=0, ldx=40, res=X, r_type=0, ldr=40, weight=X, w_type=0, eps=1e-5, rows=3, width=40, codes=X, ldc=32, scale=X, lds=2,
            r_out=X, ldro=40, stream=None)
MATMUL = dict(a=X, lda=32, a_scale=X, ldas=2, w=X, ldw=32, w_scale=X, ldws=2, bias=None, m=3, n=4, blocks=2, out=X, out_type=0, ldo=4,
              stream=None)
BAD = {
    "trs_quant_mx4": (QUANT, [("rows", -1, 1), ("width", -1, 1), ("x_type", 3, 1), ("x", None, 1), ("codes", None, 1), ("scale", None, 1),
                              ("ldx", 39, 1), ("ldc", 16, 1), ("ldc", 40, 1), ("codes", X + 8, 1), ("lds", 1, 1), ("rows", 1 << 40, 5)]),
    "trs_dequant_mx4": (DEQUANT, [("rows", -1, 1), ("width", -1, 1), ("out_type", -1, 1), ("out", None, 1), ("codes", None, 1), ("scale", None, 1),
                                  ("ldo", 39, 1), ("ldc", 16, 1), ("ldc", 33, 1), ("codes", X + 1, 1), ("lds", 1, 1), ("rows", 1 << 40, 5)]),
    "trs_rms_norm_mx4": (NORM, [("rows", -1, 1), ("width", -1, 1), ("x_type", 3, 1), ("r_type", 3, 1), ("w_type", -1, 1), ("eps", 0.0, 1), ("eps", NAN, 1),
                                ("eps", INF, 1), ("x", None, 1), ("weight", None, 1), ("codes", None, 1), ("scale", None, 1), ("r_out", None, 1),
                                ("res", None, 1), ("ldx", 39, 1), ("ldr", 39, 1), ("ldro", 39, 1), ("ldc", 16, 1), ("ldc", 36, 1),
                                ("codes", X + 4, 1), ("lds", 1, 1), ("rows", 1 << 40, 5)]),
    "trs_matmul_mx4": (MATMUL, [("m", -1, 1), ("n", -1, 1), ("blocks", -1, 1), ("out_type", 3, 1), ("a", None, 1), ("w", None, 1), ("a_scale", None, 1),
                                ("w_scale", None, 1), ("out", None, 1), ("lda", 16, 1), ("ldw", 16, 1), ("lda", 40, 1), ("ldw", 33, 1), ("a", X + 8, 1),
                                ("w", X + 1, 1), ("ldas", 1, 1), ("ldws", 1, 1), ("ldo", 3, 1), ("blocks", (1 << 26) + 1, 5), ("m", 1 << 50, 5)]),
}
REFUSED = [(n, *b) for n, (_, bad) in BAD.items() for b in bad]


@pytest.mark.parametrize("name,arg,value,status", REFUSED, ids=[f"{n}-{arg}-{i}" for i, (n, arg, _, _) in enumerate(REFUSED)])
def test_refused(name, arg, value, status):
    lib = nat.lib()
    rc = getattr(lib, name)(*{**BAD[name][0], arg: value}.values())
    assert rc == status, lib.trs_last_error()
    assert lib.trs_last_error().startswith(name.encode() + b": ")


@pytest.mark.parametrize("width", [65535 * 2048 + 1, 2 ** 31 - 65535, 2 ** 31 - 1])
def test_columns_past_the_grid_or_32_bits_are_refused(width):
    lib = nat.lib()
    wide = {"width": width, "ldc": FAR, "lds": FAR}
    assert lib.trs_quant_mx4(*{**QUANT, **wide, "ldx": FAR}.values()) == 5
    assert lib.trs_dequant_mx4(*{**DEQUANT, **wide, "ldo": FAR}.values()) == 5
    if width > 2 ** 31 - 65536:
        assert lib.trs_rms_norm_mx4(*{**NORM, **wide, "ldx": FAR, "ldr": FAR, "ldro": FAR}.values()) == 5


@pytest.mark.parametrize("m,n", [(1 << 41, 2 ** 31 - 1), (1 << 62, 2 ** 31 - 1), (1 << 40, 1), (64, 2 ** 31 - 1), (1 << 36, 64), (1, 2 ** 31 - 65535)])
def test_products_past_a_launch_are_refused(m, n):
    lib = nat.lib()
    assert lib.trs_matmul_mx4(*{**MATMUL, "m": m, "n": n, "ldo": n}.values()) == 5, lib.trs_last_error()


@pytest.mark.parametrize("first,second", [(1, 2), (2, 1)])
def test_two_different_16_bit_types_are_refused(first, second):
    assert nat.lib().trs_rms_norm_mx4(*{**NORM, "x_type": first, "r_type": second}.values()) == 1


def test_nothing_to_do_is_no_error():
    lib = nat.lib()
    for name, args in [("trs_quant_mx4", {**QUANT, "rows": 0, "x": None}), ("trs_quant_mx4", {**QUANT, "width": 0}),
                       ("trs_dequant_mx4", {**DEQUANT, "rows": 0}), ("trs_dequant_mx4", {**DEQUANT, "width": 0, "out": None}),
                       ("trs_rms_norm_mx4", {**NORM, "rows": 0}), ("trs_rms_norm_mx4", {**NORM, "width": 0}),
                       ("trs_matmul_mx4", {**MATMUL, "m": 0, "out": None}), ("trs_matmul_mx4", {**MATMUL, "n": 0})]:
        assert getattr(lib, name)(*args.values()) == 0, name


def options(**more):
    o = nat.AdamwOptions()
    nat.lib().trs_adamw_options_default(o)
    for k, v in more.items():
        setattr(o, k, v)
    return o


def tensor(**more):
    t = nat.AdamwTensor(param=X, grad=X + 256, m=X + 512, v=X + 1024, count=10, weight_decay=0.1)
    for k, v in more.items():
        setattr(t, k, v)
    return t


def adamw(tensors, o, count=None):
    lib = nat.lib()
    return lib.trs_adamw((nat.AdamwTensor * max(1, len(tensors)))(*tensors), len(tensors) if count is None else count, o, None)


def test_adamw_defaults():
    o = options()
    assert o.struct_size == ctypes.sizeof(nat.AdamwOptions) and o.tensor_size == ctypes.sizeof(nat.AdamwTensor)
    assert (o.lr, o.beta1, o.beta2, o.eps, o.grad_scale, o.step) == (1e-3, 0.9, 0.999, 1e-8, 1.0, 1)


@pytest.mark.parametrize("field,value", [("struct_size", 0), ("struct_size", 88), ("tensor_size", 72), ("beta1", 1.0), ("beta1", -0.1), ("beta2", NAN),
                                         ("beta2", 1.5), ("eps", 0.0), ("eps", -1.0), ("eps", INF), ("eps", 1e-60), ("lr", NAN), ("lr", 1e300),
                                         ("grad_scale", INF), ("step", 0), ("step", -5)])
def test_adamw_options_refused(field, value):
    assert adamw([tensor()], options(**{field: value})) == 1
    assert nat.lib().trs_last_error().startswith(b"trs_adamw: ")


@pytest.mark.parametrize("field,value,status", [("param", None, 1), ("grad", None, 1), ("m", None, 1), ("v", None, 1), ("count", -1, 1), ("param_type", 3, 1),
                                                ("grad_type", -1, 1), ("m_scale", X + 2048, 1), ("v_scale", X + 2048, 1), ("weight_decay", NAN, 1),
                                                ("count", 1 << 50, 5)])
def test_adamw_tensors_refused(field, value, status):
    assert adamw([tensor(), tensor(**{field: value})], options()) == status
    assert nat.lib().trs_last_error().startswith(b"trs_adamw: ")


def test_adamw_overlaps_refused():
    far = dict(param=X + 4096, m=X + 8192, v=X + 12288)
    for tensors in ([tensor(), tensor()], [tensor(), tensor(**{**far, "param": X + 36})], [tensor(m=X + 36)], [tensor(v=X)],
                    [tensor(copy=X + 39)], [tensor(m_scale=X + 513, v_scale=X + 4096)], [tensor(m_scale=X + 4096, v_scale=X + 4096)],
                    [tensor(), tensor(**{**far, "m": X + 1063})], [tensor(grad=X + 36)], [tensor(grad=X + 1063)], [tensor(copy=X + 295)],
                    [tensor(), tensor(**far, grad=X + 4000, count=100)]):
        assert adamw(tensors, options()) == 1
        assert b"overlaps" in nat.lib().trs_last_error()
    many = [tensor(param=X + 100_000 * i, m=X + 100_000 * i + 400, v=X + 100_000 * i + 800) for i in range(400)]
    many[399].v = many[7].m + 4
    assert adamw(many, options()) == 1 and b"overlaps" in nat.lib().trs_last_error()
    many[399].v, many[5].grad = many[398].v + 100_000, many[300].m + 39
    assert adamw(many, options()) == 1 and b"overlaps" in nat.lib().trs_last_error()


def test_adamw_of_nothing():
    assert adamw([], options()) == 0
    assert adamw([tensor(count=0, param=None, grad=None)] * 3, options()) == 0
    lib = nat.lib()
    assert lib.trs_adamw(None, 1, options(), None) == 1 and lib.trs_adamw(None, 0, options(), None) == 0
    assert lib.trs_adamw(None, 0, None, None) == 1 and adamw([tensor()], options(), count=-1) == 1


def test_a_single_rows_distance_says_nothing():
    """One row on a 16-byte boundary is taken whatever the next would be at: these calls are refused for what is checked behind it."""
    lib = nat.lib()
    assert lib.trs_rms_norm_mx4(*{**NORM, "rows": 1, "ldc": 33, "x_type": 1, "r_type": 2}.values()) == 1
    assert b"16-bit types" in lib.trs_last_error()
    assert lib.trs_matmul_mx4(*{**MATMUL, "m": 1 << 40, "n": 1, "ldw": 33, "ldo": 1}.values()) == 5
    for name, args in [("trs_quant_mx4", {**QUANT, "rows": 1, "codes": X + 8}), ("trs_quant_mx4", {**QUANT, "rows": 1, "ldc": 31}),
                       ("trs_dequant_mx4", {**DEQUANT, "rows": 1, "codes": X + 1}), ("trs_rms_norm_mx4", {**NORM, "rows": 1, "codes": X + 4}),
                       ("trs_matmul_mx4", {**MATMUL, "m": 1, "a": X + 8}), ("trs_matmul_mx4", {**MATMUL, "n": 1, "w": X + 8}),
                       ("trs_matmul_mx4", {**MATMUL, "m": 1, "lda": 31}), ("trs_quant_mx4", {**QUANT, "rows": 2, "ldc": 33})]:
        assert getattr(lib, name)(*args.values()) == 1, name


@pytest.mark.parametrize("field", ["lr_device", "grad_scale_device", "step_device", "skip"])
def test_adamw_numbers_inside_of_what_is_written(field):
    size = 8 if field == "step_device" else 4
    for at in (X, X + 36, X + 40 - size, X + 512, X + 1024 + 40 - size):
        assert adamw([tensor()], options(**{field: at})) == 1
        assert b"overlaps" in nat.lib().trs_last_error()
