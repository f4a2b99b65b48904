"""Outputs that a caller gives count as changed in place: a backward pass through what autograd saved of them before is refused,
as after torch's own in-place operations, and so is nothing else."""
import pytest
import torch

import trspmm

pytestmark = pytest.mark.gpu


def rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def calls():
    """name -> (the call, the outputs that it is given)."""
    x, res = rand((6, 64), torch.float16, 1), rand((6, 64), torch.float16, 2)
    weight = torch.ones(64, device="cuda")
    ids = torch.tensor([3, 0, 5, 5], device="cuda")
    codes, scale = trspmm.quant_mx4(x)
    q, s, _ = trspmm.rms_norm_i8(x, weight)
    new = (lambda shape, dtype: torch.zeros(shape, dtype=dtype, device="cuda"))
    out16, out32, grad, wide, eight = new((6, 64), torch.float16), new((6, 64), torch.float16), new((6, 64), torch.float16), \
        new((8, 64), torch.float32), new((6, 64), torch.int8)
    rows, scale8, dweight, square = new((4, 64), torch.float16), new(6, torch.float32), new(64, torch.float32), new((6, 6), torch.float16)
    code_out, scale_out = new((6, 32), torch.uint8), new((6, 2), torch.uint8)
    return {
        "embed": (lambda: trspmm.embed(x, ids, out=rows), [rows]),
        "embed_grad": (lambda: trspmm.embed_grad(rows, ids, 8, out=wide), [wide]),
        "rms_norm": (lambda: trspmm.rms_norm(x, weight, res, out=out16, r_out=res), [out16, res]),
        "rms_norm_i8": (lambda: trspmm.rms_norm_i8(x, weight, res, out=eight, scale=scale8, r_out=res), [eight, scale8, res]),
        "rms_norm_grad": (lambda: trspmm.rms_norm_grad(x, res, weight, out=grad, dweight=dweight), [grad, dweight]),
        "matmul_i8": (lambda: trspmm.matmul_i8(q, s, q, s, out=square), [square]),
        "quant_mx4": (lambda: trspmm.quant_mx4(x, out=code_out, scale=scale_out), [code_out, scale_out]),
        "dequant_mx4": (lambda: trspmm.dequant_mx4(codes, scale, 64, out=out32), [out32]),
        "rms_norm_mx4": (lambda: trspmm.rms_norm_mx4(x, weight, res, out=code_out, scale=scale_out, r_out=res), [code_out, scale_out, res]),
        "matmul_mx4": (lambda: trspmm.matmul_mx4(codes, scale, codes, scale, out=square), [square]),
    }, [x, weight, ids, codes, scale, q, s]


NAMES = ["embed", "embed_grad", "rms_norm", "rms_norm_i8", "rms_norm_grad", "matmul_i8", "quant_mx4", "dequant_mx4", "rms_norm_mx4", "matmul_mx4"]


@pytest.mark.parametrize("name", NAMES)
def test_given_outputs_count_as_changed(name):
    print("versions", name, flush=True)
    table, inputs = calls()
    call, written = table[name]
    was, kept = [t._version for t in written], [t._version for t in inputs]
    call()
    assert all(t._version > v for t, v in zip(written, was))
    assert [t._version for t in inputs] == kept


@pytest.mark.parametrize("name", NAMES)
def test_in_inference_mode(name):
    print("inference", name, flush=True)
    with torch.inference_mode():
        calls()[0][name][0]()


def test_a_saved_residual_that_is_written():
    print("saved residual", flush=True)
    x, weight = rand((6, 64), torch.float16, 1), torch.ones(64, device="cuda")
    for norm in (trspmm.rms_norm, trspmm.rms_norm_i8, trspmm.rms_norm_mx4):
        res = rand((6, 64), torch.float16, 2).requires_grad_()
        loss = (res * res).sum()
        norm(x, weight, res, r_out=res)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_a_refused_call_changes_nothing():
    print("refused", flush=True)
    x, out = rand((6, 64), torch.float16, 1), torch.zeros((6, 64), dtype=torch.float16, device="cuda")
    was = out._version
    with pytest.raises(trspmm._native.TrsError):
        trspmm.rms_norm(x, torch.ones(64, device="cuda"), eps=0.0, out=out)
    assert out._version == was
