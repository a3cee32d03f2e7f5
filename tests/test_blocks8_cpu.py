"""8-bit blocks: what is refused and how results are laid out, without a GPU."""
import ctypes as C

import pytest
import torch

from medicalimageanalysis_amd import _lib, blocks8


def blocks(rows, width, tiled=False):
    return blocks8.Blocks8(torch.zeros(blocks8.Blocks8.bytes_for(rows, width, tiled), dtype=torch.uint8), (rows, width), tiled)


@pytest.mark.parametrize("call,error,match", [
    (lambda: blocks8.Blocks8(torch.zeros(143, dtype=torch.uint8), (1, 5)), ValueError, "144 bytes"),
    (lambda: blocks8.Blocks8(torch.zeros(144, dtype=torch.uint8), (1, 5), offset=16), ValueError, "144 bytes"),
    (lambda: blocks8.Blocks8(torch.zeros(200, dtype=torch.uint8), (1, 5), offset=8), ValueError, "multiple of 16"),
    (lambda: blocks8.Blocks8(torch.zeros(288, dtype=torch.uint8)[::2], (1, 5)), ValueError, "dense"),
    (lambda: blocks8.Blocks8(torch.zeros(144), (1, 5)), ValueError, "uint8"),
    (lambda: blocks8.Blocks8(torch.zeros(144, dtype=torch.uint8), (3, 0)), ValueError, "shape"),
    (lambda: blocks8.quantize(torch.zeros(())), ValueError, "last dimension"),
    (lambda: blocks8.quantize(torch.zeros(3, 0)), ValueError, "last dimension"),
    (lambda: blocks8.quantize(torch.zeros(3, 4, dtype=torch.float64)), TypeError, "float32, float16 or bfloat16"),
    (lambda: blocks8.quantize(torch.zeros(3, 4), "relu"), ValueError, "activation"),
    (lambda: blocks8.quantize(torch.zeros(3, 4), "softplus", 0.0), ValueError, "beta"),
    (lambda: blocks8.quantize(torch.zeros(3, 4), "softplus", float("nan")), ValueError, "beta"),
    (lambda: blocks8.quantize(torch.zeros(3, 4)), RuntimeError, "HIP device"),
    (lambda: blocks8.Weight8(blocks(3, 5), None, torch.float32), ValueError, "tiles"),
    (lambda: blocks8.Weight8(blocks(3, 5, True), blocks(5, 4, True), torch.float32), ValueError, "transpose"),
    (lambda: blocks8.quantize_weight(torch.zeros(4)), ValueError, "matrix"),
    (lambda: blocks8.quantize_weight(torch.zeros(0, 4)), ValueError, "matrix"),
    (lambda: blocks8.matmul(torch.zeros(2, 3), blocks(2, 3)), TypeError, "Blocks8"),
    (lambda: blocks8.matmul(blocks(2, 3), blocks(2, 4)), ValueError, "shapes"),
    (lambda: blocks8.matmul(blocks(2, 3), blocks(5, 3), torch.zeros(4)), ValueError, r"shape \(5,\)"),
    (lambda: blocks8.matmul(blocks(2, 3), blocks(5, 3), dtype=torch.float64), TypeError, "float64"),
    (lambda: blocks8.softplus_grad(torch.zeros(2, 4), blocks(2, 3)), ValueError, "shapes"),
    (lambda: blocks8.softplus_grad(torch.zeros(2, 3), blocks(2, 3, True)), ValueError, "shapes"),
    (lambda: blocks8.weight_grad(torch.zeros(3, 5), blocks(2, 3)), ValueError, "shapes"),
    (lambda: blocks8.weight_grad(torch.zeros(2, 5), blocks(2, 3), dtype=torch.bfloat16), TypeError, "results"),
    (lambda: blocks8.linear(torch.zeros(2, 3), torch.zeros(5, 4)), ValueError, "weight of shape"),
    (lambda: blocks8.linear(torch.zeros(2, 3), torch.zeros(3)), ValueError, "matrix"),
    (lambda: blocks8.linear(torch.zeros(2, 3), torch.zeros(5, 3, dtype=torch.float16)), TypeError, "float16"),
    (lambda: blocks8.linear(torch.zeros(2, 3, dtype=torch.float64), torch.zeros(5, 3)), TypeError, "float64"),
    (lambda: blocks8.linear(torch.zeros(2, 3), torch.zeros(5, 3), torch.zeros(3)), ValueError, r"shape \(5,\)"),
    (lambda: blocks8.linear(torch.zeros(2, 3), torch.zeros(5, 3)), RuntimeError, "HIP device"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


@pytest.mark.parametrize("rows,width,tiled,values,exponents", [
    (1, 1, False, (1, 128), (1, 16)), (17, 128, False, (17, 128), (1, 32)), (16, 129, False, (16, 256), (2, 16)),
    (129, 300, True, (129, 384), (3, 2)), (0, 5, False, (0, 128), (1, 16))])
def test_layout(rows, width, tiled, values, exponents):
    q = blocks(rows, width, tiled)
    assert tuple(q.values.shape) == values and tuple(q.exponents.shape) == exponents
    assert q.storage.numel() % 16 == 0


def test_c_entry_refusals():
    lib = _lib.lib()
    p, odd = C.c_void_p(256), C.c_void_p(257)

    def quantize(rows=4, width=8, x=p, values=p, pitch=16, act=0, beta=1.0, dtype=0):
        return lib.vmf_blocks8_quantize(x, 8, values, p, pitch, rows, width, act, beta, dtype, None)

    assert quantize(rows=(1 << 26) + 1, pitch=1 << 27) == -4  # a launch has fewer than 2^32 threads
    assert quantize(rows=-1) == -1 and quantize(width=0) == -1 and quantize(width=(1 << 22) + 1) == -4
    assert quantize(x=None) == -1 and quantize(values=odd) == -1 and quantize(pitch=3) == -1
    assert quantize(act=2) == -1 and quantize(act=1, beta=0.0) == -1 and quantize(dtype=1) == -2
    assert quantize(rows=0, x=None) == 0
    assert lib.vmf_blocks8_quantize_tiles(p, 8, p, p, p, None, 4, 8, 0, None) == -1
    assert lib.vmf_blocks8_dequantize(p, p, 1, 0, p, 4, 8, 0, None) == -1
    assert lib.vmf_blocks8_softplus_grad(None, 8, p, p, 16, p, 4, 8, 1.0, 0, None) == -1

    def matmul(m=4, n=4, k=8, a=p, pitch=16, out=p, ws=None, nbytes=0, dtype=0, bias=None, bias_dtype=0, gate=None,
               beta=1.0):
        return lib.vmf_blocks8_matmul(a, p, pitch, 0, p, p, 16, 0, bias, bias_dtype, gate, p, 16, beta, out, m, n, k, ws,
                                      nbytes, dtype, None)

    assert matmul(m=1 << 26, n=1 << 26, pitch=1 << 26) == -1  # (b's exponent pitch)
    assert lib.vmf_blocks8_matmul(p, p, 1 << 26, 0, p, p, 1 << 26, 0, None, 0, None, p, 16, 1.0, p, 1 << 26, 1 << 26, 8, None,
                                  0, 0, None) == -4
    assert matmul(m=-1) == -1 and matmul(k=0) == -1 and matmul(a=None) == -1 and matmul(a=odd) == -1
    assert matmul(pitch=8) == -1 and matmul(out=None) == -1 and matmul(dtype=1) == -2
    assert matmul(bias=p, bias_dtype=1) == -2 and matmul(gate=p, beta=-1.0) == -1
    assert matmul(m=0) == 0
    need = C.c_int64(0)
    assert lib.vmf_blocks8_matmul_workspace(4, 4, 8, 0, need) == 0 and need.value == 0
    assert lib.vmf_blocks8_matmul_workspace(4, 4, 1 << 16, 0, need) == 0 and need.value > 0
    assert matmul(k=1 << 16, ws=p, nbytes=need.value - 1) == -1 and b"workspace" in lib.vmf_last_error_string()

    def weight_grad(m=4, n=4, k=8, g=p, gw=p, dtype=0, out_dtype=0, ws=None, nbytes=0):
        return lib.vmf_blocks8_weight_grad(g, 8, p, p, -(-m // 16) * 16, gw, None, None, None, 0, m, n, k, ws, nbytes, dtype, out_dtype,
                                           None)

    assert weight_grad(m=-1) == -1 and weight_grad(g=None) == -1 and weight_grad(gw=None) == -1
    assert weight_grad(dtype=3, out_dtype=2) == -2 and weight_grad(n=0) == 0
    assert lib.vmf_blocks8_weight_grad_workspace(1 << 16, 128, 128, 0, need) == 0 and need.value > 0
    assert weight_grad(m=1 << 16, n=128, k=128, ws=p, nbytes=need.value - 1) == -1


def test_layer_entry_refusals():
    lib = _lib.lib()
    p = C.c_void_p(256)
    need = C.c_int64(0)
    assert lib.vmf_blocks8_linear_fwd_workspace(4, 4, 8, 0, 1, 0, need) == 0 and need.value > 0

    def fwd(m=4, n=4, k=8, weight=p, dtype=0, w_dtype=0, act=0, nbytes=need.value, ws=p, wt=None, wte=None):
        return lib.vmf_blocks8_linear_fwd(p, 8, weight, 8, w_dtype, None, None, wt, wte, None, 0, act, 1.0, p, p, 16, p, m, n,
                                          k, ws, nbytes, dtype, None)

    assert fwd(m=-1) == -1 and fwd(n=0) == -1 and fwd(k=0) == -1 and fwd(act=3) == -1
    assert fwd(nbytes=need.value - 1) == -1 and fwd(ws=C.c_void_p(264)) == -1 and fwd(wt=p) == -1
    assert fwd(dtype=3, w_dtype=2) == -2
    assert fwd(m=0, weight=None) == 0  # no rows and no weight to lay out: nothing to do
    few = C.c_int64(-1)
    assert lib.vmf_blocks8_linear_fwd_workspace(1, 4096, 4096, 1, 0, 0, few) == 0 and few.value == 0  # one launch
    assert lib.vmf_blocks8_linear_fwd_workspace(17, 4096, 4096, 1, 0, 0, few) == 0 and few.value > 0
    assert lib.vmf_blocks8_linear_fwd_workspace(1, 0, 4096, 1, 0, 0, few) == -1
    assert lib.vmf_blocks8_linear_bwd_workspace(4, 4, 8, 0, need) == 0 and need.value > 0
    assert lib.vmf_blocks8_linear_bwd_workspace(4, 0, 8, 0, need) == -1
    assert lib.vmf_blocks8_linear_bwd_workspace(4, 4, 8, 0, need) == 0

    def bwd(m=4, n=4, k=8, gx=p, gw=p, gb=p, wt=p, nbytes=need.value, w_dtype=0):
        return lib.vmf_blocks8_linear_bwd(p, 8, p, p, 16, wt, p, 0, 1.0, gx, gw, gb, m, n, k, p, nbytes, 0, w_dtype, None)

    assert bwd(m=-1) == -1 and bwd(gw=None) == -1 and bwd(wt=None) == -1 and bwd(nbytes=need.value - 1) == -1
    assert bwd(w_dtype=2) == -2


def test_bias_gradient_entry_refusals():
    lib = _lib.lib()
    p = C.c_void_p(256)
    need = C.c_int64(-1)
    assert lib.vmf_blocks8_bias_grad_workspace(100, 128, 0, need) == 0 and need.value == 0
    assert lib.vmf_blocks8_bias_grad_workspace(1 << 16, 128, 0, need) == 0 and need.value > 0
    assert lib.vmf_blocks8_bias_grad_workspace(-1, 128, 0, need) == -1
    assert lib.vmf_blocks8_bias_grad_workspace(4, 0, 0, need) == -1
    assert lib.vmf_blocks8_bias_grad_workspace(4, (1 << 22) + 1, 0, need) == -4
    assert lib.vmf_blocks8_bias_grad_workspace(4, 4, 0, None) == -1

    def grad(g=p, gb=p, stride=8, m=4, ws=None, nbytes=0, dtype=0, out_dtype=0):
        return lib.vmf_blocks8_bias_grad(g, stride, gb, m, 128, ws, nbytes, dtype, out_dtype, None)

    assert grad(g=None) == -1 and grad(gb=None) == -1 and grad(stride=-1) == -1 and grad(m=-1) == -1
    assert grad(dtype=3, out_dtype=2) == -2 and grad(dtype=1, out_dtype=1) == -2
    assert grad(m=1 << 16, ws=p, nbytes=need.value - 1) == -1


def test_layer_backward_needs_xs_blocks_for_the_softplus_gradient():
    """without them gx would come out without its factor"""
    lib = _lib.lib()
    p = C.c_void_p(256)
    need = C.c_int64(0)
    assert lib.vmf_blocks8_linear_bwd_workspace(4, 4, 8, 0, need) == 0

    def bwd(a=p, ae=p, act=1, gx=p, m=4):
        return lib.vmf_blocks8_linear_bwd(None, 8, a, ae, 16, p, p, act, 1.0, gx, None, None, m, 4, 8, p, need.value, 0, 0,
                                          None)

    # (gy is null as well, so that no call gets past its checks)
    for call in (dict(a=None), dict(ae=None)):
        assert bwd(**call) == -1 and b"blocks" in lib.vmf_last_error_string()
    for act in (-1, 2):
        assert bwd(act=act) == -1 and b"activation" in lib.vmf_last_error_string()
        assert bwd(act=act, gx=None) == -1
    assert bwd() == -1 and b"null pointer" in lib.vmf_last_error_string()
    assert bwd(a=None, m=0) == 0 and bwd(a=None, gx=None) == 0


@pytest.mark.parametrize("call,error,match", [
    (lambda: blocks(3, 5).dequantize(), RuntimeError, "HIP device"),
    (lambda: blocks(3, 5, True).dequantize(torch.bfloat16), RuntimeError, "HIP device"),
    (lambda: blocks8.softplus_grad(torch.zeros(3, 5), torch.zeros(3, 5)), TypeError, "softplus_grad takes Blocks8"),
    (lambda: blocks8.weight_grad(torch.zeros(3, 4), torch.zeros(3, 5)), TypeError, "weight_grad takes Blocks8"),
    (lambda: blocks8.matmul(blocks(2, 3), torch.zeros(5, 3)), TypeError, "matmul takes Blocks8"),
    (lambda: blocks8.Weight8(torch.zeros(3, 5), None, torch.float32), TypeError, "Weight8 takes Blocks8"),
    (lambda: blocks8.Weight8(blocks(3, 5, True), torch.zeros(5, 3), torch.float32), TypeError, "Weight8 takes Blocks8"),
])
def test_refusals_of_other_operands_and_of_blocks_in_host_memory(call, error, match):
    with pytest.raises(error, match=match):
        call()
