"""Argument checks of the 8-bit block entry points, on the CPU: every refusal comes before a launch."""
import ctypes
import re
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT

P = 0x1000  # an address that no check dereferences


def rejected(status, text):
    from tcc_spmm_amd._lib import lib
    assert status == 1 and text in lib().tcc_last_error(), (status, lib().tcc_last_error())


def test_quantize_refusals():
    from tcc_spmm_amd._lib import lib
    L = lib()
    call = lambda x=P, stride=128, t=0, c=P, e=P, ct=0, rows=4, n=128: L.tcc_quantize_blocks(  # noqa: E731
        x, stride, t, c, e, ct, rows, n, None)
    rejected(call(x=None), b"null dense")
    rejected(call(stride=127), b"stride")
    rejected(call(t=3), b"element type")
    rejected(call(x=P + 2), b"aligned to its elements")
    rejected(call(x=P + 1, t=1), b"aligned to its elements")
    rejected(call(c=None), b"null codes")
    rejected(call(e=None), b"null codes")
    rejected(call(c=P + 8), b"16-byte")
    rejected(call(e=P + 2), b"4-byte")
    rejected(call(ct=2), b"code type")
    rejected(call(n=0), b"zero elements")
    rejected(call(n=(1 << 22) + 1, stride=1 << 23), b"4,194,304")
    rejected(call(rows=1 << 31), b"2^31")
    assert call(rows=0) == 0  # nothing to do, with or without a GPU
    rejected(L.tcc_dequantize_blocks(P, P, 0, None, 128, 0, 4, 128, None), b"null dense")
    rejected(L.tcc_quantize_weight_blocks(P, 128, 0, P, P, P, None, 128, 128, None), b"together")
    rejected(L.tcc_quantize_weight_blocks(P, 128, 0, None, P, None, None, 128, 128, None), b"null codes")


def test_product_refusals():
    from tcc_spmm_amd._lib import lib
    L = lib()
    matmul = lambda x=P, w=P, bias=None, y=P, stride=64, t=0, rows=100, k=128, n=64: L.tcc_matmul_blocks(  # noqa: E731
        x, P, w, P, bias, y, stride, t, rows, k, n, None)
    rejected(matmul(x=None), b"null codes")
    rejected(matmul(w=None), b"null codes")
    rejected(matmul(bias=P + 2), b"bias")
    rejected(matmul(y=None), b"null dense")
    rejected(matmul(stride=63), b"stride")
    rejected(matmul(t=7), b"element type")
    rejected(matmul(k=0), b"zero elements")
    rejected(matmul(n=0), b"zero elements")
    assert matmul(rows=0) == 0
    size = ctypes.c_size_t()
    assert L.tcc_linear_blocks_workspace(1000, 300, 64, 0, 0, ctypes.byref(size)) == 0
    assert size.value >= 1000 * (384 + 4)
    linear = lambda keep=None, keepe=None, space=P, size=size.value: L.tcc_linear_blocks(  # noqa: E731
        P, 300, 0, P, P, None, P, 64, keep, keepe, 1000, 300, 64, space, size, None)
    rejected(linear(size=size.value - 1), b"workspace too small")
    rejected(linear(space=None), b"workspace too small")
    rejected(linear(space=P + 8), b"16-byte")
    rejected(linear(keep=P), b"together")
    rejected(L.tcc_linear_blocks_workspace(1000, 300, 64, 0, 0, None), b"null")


def test_weight_gradient_refusals():
    from tcc_spmm_amd._lib import lib
    L = lib()
    size = ctypes.c_size_t()
    assert L.tcc_weight_grad_blocks_workspace(100000, 128, 128, 0, ctypes.byref(size)) == 0 and size.value
    call = lambda dy=P, x=P, dw=P, db=None, space=P, n=size.value, t=0: L.tcc_weight_grad_blocks(  # noqa: E731
        dy, 128, t, x, P, dw, db, 100000, 128, 128, space, n, None)
    rejected(call(dy=None), b"null dense")
    rejected(call(x=None), b"null codes")
    rejected(call(dw=None), b"null weight gradient")
    rejected(call(db=P + 1), b"float-aligned")
    rejected(call(n=size.value - 1), b"workspace too small")
    rejected(call(t=4), b"element type")


def test_activation_refusals():
    from tcc_spmm_amd._lib import lib
    L = lib()
    fwd = lambda x=P, stride=256, kind=0, gated=1, y=P, c=P, e=P, ct=1: L.tcc_activation_blocks(  # noqa: E731
        x, stride, 1, kind, gated, y, 128, c, e, ct, 4, 128, None)
    rejected(fwd(x=None), b"null dense")
    rejected(fwd(stride=255), b"stride")
    rejected(fwd(kind=3), b"unknown activation")
    rejected(fwd(y=None), b"null dense")
    rejected(fwd(e=None), b"together")
    rejected(fwd(ct=2), b"code type")
    bwd = lambda dy=P, c=P, dx=P, kind=0: L.tcc_activation_blocks_backward(  # noqa: E731
        dy, 128, 1, c, P if c else None, 1, kind, 0, dx, 128, 4, 128, None)
    rejected(bwd(dy=None), b"null dense")
    rejected(bwd(c=None), b"null codes")
    rejected(bwd(dx=None), b"null dense")
    rejected(bwd(kind=9), b"unknown activation")


def test_the_cxx_surface_is_exported():
    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("nm is not installed")
    from tcc_spmm_amd._lib import LIB_PATH
    text = re.sub(r"//[^\n]*", "", (ROOT / "include" / "blocks.h").read_text())
    names = set(re.findall(r"^(?:void|std::size_t)\s+([A-Za-z]\w*)\s*\(", text, flags=re.M))
    assert {"quantizeBlocks", "matmulBlocks", "linearBlocks", "weightGradBlocks", "activationBlocks",
            "activationBlocksBackward", "quantizeWeightBlocks", "dequantizeBlocks"} <= names
    out = subprocess.run([nm, "-DC", str(LIB_PATH)], capture_output=True, text=True, check=True).stdout
    assert names <= {m.group(1) for m in re.finditer(r"\sT\s+([A-Za-z_]\w*)\(", out)}
    # a kernel's host stub that its template did not get would only show when the library is loaded
    assert "__device_stub__" not in "".join(line for line in out.splitlines() if " U " in line)


def test_torch_side_refusals_need_no_gpu():
    from tcc_spmm_amd import blocks as B
    x = torch.zeros((4, 128))
    codes, exponents = torch.zeros((4, 128), dtype=B.INT8), torch.zeros((4, 4), dtype=torch.uint8)
    for make in (lambda: B.BlockTensor(codes.to(torch.uint8), exponents, 100), lambda: B.BlockTensor(codes, exponents, 129),
                 lambda: B.BlockTensor(codes, exponents[:3], 100), lambda: B.BlockTensor(codes, exponents.int(), 100),
                 lambda: B.BlockTensor(codes.t(), exponents, 100), lambda: B.BlockTensor(codes, exponents, 0),
                 lambda: B.BlockWeight(codes, exponents[:1], 100),
                 lambda: B.BlockWeight(codes.to(B.E4M3), exponents[:1], 100, codes_t=codes.to(B.E4M3)),
                 lambda: B.quantize_blocks(x.double()), lambda: B.quantize_blocks(torch.zeros((4, 0))),
                 lambda: B.quantize_weight_blocks(x[0]), lambda: B.activation_blocks(x, "tanh")):
        with pytest.raises(ValueError):
            make()
    with pytest.raises(ValueError, match="CUDA"):
        B.quantize_blocks(x)


def test_an_activation_that_keeps_nothing_has_no_gradient():
    """Said by the call itself, not by an error in its backward pass."""
    from tcc_spmm_amd import blocks as B
    with pytest.raises(ValueError, match="requires a gradient"):
        B.block_activation(torch.zeros((4, 128), requires_grad=True), codes=None)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # nothing to say against the call itself
        B.block_activation(torch.zeros((4, 128), requires_grad=True), codes=None)


def test_a_bias_gradient_needs_no_blocks():
    """Without dw nothing of x is looked at, and the workspace is for db alone."""
    from tcc_spmm_amd._lib import lib
    from tcc_spmm_amd import blocks as B
    L = lib()
    whole, alone = ctypes.c_size_t(), ctypes.c_size_t()
    assert L.tcc_weight_grad_blocks_workspace(1000000, 128, 256, 1, ctypes.byref(whole)) == 0
    assert L.tcc_weight_grad_blocks_workspace(1000000, 0, 256, 1, ctypes.byref(alone)) == 0
    assert 0 < alone.value < whole.value / 16
    call = lambda dy=P, x=None, dw=None, db=P, k=0, n=alone.value: L.tcc_weight_grad_blocks(  # noqa: E731
        dy, 256, 1, x, x, dw, db, 1000000, k, 256, P, n, None)
    rejected(call(dy=None), b"null dense")
    rejected(call(db=None), b"null weight gradient")
    rejected(call(n=alone.value - 1), b"workspace too small")
    rejected(call(dw=P), b"zero elements")  # a weight gradient of no columns
    rejected(call(dw=P, k=128), b"null codes")
    with pytest.raises(ValueError, match="asked for"):
        B.weight_grad_blocks(torch.zeros((4, 128)), None, bias=False)


def test_products_of_more_tiles_than_a_launch_takes():
    """A launch has fewer than 2^32 threads: 2^24 tiles, of 256 x 256 for 16 bits, else of 128 x 128, are refused by the
    call, not by the runtime."""
    from tcc_spmm_amd._lib import lib
    L = lib()
    most = (1 << 31) - 1
    matmul = lambda t, rows, n: L.tcc_matmul_blocks(P, P, P, P, None, P, n, t, rows, 128, n, None)  # noqa: E731
    for t, rows, n in ((1, most, 512), (2, most, 257), (1, 1 << 22, 1 << 18), (0, most, 128), (0, 1 << 30, 129)):
        rejected(matmul(t, rows, n), b"more tiles than a launch takes")
    rejected(L.tcc_quantize_weight_blocks(P, 1 << 20, 0, P, P, None, None, 1 << 20, 1 << 20, None), b"than a launch takes")
    size = ctypes.c_size_t()
    assert L.tcc_weight_grad_blocks_workspace(64, 1 << 21, 1 << 20, 1, ctypes.byref(size)) == 0 and size.value == 0
    rejected(L.tcc_weight_grad_blocks(P, 1 << 20, 0, P, P, P, None, 64, 1 << 20, 1 << 20, P, 1 << 40, None),
             b"than a launch takes")


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_layers_refuse_other_devices(device):
    """With the call's own error, with and without gradients and autocast."""
    from tcc_spmm_amd import blocks as B
    x, w = torch.zeros((4, 128), device=device), torch.zeros((8, 128), device=device, requires_grad=True)
    for context in (torch.enable_grad, torch.no_grad, lambda: torch.autocast("cuda", torch.bfloat16, enabled=False)):
        with context(), pytest.raises(ValueError, match="CUDA"):
            B.block_linear(x, w)
        with context(), pytest.raises(ValueError, match="CUDA"):
            B.block_activation(x)
