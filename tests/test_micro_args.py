"""Argument checks of the microscaled and expert entry points, on the CPU: every refusal comes before a launch."""
import ctypes
import re
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT
from test_blocks_args import P, rejected


def test_quantize_refusals():
    from tcc_spmm_amd._lib import lib
    L = lib()
    call = lambda x=P, stride=128, t=0, c=P, e=P, rows=4, n=128: L.tcc_quantize_micro(  # noqa: E731
        x, stride, t, c, e, rows, n, None)
    rejected(call(x=None), b"null dense")
    rejected(call(stride=127), b"stride")
    rejected(call(t=3), b"element type")
    rejected(call(x=P + 2), b"aligned to its elements")
    rejected(call(c=None), b"null codes")
    rejected(call(e=None), b"null codes")
    rejected(call(c=P + 8), b"16-byte")
    rejected(call(e=P + 4), b"16-byte")
    rejected(call(n=0), b"zero elements")
    rejected(call(n=(1 << 22) + 1, stride=1 << 23), b"4,194,304")
    rejected(call(rows=1 << 31), b"2^31")
    rejected(call(rows=(1 << 31) - 1, n=1 << 12, stride=1 << 12), b"2^32 runs")
    assert call(rows=0) == 0  # nothing to do, with or without a GPU
    rejected(L.tcc_dequantize_micro(P, P, None, 128, 0, 4, 128, None), b"null dense")
    weight = lambda w=P, ct=P, et=P, experts=1, outer=128: L.tcc_quantize_weight_micro(  # noqa: E731
        w, 128, 0, P, P, ct, et, experts, outer, 128, None)
    rejected(weight(w=None), b"null dense")
    rejected(weight(et=None), b"together")
    rejected(weight(ct=P + 8), b"16-byte")
    rejected(weight(experts=0), b"65,535")
    rejected(weight(experts=65536), b"65,535")
    rejected(weight(outer=0), b"zero elements")


@pytest.mark.parametrize("form", [0, 1])
def test_product_refusals(form):
    from tcc_spmm_amd._lib import lib
    L = lib()
    matmul = lambda x=P, w=P, f=form, bias=None, y=P, stride=64, t=0, rows=100, k=128, n=64: L.tcc_matmul_micro(  # noqa: E731
        x, P, f, w, P, bias, y, stride, t, rows, k, n, None)
    rejected(matmul(x=None), b"null codes")
    rejected(matmul(w=None), b"null codes")
    rejected(matmul(w=P + 8), b"16-byte")
    rejected(matmul(f=2), b"row format")
    rejected(matmul(bias=P + 2), b"bias")
    rejected(matmul(y=None), b"null dense")
    rejected(matmul(stride=63), b"stride")
    rejected(matmul(t=7), b"element type")
    rejected(matmul(k=0), b"zero elements")
    rejected(matmul(n=0), b"zero elements")
    rejected(matmul(rows=1 << 31), b"2^31")
    assert matmul(rows=0) == 0
    most = (1 << 31) - 1
    for t, rows, n in ((1, most, 512), (0, most, 512), (1, 1 << 22, 1 << 18)):
        rejected(matmul(t=t, rows=rows, n=n, stride=n), b"than a launch takes")
    size = ctypes.c_size_t()
    assert L.tcc_linear_micro_workspace(1000, 300, 64, 0, form, 0, ctypes.byref(size)) == 0
    assert size.value >= 1000 * (192 + 16 if form else 384 + 4)
    linear = lambda keep=None, keepe=None, space=P, size=size.value: L.tcc_linear_micro(  # noqa: E731
        P, 300, 0, form, P, P, None, P, 64, keep, keepe, 1000, 300, 64, space, size, None)
    rejected(linear(size=size.value - 1), b"workspace too small")
    rejected(linear(space=None), b"workspace too small")
    rejected(linear(space=P + 8), b"16-byte")
    rejected(linear(keep=P), b"together")
    if form:
        rejected(linear(keep=P, keepe=P), b"E4M3")
    rejected(L.tcc_linear_micro_workspace(1000, 300, 64, 0, form, 0, None), b"null")
    name = ctypes.c_char_p()
    assert L.tcc_linear_micro_form(1, 128, 64, 1, form, ctypes.byref(name)) == 0 and name.value == b"microTokens"
    rejected(L.tcc_matmul_micro_form(1, 128, 64, 1, 2, ctypes.byref(name)), b"row format")
    rejected(L.tcc_matmul_micro_form(1, 128, 64, 1, form, None), b"null")


def test_plan_refusals():
    from tcc_spmm_amd._lib import lib
    L = lib()
    size = ctypes.c_size_t()
    assert L.tcc_sort_experts_workspace(16384, 64, ctypes.byref(size)) == 0 and size.value == 0
    assert L.tcc_sort_experts_workspace(100000, 64, ctypes.byref(size)) == 0 and size.value
    call = lambda ids=P, wide=8, offsets=P, order=P, n=100000, experts=64, space=P, size=size.value: L.tcc_sort_experts(  # noqa: E731
        ids, wide, offsets, order, P, n, experts, space, size, None)
    rejected(call(ids=None), b"null choices")
    rejected(call(order=None), b"null choices")
    rejected(call(offsets=None), b"null choices")
    rejected(call(wide=2), b"4 or 8 bytes")
    rejected(call(ids=P + 4), b"aligned to their type")
    rejected(call(order=P + 2), b"plan not aligned")
    rejected(call(experts=0), b"1 to 1024")
    rejected(call(experts=1025), b"1 to 1024")
    rejected(call(n=1 << 31), b"2^31")
    rejected(call(size=size.value - 1), b"workspace too small")
    rejected(call(space=None), b"workspace too small")
    rejected(call(space=P + 8), b"16-byte")


def test_rows_refusals():
    from tcc_spmm_amd._lib import lib
    L = lib()
    gather = lambda x=P, offsets=P, n=8, each=2, experts=4, rows=P, width=64, stride=64: L.tcc_gather_experts(  # noqa: E731
        x, 64, 1, offsets, P, n, each, experts, rows, stride, width, None)
    rejected(gather(x=None), b"null dense")
    rejected(gather(rows=None), b"null dense")
    rejected(gather(stride=63), b"stride")
    rejected(gather(offsets=None), b"null plan")
    rejected(gather(offsets=P + 2), b"plan not aligned")
    rejected(gather(each=3), b"whole tokens")
    rejected(gather(each=0), b"1 to 1024")
    rejected(gather(experts=0), b"1 to 1024")
    rejected(gather(n=1 << 31), b"2^31")
    rejected(gather(width=0), b"zero elements")
    rejected(L.tcc_gather_experts(P, 2048, 1, P, P, 1 << 25, 2, 4, P, 2048, 2048, None), b"than a launch takes")
    assert gather(n=0, offsets=None) == 0
    combine = lambda rows=P, w=P, wt=0, y=P: L.tcc_combine_experts(  # noqa: E731
        rows, 64, 1, P, P, 8, 2, 4, w, wt, y, 64, 64, None)
    rejected(combine(rows=None), b"null dense")
    rejected(combine(w=P + 2), b"weights not aligned")
    rejected(combine(wt=3), b"element type")
    rejected(combine(y=None), b"null dense")
    back = lambda dy=P, rows=P, w=P, drows=P, dw=P: L.tcc_combine_experts_backward(  # noqa: E731
        dy, 64, rows, 64, 1, P, P, 8, 2, 4, w, 0, drows, 64, dw, 64, None)
    rejected(back(dy=None), b"null dense")
    rejected(back(rows=None), b"null dense")
    rejected(back(drows=None, dw=None), b"asked for")
    rejected(back(dw=P + 2), b"weights not aligned")


def test_expert_product_refusals():
    from tcc_spmm_amd._lib import lib
    L = lib()
    matmul = lambda x=P, f=1, by=0, w=P, order=P, n=80, each=2, experts=4, k=128: L.tcc_matmul_experts(  # noqa: E731
        x, P, f, by, w, P, None, P, 64, 1, P, order, n, each, experts, k, 64, None)
    rejected(matmul(x=None), b"null codes")
    rejected(matmul(w=None), b"null codes")
    rejected(matmul(f=3), b"row format")
    rejected(matmul(order=None), b"null plan")
    rejected(matmul(each=3), b"whole tokens")
    rejected(matmul(experts=1025), b"1 to 1024")
    rejected(matmul(k=0), b"zero elements")
    rejected(matmul(by=1, n=1 << 26, k=1 << 8), b"gather them")
    assert matmul(n=0) == 0
    size = ctypes.c_size_t()
    assert L.tcc_linear_experts_workspace(80, 2, 4, 1, 300, 64, 1, 0, ctypes.byref(size)) == 0 and 40 * 388 <= size.value < 80 * 388
    call = lambda x=P, space=P, size=size.value: L.tcc_linear_experts(  # noqa: E731
        x, 300, 1, 0, 1, P, P, None, P, 64, P, P, 80, 2, 4, 300, 64, space, size, None)
    rejected(call(x=None), b"null dense")
    rejected(call(size=size.value - 1), b"workspace too small")
    rejected(call(space=None), b"workspace too small")
    rejected(call(space=P + 8), b"16-byte")
    name = ctypes.c_char_p()
    assert L.tcc_matmul_experts_form(80, 8, 128, 64, 1, 1, ctypes.byref(name)) == 0 and name.value == b"microTiles64"
    rejected(L.tcc_matmul_experts_form(80, 0, 128, 64, 1, 1, ctypes.byref(name)), b"1 to 1024")


def test_the_cxx_surface_is_exported():
    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("nm is not installed")
    from tcc_spmm_amd._lib import LIB_PATH
    names = set()
    for header in ("micro.h", "experts.h"):
        text = re.sub(r"//[^\n]*", "", (ROOT / "include" / header).read_text())
        names |= set(re.findall(r"^(?:void|std::size_t|const char\*)\s+([A-Za-z]\w*)\s*\(", text, flags=re.M))
    assert {"quantizeMicro", "linearMicro", "matmulMicroForm", "sortExperts", "combineExpertsBackward", "linearExperts"} <= names
    out = subprocess.run([nm, "-DC", str(LIB_PATH)], capture_output=True, text=True, check=True).stdout
    assert names <= {m.group(1) for m in re.finditer(r"\sT\s+([A-Za-z_]\w*)\(", out)}


def test_torch_side_refusals_need_no_gpu():
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd import micro as M
    x = torch.zeros((4, 128))
    codes, exponents = torch.zeros((4, 64), dtype=torch.uint8).view(M.E2M1), torch.zeros((4, 16), dtype=torch.uint8)
    stack, many = codes.view(torch.uint8).reshape(1, 4, 64).view(M.E2M1), exponents.reshape(1, 4, 16)
    assert M.MicroWeight(stack, many, 100).experts == 1 and M.MicroWeight(codes, exponents, 100).experts is None
    for make in (lambda: M.MicroTensor(codes.view(torch.uint8), exponents, 100), lambda: M.MicroTensor(codes, exponents, 129),
                 lambda: M.MicroTensor(codes, exponents[:3], 100), lambda: M.MicroTensor(codes, exponents.int(), 100),
                 lambda: M.MicroTensor(stack, many, 100), lambda: M.MicroTensor(codes, exponents, 0),
                 lambda: M.MicroTensor(codes, exponents[:, :12], 100),
                 lambda: M.MicroWeight(codes[:0], exponents[:0], 100),
                 lambda: M.MicroWeight(codes, exponents, 100, codes_t=codes),
                 lambda: M.MicroWeight(codes, exponents, 100, codes, exponents),
                 lambda: M.MicroWeight(codes, exponents, 100).transposed(),
                 lambda: M.quantize_micro(x.double()), lambda: M.quantize_micro(torch.zeros((4, 0))),
                 lambda: M.quantize_weight_micro(x[0]), lambda: M.quantize_weight_micro(x, transposed=True),
                 lambda: X.sort_experts(x, 4), lambda: X.sort_experts(x.long(), 0)):
        with pytest.raises(ValueError):
            make()
    for call in (lambda: M.quantize_micro(x), lambda: X.sort_experts(x.long(), 4),
                 lambda: M.linear_micro(x, M.MicroWeight(codes, exponents, 128)), lambda: M.MicroWeight(codes, exponents, 128).dequantize()):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_layers_refuse_other_devices(device):
    """With the call's own error, with and without gradients."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd import micro as M
    x, w = torch.zeros((4, 128), device=device), torch.zeros((8, 128), device=device, requires_grad=True)
    lists = [torch.zeros(n, dtype=torch.int32, device=device) for n in (3, 8, 8)]
    plan = X.ExpertPlan(*lists, (4,), 2)
    for context in (torch.enable_grad, torch.no_grad):
        with context(), pytest.raises(ValueError, match="CUDA"):
            M.micro_linear(x, w)
        with context(), pytest.raises(ValueError, match="CUDA"):
            X.expert_gather(x, plan)
        with context(), pytest.raises(ValueError, match="CUDA"):
            X.expert_combine(torch.zeros((8, 128), device=device), plan)
