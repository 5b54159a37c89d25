"""Each kernel of the block products and of the weight gradient, at sizes that it takes: the calls' own rules say which, so
that a rule set to other figures cannot leave a kernel without a test."""
import ctypes

import numpy as np
import pytest
import torch

import blocks_oracle as O
import test_gpu_blocks as base
from blocks_oracle import DTYPES, f64
from test_gpu_blocks import U, near, random

TYPES = {"f32": 0, "bf16": 1, "f16": 2}


def product_form(rows, inner, outer, dtype, call="linear"):
    from tcc_spmm_amd._lib import check, lib
    form = ctypes.c_char_p()
    check(getattr(lib(), f"tcc_{call}_blocks_form")(rows, inner, outer, TYPES[dtype], ctypes.byref(form)))
    return form.value.decode()


def gradient_form(at, stride, dtype, rows, inner, outer):
    """(kernel, splits) for a dy at this address."""
    from tcc_spmm_amd._lib import check, lib
    form, splits = ctypes.c_char_p(), ctypes.c_uint32()
    check(lib().tcc_weight_grad_blocks_form(at, stride, TYPES[dtype], rows, inner, outer, ctypes.byref(form),
                                            ctypes.byref(splits)))
    return form.value.decode(), splits.value


# Odd and even numbers of blocks and of groups of four, ragged edges, one tile and many.
PRODUCTS = [
    ("multiplyWide", "bf16", 3900, 600, 4000), ("multiplyWide", "f16", 3900, 600, 4000),
    ("multiplyWide", "bf16", 4096, 1024, 4096), ("multiplyWide", "f16", 3840, 1300, 4090),
    ("multiplyTiles128", "bf16", 4091, 300, 4099), ("multiplyTiles128", "f16", 1900, 1500, 2300),
    ("multiplyTiles128", "bf16", 2048, 1024, 4096), ("multiplyTiles128", "f16", 2500, 900, 1700),
    ("multiplyTiles64", "bf16", 777, 1001, 1437), ("multiplyTiles64", "f16", 300, 384, 513),
    ("multiplyTiles32", "bf16", 32, 2900, 513), ("multiplyTiles32", "f16", 24, 4096, 1000),
    ("multiplyTilesExact", "f32", 600, 300, 600), ("multiplyTilesExact", "f32", 700, 2048, 1000),
    ("multiplyTokens", "f32", 16, 512, 64), ("multiplyTokens", "f32", 32, 2900, 513), ("multiplyTokens", "f32", 200, 1300, 257),
    ("multiplyTokensDense", "f32", 1, 4096, 130), ("multiplyTokensDense", "bf16", 3, 100, 77),
    ("multiplyTokensDense", "f16", 4, 1001, 50),
    *(("multiplyRows", t, *size) for t in TYPES for size in ((8199, 120, 40), (16400, 250, 130), (16391, 300, 100),
                                                            (16401, 512, 60))),
]
PRODUCT_KERNELS = {"multiplyWide", "multiplyTiles128", "multiplyTiles64", "multiplyTiles32", "multiplyTilesExact",
                   "multiplyTokens", "multiplyTokensDense", "multiplyRows"}

# kernel, splits, type, rows, inner, outer
GRADIENTS = [
    ("sumRowsInPlace256", 1, "bf16", 3000, 4000, 4040), ("sumRowsInPlace256", 3, "bf16", 4100, 2000, 2056),
    ("sumRowsInPlace256", 1, "bf16", 1990, 2900, 4104),
    ("sumRowsInPlace128", 1, "bf16", 1030, 1000, 2056), ("sumRowsInPlace128", 6, "bf16", 4000, 1000, 520),
    ("sumRows128", 1, "f32", 1030, 2900, 2050), ("sumRows128", 6, "f16", 4000, 1000, 520), ("sumRows128", 79, "bf16", 5003, 128, 201),
    ("sumRows64", 1, "f32", 100, 130, 40), ("sumRows64", 157, "f16", 20000, 128, 64), ("sumRows64", 1, "bf16", 100, 130, 41),
    ("sumRowsNarrow", 1, "f32", 100, 130, 5), ("sumRowsNarrow", 79, "f16", 5003, 100, 3), ("sumRowsNarrow", 1, "bf16", 65, 300, 7),
]
GRADIENT_KERNELS = {"sumRowsInPlace256", "sumRowsInPlace128", "sumRows128", "sumRows64", "sumRowsNarrow"}


def test_the_sizes_below_take_every_kernel():
    for form, dtype, rows, inner, outer in PRODUCTS:
        assert product_form(rows, inner, outer, dtype) == form
        given = product_form(rows, inner, outer, dtype, "matmul")
        assert given == form or form in ("multiplyTokensDense", "multiplyRows") and given != form
    for form, splits, dtype, rows, inner, outer in GRADIENTS:
        assert gradient_form(0x1000, outer, dtype, rows, inner, outer) == (form, splits)
    assert {p[0] for p in PRODUCTS} == PRODUCT_KERNELS and {g[0] for g in GRADIENTS} == GRADIENT_KERNELS
    # each type that a kernel is built for
    assert {p[:2] for p in PRODUCTS} >= {(k, t) for k in PRODUCT_KERNELS if "Tiles" in k and "Exact" not in k or "Wide" in k
                                        for t in ("bf16", "f16")} | {("multiplyRows", t) for t in TYPES}


def test_form_refusals():
    from tcc_spmm_amd._lib import lib
    form = ctypes.c_char_p()
    L = lib()
    assert L.tcc_linear_blocks_form(4, 0, 4, 0, ctypes.byref(form)) == 1
    assert L.tcc_matmul_blocks_form(4, 4, 4, 3, ctypes.byref(form)) == 1
    assert L.tcc_matmul_blocks_form(4, 4, 4, 0, None) == 1
    assert L.tcc_weight_grad_blocks_form(None, 4, 3, 4, 4, 4, ctypes.byref(form), None) == 1
    assert L.tcc_weight_grad_blocks_form(None, 4, 0, 4, 4, 4, ctypes.byref(form), None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("form,dtype,rows,inner,outer", PRODUCTS)
def test_products(gpu, form, dtype, rows, inner, outer):
    assert product_form(rows, inner, outer, dtype) == form
    base.test_linear(gpu, rows, inner, outer, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("form,splits,dtype,rows,inner,outer", GRADIENTS)
def test_gradients(gpu, form, splits, dtype, rows, inner, outer):
    """Sums of n products through the MFMA, which adds at least four at once, in a few splits: (n / 4 + 64) roundings of
    2^-24 of the magnitudes' sum."""
    from tcc_spmm_amd.blocks import quantize_blocks, weight_grad_blocks
    x, dy = random((rows, inner), 1, dtype), random((rows, outer), 2, dtype, 1e-2)
    assert gradient_form(dy.data_ptr(), outer, dtype, rows, inner, outer) == (form, splits)
    kept = quantize_blocks(x)
    xv, g = O.quantize(f64(x))[2], f64(dy)
    dw, db = weight_grad_blocks(dy, kept)
    near(dw, g.T @ xv, (rows / 4 + 64) * U * (np.abs(g).T @ np.abs(xv)) + 1e-30, "dw")
    near(db, g.sum(0), (rows / 4 + 64) * U * np.abs(g).sum(0) + 1e-30, "db")
    again = weight_grad_blocks(dy, kept)
    assert torch.equal(dw, again[0]) and torch.equal(db, again[1]), "repeated calls give the same bits"
    assert torch.equal(weight_grad_blocks(dy, kept, bias=False)[0], dw)


@pytest.mark.gpu
@pytest.mark.parametrize("form,dtype,rows,inner,outer", [p for i, p in enumerate(PRODUCTS) if p[:2] not in
                                                         {q[:2] for q in PRODUCTS[:i]} or p[0] in ("multiplyRows", "multiplyTokens")])
def test_nan_stays_in_its_rows_and_columns(gpu, form, dtype, rows, inner, outer):
    """A NaN or an infinity in x makes its row NaN, in the weight the columns of its tile, and everything else is what it
    is without it."""
    from tcc_spmm_amd.blocks import linear_blocks, quantize_weight_blocks
    x, w = random((rows, inner), 1, dtype), random((outer, inner), 2)
    clean = linear_blocks(x, quantize_weight_blocks(w))
    bad = torch.zeros((rows, outer), dtype=torch.bool, device="cuda")
    if outer > 128:
        w[outer - 1, inner - 1] = float("nan")
        bad[:, (outer - 1) // 128 * 128:] = True
    for row, column, value in ((0, 0, float("nan")), (rows // 2, inner - 1, float("inf")), (rows - 1, inner // 2, float("-inf"))):
        x[row, column] = value
        bad[row] = True
    y = linear_blocks(x, quantize_weight_blocks(w))
    assert y[bad].isnan().all() and torch.equal(y[~bad], clean[~bad])
    kept = linear_blocks(x, quantize_weight_blocks(w), keep=True)[1]
    base.check_blocks(kept, x, "e4m3")


@pytest.mark.gpu
@pytest.mark.parametrize("form,splits,dtype,rows,inner,outer", GRADIENTS)
def test_nan_stays_in_its_columns_of_the_gradient(gpu, form, splits, dtype, rows, inner, outer):
    """A NaN in dy makes its row of dw NaN and its sum, one in x the columns of its block."""
    from tcc_spmm_amd.blocks import quantize_blocks, weight_grad_blocks
    x, dy = random((rows, inner), 1, dtype), random((rows, outer), 2, dtype)
    clean, clean_db = weight_grad_blocks(dy, quantize_blocks(x))
    bad = torch.zeros((outer, inner), dtype=torch.bool, device="cuda")
    if inner > 128:
        x[rows - 1, inner - 1] = float("inf")
        bad[:, (inner - 1) // 128 * 128:] = True
    dy[rows // 2, outer - 1] = float("nan")
    bad[outer - 1] = True
    dw, db = weight_grad_blocks(dy, quantize_blocks(x))
    assert dw[bad].isnan().all() and torch.equal(dw[~bad], clean[~bad])
    assert db[-1].isnan() and torch.equal(db[:-1], clean_db[:-1])


@pytest.mark.gpu
@pytest.mark.parametrize("form,splits,dtype,rows,inner,outer", [g for g in GRADIENTS if "InPlace" in g[0]] +
                         [("sumRowsInPlace128", 1, "bf16", 300, 256, 136), ("sumRowsInPlace128", 1, "bf16", 1, 300, 8)])
@pytest.mark.parametrize("left,right", [(8, 0), (16, 8), (0, 72)])
def test_gradients_of_aligned_slices(gpu, form, splits, dtype, rows, inner, outer, left, right):
    """A slice of a wider dy whose rows keep their alignment takes the same kernel as dy by itself, gives the same bits, and
    reads nothing beside it."""
    from tcc_spmm_amd.blocks import quantize_blocks, weight_grad_blocks
    kept, dy = quantize_blocks(random((rows, inner), 1, dtype)), random((rows, outer), 2, dtype)
    wide = base.cut(dy, left, right)
    assert rows == 1 or wide.stride(0) > outer
    assert gradient_form(wide.data_ptr(), wide.stride(0), dtype, rows, inner, outer) == (form, splits)
    want, got = weight_grad_blocks(dy, kept), weight_grad_blocks(wide, kept)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = base.cut(dy, 3, 2)
    assert not gradient_form(odd.data_ptr(), odd.stride(0), dtype, rows, inner, outer)[0].startswith("sumRowsInPlace")
