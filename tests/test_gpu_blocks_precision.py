"""What include/blocks.h says about the sums and the range of the block products, at inputs made to reach it."""
import numpy as np
import pytest
import torch

from blocks_oracle import CODES, DTYPES, ROUNDING, f64

pytestmark = pytest.mark.gpu


def given(values, exponents, weight=False):
    """Blocks of these codes; exponents one a block, the same in every row."""
    from tcc_spmm_amd.blocks import BlockTensor, BlockWeight
    q = torch.from_numpy(values.astype(np.float32)).cuda().to(CODES["e4m3"])
    assert np.array_equal(f64(q.float()), values)
    rows, blocks = values.shape[0], len(exponents)
    e = torch.full((-(-rows // 128) if weight else rows, -(-blocks // 4) * 4), 127, dtype=torch.uint8)
    e[:, :blocks] = torch.tensor(exponents, dtype=torch.uint8)
    return (BlockWeight if weight else BlockTensor)(q, e.cuda(), values.shape[1])


# Rows and outer widths that take each kernel of the 16-bit product.
@pytest.mark.parametrize("rows,outer", [(3, 40), (24, 512), (300, 400), (1500, 2048), (4096, 4096), (20000, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_sums_of_eight_products(gpu, rows, outer, dtype):
    """A product of 256 in every eight of a block and seven just below 2^-13 of it, which the 8-bit MFMA cuts off; the
    next block takes the large ones away. A 16-bit sum is off by no more than 7 * 2^-13 of the terms' magnitudes, an
    FP32 one not at all: every partial sum is a multiple of 15 * 2^-9 below 2^13."""
    from tcc_spmm_amd.blocks import linear_blocks, matmul_blocks
    x, w = np.full((rows, 256), 0.5), np.full((outer, 256), 1.875 * 2.0 ** -5)
    x[:, ::8], w[:, ::8] = 16.0, 16.0
    x[:, 128:], x[:, 128::8] = 0.0, -16.0
    x[::2] *= -1.0
    want, terms = x @ w.T, np.abs(x) @ np.abs(w).T
    assert abs(want[0, 0]) == 16 * 7 * 1.875 * 2.0 ** -6
    blocks, weight = given(x, [127, 127]), given(w, [127, 127], weight=True)
    exact = f64(matmul_blocks(blocks, weight, dtype=torch.float32))
    assert np.array_equal(exact, want)
    dense = torch.from_numpy(x).cuda().to(DTYPES[dtype])  # quantizes to the same values
    for y in (matmul_blocks(blocks, weight, dtype=DTYPES[dtype]), linear_blocks(dense, weight)):
        off = np.abs(f64(y) - want)
        assert (off <= 7 * 2.0 ** -13 * terms + ROUNDING[dtype] * np.abs(want)).all(), off.max()


@pytest.mark.parametrize("rows,inner,outer", [(1, 4096, 512), (777, 1001, 700), (2048, 1024, 1024), (20000, 128, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_random_sums_differ_from_fp32_ones_by_few_roundings(gpu, rows, inner, outer, dtype):
    """16-bit outputs against FP32 sums, rounded. Sums that are off by d = 2.4e-5 of their norm, twice what random
    numbers give, move a part d / unit of the outputs to the other side of a rounding, each by a unit, which is at most
    2 * ROUNDING of it: together sqrt(d / unit) * unit = sqrt(d * 2 * ROUNDING) of the norm."""
    from tcc_spmm_amd.blocks import matmul_blocks, quantize_blocks, quantize_weight_blocks
    gen = torch.Generator().manual_seed(rows)
    x = quantize_blocks(torch.randn((rows, inner), generator=gen).cuda())
    weight = quantize_weight_blocks((torch.randn((outer, inner), generator=gen) * inner ** -0.5).cuda())
    exact = matmul_blocks(x, weight, dtype=torch.float32)
    y = matmul_blocks(x, weight, dtype=DTYPES[dtype])
    off = (y.float() - exact.to(DTYPES[dtype]).float()).norm() / exact.norm()
    assert float(off) <= np.sqrt(2.4e-5 * 2 * ROUNDING[dtype])
    assert torch.equal(y, matmul_blocks(x, weight, dtype=DTYPES[dtype])), "repeated calls give the same bits"
