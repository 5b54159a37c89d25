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


# Codes of every kind: subnormal ones, an odd one among them, the smallest normal one, the largest.
KINDS = np.array([2.0 ** -9, 3 * 2.0 ** -9, 7 * 2.0 ** -9, 2.0 ** -6, 1.0, 1.875, 240.0, 448.0])


def in_bf16(v):
    return torch.from_numpy(v).float().bfloat16().double().numpy()


@pytest.mark.parametrize("e", [0, 1, 2, 3, 4, 127, 245, 246, 247, 248, 254])
@pytest.mark.parametrize("rows,outer", [(8, 40), (600, 600)])
def test_values_at_the_ends_of_the_range(gpu, rows, outer, e):
    """One product a sum, so that it shows what a code and its exponent stand for: in a 16-bit output always the value,
    in an FP32 output and in the weight gradient the value as bf16 has it, which is the same for exponents of 3 to 246."""
    from tcc_spmm_amd.blocks import matmul_blocks, weight_grad_blocks
    f = min(max(254 - e, 30), 220)  # brings the products back to the middle of the range
    value, factor = KINDS * 2.0 ** (e - 127), 2.0 ** (f - 127)
    if 3 <= e <= 246:
        assert np.array_equal(in_bf16(value), value)
    one, kinds = np.zeros((outer, 128)), np.zeros((rows, 128))
    one[:, 0], kinds[:8, 0] = 1.0, KINDS
    x, w = given(kinds, [e]), given(one, [f], weight=True)
    assert np.array_equal(f64(matmul_blocks(x, w, dtype=torch.bfloat16))[:8, 0], value * factor)
    assert np.array_equal(f64(matmul_blocks(x, w, dtype=torch.float32))[:8, 0], in_bf16(value) * factor)
    # the same codes in the weight
    one, kinds = np.zeros((rows, 128)), np.zeros((outer, 128))
    one[:, 0], kinds[:8, 0] = 1.0, KINDS
    y = matmul_blocks(given(one, [f]), given(kinds, [e], weight=True), dtype=torch.float32)
    assert np.array_equal(f64(y)[0, :8], in_bf16(value) * factor)
    if e > 246:  # an infinite value of another row makes the sum NaN
        return
    factor = 2.0 ** (100 if e < 100 else -100 if e > 200 else 0)
    for dtype in (torch.float32, torch.bfloat16):
        for columns in (outer, outer + 1):
            dy = torch.zeros((rows, columns), device="cuda", dtype=dtype)
            dy[torch.arange(8), torch.arange(8)] = factor
            assert np.array_equal(f64(weight_grad_blocks(dy, x)[0])[:8, 0], in_bf16(value) * factor)


@pytest.mark.parametrize("rows", [3, 40, 500, 9000])
def test_rows_near_the_smallest_numbers(gpu, rows):
    """FP32 rows whose blocks have the least exponents, through a layer: bf16 keeps a value to 2^-134."""
    from tcc_spmm_amd.blocks import linear_blocks, quantize_blocks
    x = torch.zeros((rows, 128), device="cuda")
    x[:, 0], x[:, 1] = 2.0 ** -118, 3 * 2.0 ** -135
    kept = quantize_blocks(x)
    assert (kept.exponents[:, 0] == 1).all() and np.array_equal(f64(kept.dequantize()), f64(x))
    w = np.zeros((64, 128))
    w[:, 1] = 1.0
    y = linear_blocks(x, given(w, [227], weight=True))
    assert np.array_equal(f64(y), np.full((rows, 64), in_bf16(np.array(3 * 2.0 ** -135)) * 2.0 ** 100))
