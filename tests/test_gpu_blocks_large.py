"""The block kernels at sizes that pass 32 bits somewhere."""
import pytest
import torch

from test_gpu_blocks import random

pytestmark = pytest.mark.gpu


@pytest.fixture
def room(gpu):
    """Skips where the card has less free memory than the test asks for, in GB; frees what it took."""
    def need(gigabytes):
        torch.cuda.empty_cache()
        if torch.cuda.mem_get_info()[0] < gigabytes * 1e9:
            pytest.skip(f"needs {gigabytes} GB of GPU memory")
    yield need
    torch.cuda.empty_cache()


def test_more_blocks_than_a_launch_takes_threads_for(room):
    """2^28 + 1000 rows of one block, of 16 threads each: more than 2^32 threads. Some rows from each part of the range
    are those of a call on them alone."""
    from tcc_spmm_amd import blocks as B
    room(120)
    rows = (1 << 28) + 1000
    x = torch.randn((rows, 4), device="cuda", dtype=torch.bfloat16)
    parts = [slice(at, at + 500) for at in (0, (1 << 27) - 250, (1 << 28) - 250, rows - 500)]
    kept = B.quantize_blocks(x)
    values = kept.dequantize(torch.bfloat16)
    for p in parts:
        want = B.quantize_blocks(x[p])
        assert torch.equal(kept.codes[p].view(torch.uint8), want.codes.view(torch.uint8))
        assert torch.equal(kept.exponents[p], want.exponents) and torch.equal(values[p], want.dequantize(torch.bfloat16))
    del kept, values
    y, act = B.activation_blocks(x, "silu")
    dx = B.activation_blocks_backward(y, act, "silu")
    for p in parts:
        want, want_act = B.activation_blocks(x[p], "silu")
        assert torch.equal(y[p], want) and torch.equal(act.codes[p], want_act.codes)
        assert torch.equal(dx[p], B.activation_blocks_backward(y[p], want_act, "silu"))


def test_product_of_more_rows_than_small_tiles_have_threads_for(room):
    """2^30 + 300 rows are too many tiles of 64 rows for a launch. Most rows are zeros; the others are those of a product
    of them alone."""
    from tcc_spmm_amd import blocks as B
    room(190)
    rows, outer = (1 << 30) + 300, 8
    codes = torch.zeros((rows, 128), device="cuda", dtype=torch.uint8).view(B.E4M3)
    exponents = torch.full((rows, 4), 127, device="cuda", dtype=torch.uint8)
    weight = B.quantize_weight_blocks(random((outer, 128), 1))
    parts = [slice(at, at + 300) for at in (0, (1 << 29) - 100, rows - 300)]
    for i, p in enumerate(parts):
        some = B.quantize_blocks(random((300, 128), 2 + i))
        codes[p], exponents[p] = some.codes, some.exponents
    y = B.matmul_blocks(B.BlockTensor(codes, exponents, 128), weight)
    for p in parts:
        alone = B.BlockTensor(codes[p].contiguous(), exponents[p].contiguous(), 128)
        # One block is one instruction's sum in every form of the product.
        assert torch.equal(y[p], B.matmul_blocks(alone, weight))
    assert not y[1000:100000].any()
