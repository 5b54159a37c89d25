"""Workgroups that go through many tiles, and plans of more runs than one step of their prefix sums takes, against the
definitions in 64 bits: every element, on the GPU."""
import numpy as np
import pytest
import torch

import micro_oracle as O
from blocks_oracle import DTYPES, ROUNDING
from test_gpu_blocks import U, random
from test_gpu_micro import FORMATS
from test_micro_forms import expert_form, product_form

pytestmark = pytest.mark.gpu


def coded(x, codes):
    from tcc_spmm_amd.blocks import quantize_blocks
    from tcc_spmm_amd.micro import quantize_micro
    return (quantize_blocks if codes == "e4m3" else quantize_micro)(x)


def check(y, x, w, dtype, codes, bias=0.0):
    """y against x w^T + bias in 64 bits, by the room that test_gpu_micro.py derives."""
    want, terms = torch.matmul(x, w.t().contiguous()), torch.matmul(x.abs(), w.abs().t().contiguous())
    room = (x.shape[1] / 4 + 16) * U * terms
    if codes == "e4m3" and dtype != "f32":
        room += 7 * 2.0 ** -13 * terms
    want = want + bias
    room = (room + 4 * U * want.abs()) * 1.01 + ROUNDING[dtype] * want.abs() + (2.0 ** -25 if dtype == "f16" else 0)
    assert ((y.double() - want).abs() <= room).all(), float(((y.double() - want).abs() - room).max())


# 36 x 37 tiles of 256 for 256 workgroups; odd and even numbers of steps, and of pairs of them
@pytest.mark.parametrize("inner", [600, 1024, 520])
@pytest.mark.parametrize("dtype,codes", [("bf16", "e4m3"), ("f16", "e4m3"), ("bf16", "e2m1"), ("f32", "e2m1"), ("f16", "e2m1")])
@pytest.mark.parametrize("packed", [False, True])
def test_more_than_five_tiles_a_workgroup(gpu, inner, dtype, codes, packed):
    from tcc_spmm_amd.micro import linear_micro, matmul_micro, quantize_weight_micro
    rows, outer = 9001, 9300
    assert product_form(rows, inner, outer, dtype, codes, "matmul") == "microWide"
    x, bias = random((rows, inner), 1, dtype), random((outer,), 2)
    weight = quantize_weight_micro(random((outer, inner), 3, "bf16", inner ** -0.5))
    rows_ = coded(x, codes)
    call = (lambda: linear_micro(x, weight, bias, codes=FORMATS[codes])) if packed else (
        lambda: matmul_micro(rows_, weight, bias, dtype=DTYPES[dtype]))
    y = call()
    check(y, rows_.dequantize().double(), weight.dequantize().double(), dtype, codes, bias.double())
    assert torch.equal(y, call()), "repeated calls give the same bits"


@pytest.mark.parametrize("dtype,codes", [("bf16", "e4m3"), ("bf16", "e2m1"), ("f32", "e2m1")])
@pytest.mark.parametrize("by_token", [False, True])
def test_experts_of_more_than_4096_possible_tiles(gpu, dtype, codes, by_token):
    """128 experts, each with a row more than whole tiles: 639 row tiles of 640 that there can be, by 8, for a launch of more
    than 256 workgroups, each with up to 16, as many as it has room for."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import quantize_weight_micro
    count, each, inner, outer = 128, 4, 1030, 2000
    rng = np.random.default_rng(0)
    tiles = rng.multinomial(511, np.ones(count) / count)
    ids = np.repeat(np.arange(count), 256 * tiles + 1)
    rng.shuffle(ids)
    choices, tokens = ids.size, ids.size // each
    assert choices == 130944 and (choices // 256 + count + 1) * -(-outer // 256) > 4096
    assert expert_form(choices, count, inner, outer, dtype, codes) == "microWide"
    plan = X.sort_experts(torch.from_numpy(ids.reshape(tokens, each)).cuda(), count)
    weight = quantize_weight_micro(random((count, outer, inner), 1, "bf16", inner ** -0.5))
    bias = random((count, outer), 2)
    x = random((tokens if by_token else choices, inner), 3, dtype)
    y = X.linear_experts(x, weight, plan, bias, by_token=by_token, codes=FORMATS[codes])
    values = coded(x, codes).dequantize()
    if by_token:
        values = values[plan.order.long() // each]
    bounds = plan.offsets.tolist()
    stack = weight.dequantize()
    for e in range(count):
        span = slice(bounds[e], bounds[e + 1])
        check(y[span], values[span].double(), stack[e].double(), dtype, codes, bias[e].double())
    assert torch.equal(y, X.linear_experts(x, weight, plan, bias, by_token=by_token, codes=FORMATS[codes]))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,each,count", [(5_000_000, 1, 70), (1_100_000, 4, 1024)])
def test_plans_of_more_than_1024_runs(gpu, tokens, each, count, dtype):
    from tcc_spmm_amd.experts import sort_experts
    ids = np.random.default_rng(0).integers(-3, count + 3, (tokens, each))
    plan = sort_experts(torch.from_numpy(ids).to(dtype).cuda(), count)
    for got, want in zip((plan.offsets, plan.order, plan.places), O.plan(ids, count)):
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("rows,inner,outer,form", [(1, 4096, 4096, "microTokens"), (16, 4096, 1000, "microTiles32"),
                                                   (48, 4096, 8191, "microTiles64x32"), (777, 1001, 1437, "microTiles64"),
                                                   (4091, 300, 4099, "microTiles128"), (3900, 600, 4000, "microWide")])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_repeated_calls_give_the_same_bits(gpu, rows, inner, outer, form, dtype):
    """8-bit rows through every kernel, with other work of the card's between the calls."""
    from tcc_spmm_amd.micro import linear_micro, quantize_weight_micro
    assert dtype == "f32" or product_form(rows, inner, outer, dtype, "e4m3") == form
    x, weight = random((rows, inner), 1, dtype), quantize_weight_micro(random((outer, inner), 2, spread=inner ** -0.5))
    first = linear_micro(x, weight)
    for _ in range(5):
        torch.mm(x.float(), x.float().t().contiguous())
        assert torch.equal(linear_micro(x, weight), first)
