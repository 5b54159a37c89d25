"""The experts' input gradient against its formula in 64 bits and against differences."""
import numpy as np
import pytest

import micro_oracle as O
from blocks_oracle import ROUNDING, f64
from test_gpu_blocks import U, near, random, rounded
from test_gpu_experts import choices
from test_gpu_micro import FORMATS, product_room, row_values

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 1, 1, 1), (24, 4, 32, 200, 130), (50, 3, 5, 33, 300), (700, 2, 3, 264, 520), (2500, 2, 4, 300, 600)]


@pytest.mark.parametrize("tokens,each,count,inner,outer", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
@pytest.mark.parametrize("by_token", [False, True])
def test_input_gradient(gpu, tokens, each, count, inner, outer, dtype, codes, by_token):
    """dx[r] = Q(dy[r]) W[e] of each row, rounded to x's type; by token the sum of its choices' in FP32, rounded again. Rows of no
    expert count nothing, whatever their gradient holds."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import quantize_weight_micro
    ids = choices(tokens, each, count, 1, 0.2)
    plan = X.sort_experts(ids, count)
    offsets, _, places = O.plan(ids.cpu().numpy(), count)
    w = random((count, outer, inner), 2, spread=outer ** -0.5)
    stack = quantize_weight_micro(w, tiles=True, transposed=True)
    x = random((tokens if by_token else tokens * each, inner), 3, dtype).requires_grad_()
    dy = random((tokens * each, outer), 4, dtype)
    X.expert_linear(x, stack, plan, by_token=by_token, codes=FORMATS[codes]).backward(dy)
    gv = row_values(dy, codes)
    want, room = np.zeros((tokens * each, inner)), np.zeros((tokens * each, inner))
    for e in range(count):
        span = slice(offsets[e], offsets[e + 1])
        wv = O.quantize_tiles(f64(w[e]))[2]
        want[span] = gv[span] @ wv
        room[span] = product_room(gv[span], wv.T, dtype, codes)
    room = (room + 4 * U * np.abs(want)) * 1.01 + rounded(want, dtype)
    if by_token:
        rows, spread = want[places].reshape(tokens, each, inner), room[places].reshape(tokens, each, inner)
        want = rows.sum(1)
        room = spread.sum(1) + (each + 1) * U * (np.abs(rows) + spread).sum(1)
        room = room + rounded(want, dtype) + ROUNDING[dtype] * room
    near(x.grad, want, room, "dx")


@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
def test_against_differences(gpu, codes):
    """The layer is linear in the values of its codes: differences of sum(Q(dy) y) along a direction of x are the gradient's
    product with it, by the values that the stack's own rows stand for, which its transposed copy shares."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import quantize_weight_micro
    tokens, each, count, inner, outer = 60, 3, 5, 150, 90
    plan = X.sort_experts(choices(tokens, each, count, 1, 0.1), count)
    stack = quantize_weight_micro(random((count, outer, inner), 2), tiles=True, transposed=True)
    x = random((tokens, inner), 3).requires_grad_()
    dy = random((tokens * each, outer), 4)
    X.expert_linear(x, stack, plan, by_token=True, codes=FORMATS[codes]).backward(dy)
    values, g = f64(stack.dequantize()), row_values(dy, codes)
    offsets, order = plan.offsets.tolist(), plan.order.cpu().numpy()

    def loss(v):
        total = 0.0
        for e in range(count):
            span = slice(offsets[e], offsets[e + 1])
            total += (g[span] * (v[order[span] // each] @ values[e].T)).sum()
        return total

    at = f64(x)
    for seed in range(3):
        v = np.random.default_rng(seed).standard_normal(at.shape)
        diff = (loss(at + v) - loss(at - v)) / 2
        grad = f64(x.grad)
        # FP32 sums of at most 90 terms, of three choices
        assert abs((grad * v).sum() - diff) <= 1e-5 * np.abs(grad * v).sum()
