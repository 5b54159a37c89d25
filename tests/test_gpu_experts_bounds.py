"""The calls of a layer of experts write within what they are given and nowhere else, whatever the plan holds: outputs in the
middle of larger buffers of a known pattern, rows further apart than a row is wide."""
import numpy as np
import pytest
import torch

from test_gpu_blocks import random
from test_gpu_experts import choices
from test_micro_forms import FORMATS, TYPES, expert_form

pytestmark = pytest.mark.gpu

GUARD = 1 << 19  # elements in front and behind
KINDS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


class Guarded:
    """[rows, columns] of a type, `apart` elements from row to row, in a buffer of a known pattern."""

    def __init__(self, rows, columns, dtype, apart=0):
        apart = apart or columns
        self.size = rows * apart
        self.flat = torch.full((2 * GUARD + self.size,), -123.0 if dtype.is_floating_point else -123, device="cuda", dtype=dtype)
        self.start = self.flat.clone()
        self.rows = self.flat[GUARD:GUARD + self.size].view(rows, apart)[:, :columns]
        self.gaps = self.flat[GUARD:GUARD + self.size].view(rows, apart)[:, columns:]

    def check(self):
        assert torch.equal(self.flat[:GUARD], self.start[:GUARD]), "in front of the output"
        assert torch.equal(self.flat[GUARD + self.size:], self.start[GUARD + self.size:]), "behind the output"
        assert (self.gaps == -123.0).all(), "between the output's rows"


def lists_of(kind, choices_, count, seed):
    """(offsets, order, places) that are no plan of these sizes."""
    rng = np.random.default_rng(seed)
    if kind == "any":
        lists = [rng.integers(-2 ** 31, 2 ** 31, n) for n in (count + 1, choices_, choices_)]
    elif kind == "near":  # about the sizes that there are, in no order
        lists = [rng.integers(-3, choices_ + 4, n) for n in (count + 1, choices_, choices_)]
    else:  # all at the ends
        lists = [rng.choice([-2 ** 31, -1, 0, choices_, 2 ** 31 - 1], n) for n in (count + 1, choices_, choices_)]
    return [torch.from_numpy(t.astype(np.int32)).cuda() for t in lists]


# tokens, each, experts, inner, outer, type, codes, form
PRODUCTS = [(30, 2, 3, 64, 40, "f32", "e4m3", "microTiles64"), (30, 2, 3, 64, 40, "bf16", "e2m1", "microTiles64"),
            (90, 3, 200, 130, 70, "f16", "e4m3", "microTiles64"), (3001, 2, 8, 2048, 1000, "bf16", "e4m3", "microTiles128"),
            (3001, 2, 8, 2048, 1000, "f32", "e2m1", "microTiles128"), (3001, 2, 8, 1000, 2048, "bf16", "e4m3", "microWide"),
            (15000, 2, 70, 1000, 520, "bf16", "e2m1", "microWide")]


def product(given, plan, by_token, y):
    from tcc_spmm_amd._lib import check, lib
    x, weight, tokens, each, count, inner, outer, dtype, codes = given
    offsets, order = plan
    check(lib().tcc_matmul_experts(x.codes.data_ptr(), x.exponents.data_ptr(), FORMATS[codes], by_token, weight.codes.data_ptr(),
                                   weight.exponents.data_ptr(), 0, y.rows.data_ptr(), y.rows.stride(0), TYPES[dtype],
                                   offsets.data_ptr(), order.data_ptr(), tokens * each, each, count, inner, outer,
                                   torch.cuda.current_stream().cuda_stream))


def operands(tokens, each, count, inner, outer, dtype, codes, by_token):
    from tcc_spmm_amd.blocks import quantize_blocks
    from tcc_spmm_amd.micro import quantize_micro, quantize_weight_micro
    x = random((tokens if by_token else tokens * each, inner), 1, dtype)
    weight = quantize_weight_micro(random((count, outer, inner), 2, spread=inner ** -0.5))
    return (quantize_blocks if codes == "e4m3" else quantize_micro)(x), weight, tokens, each, count, inner, outer, dtype, codes


@pytest.mark.parametrize("tokens,each,count,inner,outer,dtype,codes,form", PRODUCTS)
@pytest.mark.parametrize("kind", ["any", "near", "ends"])
@pytest.mark.parametrize("by_token", [False, True])
def test_products_of_lists_that_are_no_plan(gpu, tokens, each, count, inner, outer, dtype, codes, form, kind, by_token):
    assert expert_form(tokens * each, count, inner, outer, dtype, codes) == form
    given = operands(tokens, each, count, inner, outer, dtype, codes, by_token)
    for seed in range(3):
        y = Guarded(tokens * each, outer, KINDS[dtype], outer + 3)
        product(given, lists_of(kind, tokens * each, count, seed)[:2], by_token, y)
        torch.cuda.synchronize()
        y.check()


@pytest.mark.parametrize("tokens,each,count,inner,outer,dtype,codes,form", PRODUCTS)
@pytest.mark.parametrize("part", [0.5, 1.4])
def test_products_of_another_call_s_plan(gpu, tokens, each, count, inner, outer, dtype, codes, form, part):
    """Offsets of fewer or of more choices: rows that they give an expert have its results, those behind them are zeros."""
    from tcc_spmm_amd import experts as X
    given = operands(tokens, each, count, inner, outer, dtype, codes, False)
    other = X.sort_experts(choices(int(tokens * part), each, count, 5), count)
    y = Guarded(tokens * each, outer, KINDS[dtype], outer + 3)
    product(given, (other.offsets, other.order), False, y)
    torch.cuda.synchronize()
    y.check()
    # the same rows' own choices, so that a plan of the call's sizes gives each row the expert that the offsets give it
    ends = other.offsets.clamp(max=tokens * each)
    mine = torch.searchsorted(ends[1:].contiguous(), torch.arange(tokens * each, device="cuda", dtype=torch.int32), right=True)
    plan = X.sort_experts(torch.where(mine < count, mine, -1).reshape(tokens, each), count)
    assert torch.equal(plan.order, torch.arange(tokens * each, device="cuda", dtype=torch.int32))
    assert torch.equal(y.rows, X.matmul_experts(given[0], given[1], plan, dtype=KINDS[dtype]))


@pytest.mark.parametrize("tokens,each,count,width", [(1, 1, 1, 1), (30, 2, 3, 64), (7, 9, 20, 500), (200, 8, 64, 1001), (40, 5, 6, 8200)])
@pytest.mark.parametrize("kind", ["plan", "any", "near", "ends"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_there_and_back(gpu, tokens, each, count, width, kind, dtype):
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd._lib import check, lib
    n, apart = tokens * each, width + 5
    offsets, _, places = lists_of(kind, n, count, 1)
    if kind == "plan":
        plan = X.sort_experts(choices(tokens, each, count, 1, 0.2), count)
        offsets, places = plan.offsets, plan.places
    x, rows, weights = random((tokens, width), 1, dtype), random((n, width), 2, dtype), random((tokens, each), 3)
    stream = torch.cuda.current_stream().cuda_stream
    sizes = (offsets.data_ptr(), places.data_ptr(), n, each, count)
    outs = [Guarded(n, width, KINDS[dtype], apart), Guarded(tokens, width, KINDS[dtype], apart),
            Guarded(n, width, KINDS[dtype], apart), Guarded(tokens, each, torch.float32)]
    check(lib().tcc_gather_experts(x.data_ptr(), width, TYPES[dtype], *sizes, outs[0].rows.data_ptr(), apart, width, stream))
    check(lib().tcc_combine_experts(rows.data_ptr(), width, TYPES[dtype], *sizes, weights.data_ptr(), 0, outs[1].rows.data_ptr(),
                                    apart, width, stream))
    check(lib().tcc_combine_experts_backward(x.data_ptr(), width, rows.data_ptr(), width, TYPES[dtype], *sizes, weights.data_ptr(), 0,
                                             outs[2].rows.data_ptr(), apart, outs[3].rows.data_ptr(), width, stream))
    torch.cuda.synchronize()
    for out in outs:
        out.check()
    if kind == "plan":
        want = (X.gather_experts(x, plan), X.combine_experts(rows, plan, weights),
                *X.combine_experts_backward(x, rows, plan, weights))
        assert all(torch.equal(out.rows, t) for out, t in zip(outs, want))


@pytest.mark.parametrize("tokens,each,count", [(1, 1, 1), (100, 3, 1023), (1500, 7, 64), (16385, 1, 6), (200003, 2, 70)])
def test_plans(gpu, tokens, each, count):
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd._lib import check, lib
    ids = choices(tokens, each, count, 1, 0.3)
    plan = X.sort_experts(ids, count)
    outs = [Guarded(1, n, torch.int32) for n in (count + 1, tokens * each, tokens * each)]
    space = Guarded(1, 1 << 20, torch.int32)
    check(lib().tcc_sort_experts(ids.data_ptr(), 8, *(out.rows.data_ptr() for out in outs), tokens * each, count,
                                 space.rows.data_ptr(), 4 << 20, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    for out, t in zip(outs, (plan.offsets, plan.order, plan.places)):
        out.check()
        assert torch.equal(out.rows[0], t)
    space.check()
