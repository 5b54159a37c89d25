"""Tokens sorted by expert and back, and the experts' products, against their definitions in 64 bits (tests/micro_oracle.py).

Plans and gathered rows have to be equal. What the other tolerances allow for:
- a token's sum of k products in FP32: k + 1 roundings of 2^-24 of the terms' magnitudes;
- a dot product of n terms, which each thread adds 8 at a time and the threads add in pairs: (n / 256 + 24) roundings, and
  no fewer than its own terms' n where a row is held by fewer threads: min(n, n / 256 + 24) + 8;
- products as in test_gpu_micro.py; one rounding to the output's type.
"""
import numpy as np
import pytest
import torch

import micro_oracle as O
from blocks_oracle import DTYPES, ROUNDING, f64
from test_gpu_blocks import U, cut, near, random, rounded
from test_gpu_micro import FORMATS, product_room, row_values

pytestmark = pytest.mark.gpu


def choices(tokens, each, experts, seed=0, away=0.0, dtype=torch.int64, kind="any"):
    rng = np.random.default_rng(seed)
    if kind == "one":  # every token to one expert
        ids = np.full((tokens, each), experts - 1)
    elif kind == "none":
        ids = np.full((tokens, each), -1)
    else:
        ids = rng.integers(0, experts, (tokens, each))
        if kind == "few":  # most experts get nothing
            ids = ids // 7 * 7
    ids = np.where(rng.random(ids.shape) < away, rng.choice([-1, experts, -2 ** 31, 2 ** 31 - 1], ids.shape), ids)
    return torch.from_numpy(ids).to(dtype).cuda()


PLANS = [(1, 1, 1), (1, 4, 8), (5, 3, 7), (24, 4, 32), (64, 8, 64), (1000, 4, 64), (1024, 4, 1024), (1025, 4, 1000), (4097, 1, 3),
         (4096, 8, 128), (30001, 6, 130), (100, 1, 1023), (3, 1024, 9), (16385, 1, 6), (200003, 2, 70)]


@pytest.mark.parametrize("tokens,each,experts", PLANS)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("away,kind", [(0.0, "any"), (0.3, "any"), (0.0, "one"), (0.0, "none"), (0.1, "few")])
def test_plan(gpu, tokens, each, experts, dtype, away, kind):
    from tcc_spmm_amd.experts import sort_experts
    ids = choices(tokens, each, experts, 1, away, dtype, kind)
    want = O.plan(ids.cpu().numpy(), experts)
    for given in (ids, ids.t().contiguous().t()):
        plan = sort_experts(given, experts)
        for got, exact in zip((plan.offsets, plan.order, plan.places), want):
            assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), exact)
    assert (plan.tokens, plan.each, plan.experts, plan.choices) == (tokens, each, experts, tokens * each)


def test_plan_of_wide_numbers_and_of_nothing(gpu):
    """int64 numbers whose low halves are experts; no tokens; leading dimensions."""
    from tcc_spmm_amd import experts as X
    ids = torch.tensor([[1, 1 + (1 << 32)], [-(1 << 40) + 2, 2]], device="cuda")
    plan = X.sort_experts(ids, 4)
    assert plan.order.tolist() == [0, 3, 1, 2] and plan.offsets.tolist() == [0, 0, 1, 2, 2]
    empty = X.sort_experts(ids[:0], 4)
    assert empty.offsets.tolist() == [0] * 5 and empty.choices == 0
    x = random((0, 16), 1)
    assert X.gather_experts(x, empty).shape == (0, 16) and X.combine_experts(x, empty).shape == (0, 16)
    assert X.combine_experts_backward(x, x, empty, torch.empty((0, 2), device="cuda"))[1].shape == (0, 2)
    deep = X.sort_experts(choices(12, 2, 5).reshape(3, 4, 2), 5)
    assert deep.lead == (3, 4) and X.combine_experts(random((24, 8), 1), deep).shape == (3, 4, 8)


WIDTHS = [(1, 1, 1, 1), (24, 4, 32, 2048), (5, 3, 7, 33), (33, 2, 8, 8), (7, 9, 20, 500), (200, 8, 64, 1000), (65, 1, 5, 4100),
          (3, 17, 40, 129), (40, 5, 6, 8200)]


@pytest.mark.parametrize("tokens,each,experts,width", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("away", [0.0, 0.4])
def test_rows_and_back(gpu, tokens, each, experts, width, dtype, away):
    """Gather, combine and their gradients; NaN in rows of no expert and in the weights of choices for none stays out."""
    from tcc_spmm_amd import experts as X
    ids = choices(tokens, each, experts, 2, away)
    plan = X.sort_experts(ids, experts)
    offsets, order, places = O.plan(ids.cpu().numpy(), experts)
    here = offsets[-1]
    x, rows, dy = random((tokens, width), 1, dtype), random((tokens * each, width), 2, dtype), random((tokens, width), 3, dtype)
    weights = random((tokens, each), 4).abs()
    used = (places < here).reshape(tokens, each)
    rows[here:] = float("nan")
    weights[torch.from_numpy(~used).cuda()] = float("nan")
    want = np.zeros((tokens * each, width))
    want[:here] = f64(x)[order[:here] // each]
    for given in (x, cut(x)):
        assert np.array_equal(f64(X.gather_experts(given, plan)), want)
    r, g = np.where(np.arange(tokens * each)[:, None] < here, f64(rows), 0.0)[places].reshape(tokens, each, width), f64(dy)
    for kind in (None, "f32", "bf16", "f16"):
        w = None if kind is None else weights.to(DTYPES[kind])
        wd = np.where(used, 1.0 if w is None else np.nan_to_num(f64(w)), 0.0)
        terms = np.abs(wd[:, :, None] * r).sum(1)
        want = (wd[:, :, None] * r).sum(1)
        y = X.combine_experts(rows, plan, w)
        near(y, want, (each + 1) * U * terms + rounded(want, dtype), "y")
        assert torch.equal(X.combine_experts(cut(rows), plan, w), y)
        if w is None:
            drows, dweights = X.combine_experts_backward(dy, None, plan, need=(True, False))
            assert dweights is None
        else:
            drows, dweights = X.combine_experts_backward(dy, rows, plan, w)
            want = np.where(used, (g[:, None] * r).sum(2), 0.0)
            room = (min(width, width / 256 + 24) + 8) * U * np.abs(g[:, None] * r).sum(2)
            near(dweights, want, room + ROUNDING[kind] * np.abs(want) + (2.0 ** -25 if kind == "f16" else 0), "dweights")
            more = X.combine_experts_backward(cut(dy), cut(rows), plan, w)
            assert torch.equal(more[0], drows) and torch.equal(more[1], dweights)
            assert torch.equal(X.combine_experts_backward(dy, rows, plan, w, need=(False, True))[1], dweights)
            assert torch.equal(X.combine_experts_backward(dy, None, plan, w, need=(True, False))[0], drows)
        flat = np.zeros((tokens * each, width))
        flat[:here] = (wd[:, :, None] * g[:, None]).reshape(-1, width)[order[:here]]
        near(drows, flat, U * np.abs(flat) + rounded(flat, dtype), "drows")


def test_the_same_expert_twice(gpu):
    """A token may choose an expert more than once: each choice has its row and its weight."""
    from tcc_spmm_amd import experts as X
    plan = X.sort_experts(torch.tensor([[2, 2, 0], [1, 1, 1]], device="cuda"), 3)
    assert plan.order.tolist() == [2, 3, 4, 5, 0, 1]
    rows, w = random((6, 40), 1), random((2, 3), 2)
    want = (rows[plan.places.long()].reshape(2, 3, 40) * w[:, :, None]).sum(1)
    assert torch.allclose(X.combine_experts(rows, plan, w), want, atol=1e-6)


# --------------------------------------------------------------------------------------------------
# The experts' products

PRODUCTS = [(1, 1, 1, 1, 1), (24, 4, 32, 512, 200), (3, 2, 5, 130, 33), (200, 4, 8, 300, 129), (300, 2, 3, 700, 264),
            (64, 8, 130, 128, 64), (700, 3, 4, 1100, 300), (1500, 2, 2, 256, 260), (33, 1, 70, 100, 16)]


@pytest.mark.parametrize("tokens,each,experts,inner,outer", PRODUCTS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
@pytest.mark.parametrize("away,kind", [(0.0, "any"), (0.3, "few"), (0.0, "one")])
def test_linear_experts(gpu, tokens, each, experts, inner, outer, dtype, codes, away, kind):
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.blocks import quantize_blocks
    from tcc_spmm_amd.micro import quantize_micro, quantize_weight_micro
    ids = choices(tokens, each, experts, 3, away, kind=kind)
    plan = X.sort_experts(ids, experts)
    offsets, order, _ = O.plan(ids.cpu().numpy(), experts)
    x = random((tokens, inner), 5, dtype) * random((tokens, 1), 6).exp().to(DTYPES[dtype])
    w, bias = random((experts, outer, inner), 7, spread=inner ** -0.5), random((experts, outer), 8)
    weight = quantize_weight_micro(w)
    xv, wv = row_values(x, codes), weight.dequantize().double().cpu().numpy()
    want, room = np.zeros((tokens * each, outer)), np.zeros((tokens * each, outer))
    bare = want.copy()
    for e in range(experts):
        span = slice(offsets[e], offsets[e + 1])
        mine = xv[order[span] // each]
        bare[span] = mine @ wv[e].T
        want[span] = bare[span] + f64(bias[e])
        room[span] = product_room(mine, wv[e], dtype, codes)
    allowed = (room + 4 * U * np.abs(want)) * 1.01 + rounded(want, dtype)
    y = X.linear_experts(x, weight, plan, bias, by_token=True, codes=FORMATS[codes])
    near(y, want, allowed, "y by token")
    rows = X.gather_experts(x, plan)
    rows[offsets[-1]:] = float("nan")  # rows of no expert count nothing
    sorted_y = X.linear_experts(rows, weight, plan, bias, codes=FORMATS[codes])
    assert torch.equal(sorted_y, y), "a row's result does not depend on where it comes from"
    assert torch.equal(X.linear_experts(cut(x), weight, plan, bias, by_token=True, codes=FORMATS[codes]), y)
    near(X.linear_experts(x, weight, plan, by_token=True, codes=FORMATS[codes]), bare,
         (room + 4 * U * np.abs(bare)) * 1.01 + rounded(bare, dtype), "y without bias")
    assert not y[offsets[-1]:].any()
    coded = (quantize_blocks if codes == "e4m3" else quantize_micro)(x)
    assert torch.equal(X.matmul_experts(coded, weight, plan, bias, by_token=True, dtype=DTYPES[dtype]), y)
    coded = (quantize_blocks if codes == "e4m3" else quantize_micro)(rows)
    assert torch.equal(X.matmul_experts(coded, weight, plan, bias, dtype=DTYPES[dtype]), y)


@pytest.mark.parametrize("tokens,each,experts,inner,outer", [(2100, 3, 5, 500, 600), (1100, 2, 2, 1153, 520), (900, 4, 7, 100, 3000)])
@pytest.mark.parametrize("dtype,codes", [("bf16", "e4m3"), ("f32", "e2m1"), ("f16", "e2m1")])
def test_linear_experts_wide(gpu, tokens, each, experts, inner, outer, dtype, codes):
    """Experts of many rows, which the largest tile takes."""
    test_linear_experts(gpu, tokens, each, experts, inner, outer, dtype, codes, 0.1, "any")


@pytest.mark.parametrize("tokens", [7, 500])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
def test_a_nan_stays_with_its_token_and_its_expert(gpu, tokens, dtype, codes):
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import quantize_weight_micro
    ids = choices(tokens, 2, 5, 1)
    plan = X.sort_experts(ids, 5)
    x, w = random((tokens, 200), 1, dtype), random((5, 150, 200), 2)
    weight = quantize_weight_micro(w)
    clean = X.linear_experts(x, weight, plan, by_token=True, codes=FORMATS[codes])
    x[3, 150], w[2, 10, 5] = float("nan"), float("inf")
    y = X.linear_experts(x, quantize_weight_micro(w), plan, by_token=True, codes=FORMATS[codes])
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[plan.order // 2 == 3] = True
    bad[plan.offsets[2]:plan.offsets[3], 10] = True
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], clean[~bad])


def test_a_plan_of_other_sizes_is_held_to_the_call(gpu):
    """Lists that are no plan: the call ends, within its buffers; rows that some expert is given have its results."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import quantize_weight_micro
    rng = np.random.default_rng(0)
    weight = quantize_weight_micro(random((3, 40, 64), 1))
    for seed in range(4):
        lists = [torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31, n).astype(np.int32)).cuda() for n in (4, 60, 60)]
        plan = X.ExpertPlan(*lists, (30,), 2)
        x = random((30, 64), 1)
        X.linear_experts(x, weight, plan, by_token=True)
        X.gather_experts(x, plan)
        X.combine_experts(random((60, 64), 2), plan)
        X.combine_experts_backward(x, random((60, 64), 2), plan, random((30, 2), 3))
    torch.cuda.synchronize()


# --------------------------------------------------------------------------------------------------
# Under autograd, together


def test_gradients_of_the_layer(gpu):
    """A layer of gated experts and its router's weights, by token: the autograd functions give the gradients of the calls that
    they are made of, and those agree with differences of the layer without quantization of gradients."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.blocks import activation_blocks, activation_blocks_backward, block_activation
    from tcc_spmm_amd.micro import quantize_weight_micro
    tokens, each, count, width, hidden = 50, 2, 6, 96, 64
    plan = X.sort_experts(choices(tokens, each, count, 1, 0.1), count)
    up = quantize_weight_micro(random((count, 2 * hidden, width), 2, spread=0.1), tiles=True, transposed=True)
    down = quantize_weight_micro(random((count, width, hidden), 3, spread=0.1), tiles=True, transposed=True)
    x, weights, dy = random((tokens, width), 4).requires_grad_(), random((tokens, each), 5).requires_grad_(), random((tokens, width), 6)
    h = X.expert_linear(x, up, plan, by_token=True)
    rows = X.expert_linear(block_activation(h, "silu", gated=True), down, plan)
    y = X.expert_combine(rows, plan, weights)
    y.backward(dy)
    with torch.no_grad():
        h2 = X.linear_experts(x, up, plan, by_token=True)
        a2, kept = activation_blocks(h2, "silu", gated=True)
        rows2 = X.linear_experts(a2, down, plan)
        assert torch.equal(y, X.combine_experts(rows2, plan, weights))
        drows, dweights = X.combine_experts_backward(dy, rows2, plan, weights)
        da = X.linear_experts(drows, down.transposed(), plan)
        dh = activation_blocks_backward(da, kept, "silu", gated=True)
        dx = X.combine_experts(X.linear_experts(dh, up.transposed(), plan), plan)
    assert torch.equal(x.grad, dx) and torch.equal(weights.grad, dweights)


def test_gather_and_combine_against_differences(gpu):
    """Both are linear, so differences along a direction are exact but for roundings."""
    from tcc_spmm_amd import experts as X
    plan = X.sort_experts(choices(40, 3, 5, 1, 0.2), 5)
    x, w = random((40, 70), 1).requires_grad_(), random((40, 3), 2).requires_grad_()
    dy = random((40, 70), 3)
    X.expert_combine(X.expert_gather(x, plan), plan, w).backward(dy)
    with torch.no_grad():
        loss = lambda a, b: (X.combine_experts(X.gather_experts(a, plan), plan, b).double() * dy).sum()  # noqa: E731
        for at, grad in ((0, x.grad), (1, w.grad)):
            v = random(grad.shape, 4)
            step = [torch.zeros_like(x), torch.zeros_like(w)]
            step[at] = v
            diff = (loss(x + step[0], w + step[1]) - loss(x - step[0], w - step[1])) / 2
            assert abs((grad.double() * v).sum() - diff) <= 1e-5 * (grad * v).abs().sum()


def test_only_what_is_needed(gpu):
    """Gradients of broadcast outputs and inputs; rows are kept for the weights' gradient alone."""
    from tcc_spmm_amd import experts as X
    plan = X.sort_experts(choices(30, 2, 4), 4)
    rows, w = random((60, 24), 1), random((30, 1), 2).requires_grad_()
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.shape) or t, lambda t: t):
        X.expert_combine(rows.clone().requires_grad_(), plan, w.detach().expand(30, 2)).sum().backward()
    assert all(s == (30, 2) for s in saved)
    X.expert_combine(rows, plan, w.expand(30, 2)).sum().backward()
    want = torch.zeros(30, device="cuda").index_add_(0, plan.order.long() // 2, rows.sum(1))
    assert w.grad.shape == (30, 1) and torch.allclose(w.grad[:, 0], want, atol=1e-4)
    assert not X.expert_combine(rows, plan, w.detach().expand(30, 2)).requires_grad


def test_calls_on_another_stream_and_captured(gpu):
    """A whole layer on another stream, and captured into a graph that is replayed with other choices and tokens."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.blocks import activation_blocks
    from tcc_spmm_amd.micro import quantize_weight_micro
    up = quantize_weight_micro(random((8, 128, 96), 2, spread=0.1), tiles=True, transposed=True)
    down = quantize_weight_micro(random((8, 96, 64), 3, spread=0.1))

    def layer(ids, x, w, stream=None):
        plan = X.sort_experts(ids, 8, stream=stream)
        h = X.linear_experts(x, up, plan, by_token=True, stream=stream)
        a, _ = activation_blocks(h, "silu", gated=True, codes=None, stream=stream)
        rows = X.linear_experts(a, down, plan, stream=stream)
        dx = X.linear_experts(h, up.transposed(), plan, stream=stream)
        return (X.combine_experts(rows, plan, w, stream=stream), X.gather_experts(x, plan, stream=stream), dx,
                *X.combine_experts_backward(x, rows, plan, w, stream=stream))

    for tokens in (40, 3000):
        ids, x, w = choices(tokens, 2, 8, 1), random((tokens, 96), 4, "bf16"), random((tokens, 2), 5)
        want = layer(ids, x, w)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        got = layer(ids, x, w, side)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(ids, x, w)
        for seed, kind in ((11, "any"), (12, "one"), (13, "none"), (14, "few")):
            ids.copy_(choices(tokens, 2, 8, seed, 0.1, kind=kind))
            x.copy_(random((tokens, 96), seed, "bf16"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, layer(ids, x, w)))


def test_two_calls_at_once(gpu):
    """Two streams with one stack of weights, a plan of their own each, sizes that take the widest tile beside single tokens."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import E2M1, quantize_weight_micro
    weight = quantize_weight_micro(random((8, 2048, 1024), 2, spread=0.03))
    given = [(choices(n, 2, 8, n), random((n, 1024), n, "bf16"), random((n, 2), n + 1)) for n in (3001, 24, 2000)]

    def calls(ids, x, w, stream=None):
        plan = X.sort_experts(ids, 8, stream=stream)
        rows = X.linear_experts(x, weight, plan, by_token=True, codes=E2M1, stream=stream)
        return rows, X.combine_experts(rows, plan, w, stream=stream)

    want = [calls(*g) for g in given]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in given]
    for _ in range(5):
        got = [calls(*g, stream) for g, stream in zip(given, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for one, two in zip(got, want) for a, b in zip(one, two))


def test_refusals(gpu):
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import quantize_micro, quantize_weight_micro
    ids = choices(10, 2, 4)
    plan = X.sort_experts(ids, 4)
    x, w = random((10, 64), 1), random((10, 2), 2)
    stack, one = quantize_weight_micro(random((4, 32, 64), 1)), quantize_weight_micro(random((32, 64), 1))
    rows = random((20, 64), 3)
    for call in (lambda: X.sort_experts(ids.float(), 4), lambda: X.sort_experts(ids, 0), lambda: X.sort_experts(ids, 1025),
                 lambda: X.sort_experts(ids[:, :0], 4), lambda: X.sort_experts(ids.cpu(), 4),
                 lambda: X.gather_experts(rows, plan), lambda: X.gather_experts(x.double(), plan),
                 lambda: X.gather_experts(x.cpu(), plan), lambda: X.combine_experts(x, plan),
                 lambda: X.combine_experts(rows, plan, w[:, :1]), lambda: X.combine_experts(rows, plan, w.double()),
                 lambda: X.combine_experts(rows, plan, w.cpu()), lambda: X.combine_experts_backward(x, rows, plan),
                 lambda: X.combine_experts_backward(x, None, plan, w),
                 lambda: X.combine_experts_backward(x, rows, plan, w, need=(False, False)),
                 lambda: X.combine_experts_backward(x, rows.bfloat16(), plan, w),
                 lambda: X.linear_experts(x, one, plan, by_token=True), lambda: X.linear_experts(x, stack, plan),
                 lambda: X.linear_experts(rows, stack, plan, by_token=True),
                 lambda: X.linear_experts(rows[:, :63], stack, plan),
                 lambda: X.linear_experts(rows, stack, plan, torch.zeros(32, device="cuda")),
                 lambda: X.linear_experts(rows, stack, plan, codes=torch.int8),
                 lambda: X.matmul_experts(quantize_micro(x), stack, plan), lambda: X.matmul_experts(quantize_micro(rows), one, plan),
                 lambda: X.matmul_experts(quantize_micro(rows), stack, plan, dtype=torch.float64),
                 lambda: X.matmul_experts(quantize_micro(rows[:, :63]), stack, plan),
                 lambda: X.expert_linear(rows.clone().requires_grad_(), stack, plan),
                 lambda: X.expert_linear(rows, stack, plan, torch.zeros((4, 32), device="cuda", requires_grad=True)),
                 lambda: X.ExpertPlan(plan.offsets, plan.order[:-1], plan.places, (10,), 2),
                 lambda: X.ExpertPlan(plan.offsets.long(), plan.order, plan.places, (10,), 2)):
        with pytest.raises(ValueError):
            call()
