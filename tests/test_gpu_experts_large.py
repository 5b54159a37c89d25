"""Microscaled layers and experts at sizes that pass 32 bits somewhere."""
import pytest
import torch

from test_gpu_blocks import random
from test_gpu_blocks_large import room  # noqa: F401  (a fixture)
from test_gpu_experts import choices
from test_gpu_micro import FORMATS

pytestmark = pytest.mark.gpu


def test_quantize_past_32_bits(room):  # noqa: F811
    """2^28 + 1000 rows of one run, of 16 threads each: more threads than a dimension of a launch takes; x passes 2^32 bytes."""
    from tcc_spmm_amd.micro import quantize_micro
    room(60)
    rows = (1 << 28) + 1000
    x = torch.randn((rows, 12), device="cuda", dtype=torch.bfloat16)
    kept = quantize_micro(x)
    for at in (0, (1 << 27) - 250, (1 << 28) - 250, rows - 500):
        part = slice(at, at + 500)
        want = quantize_micro(x[part])
        assert torch.equal(kept.codes[part].view(torch.uint8), want.codes.view(torch.uint8))
        assert torch.equal(kept.exponents[part], want.exponents)
    values = kept.dequantize(torch.bfloat16)
    assert torch.equal(values[-500:], want.dequantize(torch.bfloat16))


@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
def test_product_past_32_bits(room, codes):  # noqa: F811
    """x, its codes and y pass 2^32 bytes; the last rows are those of a call on them alone, of as many tiles' kind."""
    from tcc_spmm_amd.micro import linear_micro, quantize_weight_micro
    room(120)
    x = torch.randn((17_000_000, 512), device="cuda", dtype=torch.bfloat16)
    weight = quantize_weight_micro(random((300, 512), 2))
    y = linear_micro(x, weight, codes=FORMATS[codes])
    for part in (slice(0, 70_000), slice(8_400_000, 8_470_000), slice(-70_000, None)):
        want = linear_micro(x[part], weight, codes=FORMATS[codes])
        # other numbers of rows may take other tiles, whose 16-bit sums differ in the last place
        assert (y[part].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
        assert (y[part] != want).float().mean() < 0.01


def test_product_of_more_rows_than_small_tiles_have_threads_for(room):  # noqa: F811
    """2^30 + 300 rows are too many tiles of 64 rows for a launch. Most rows are zeros; the others are those of a product
    of them alone."""
    from tcc_spmm_amd import micro as M
    room(140)
    rows, outer = (1 << 30) + 300, 8
    codes = torch.zeros((rows, 64), device="cuda", dtype=torch.uint8)
    exponents = torch.full((rows, 16), 127, device="cuda", dtype=torch.uint8)
    weight = M.quantize_weight_micro(random((outer, 128), 1))
    parts = [slice(at, at + 300) for at in (0, (1 << 29) - 100, rows - 300)]
    for i, p in enumerate(parts):
        some = M.quantize_micro(random((300, 128), 2 + i))
        codes[p], exponents[p] = some.codes.view(torch.uint8), some.exponents
    y = M.matmul_micro(M.MicroTensor(codes.view(M.E2M1), exponents, 128), weight)
    for p in parts:
        want = M.matmul_micro(M.MicroTensor(codes[p].view(M.E2M1), exponents[p], 128), weight)
        # products of 4-bit codes are added exactly as far as FP32 goes, in whatever tile
        assert (y[p].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
    assert not y[1000:2000].any()


def test_weight_stack_past_32_bits(room):  # noqa: F811
    """Experts whose stacked codes pass 2^32 bytes, in tiles, with the transposed copies: the last expert's rows are those of
    that expert alone."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import quantize_weight_micro
    room(120)
    w = torch.empty((130, 8192, 8192), device="cuda", dtype=torch.bfloat16)
    for e in range(130):
        w[e] = torch.randn((8192, 8192), device="cuda", dtype=torch.bfloat16) * 0.02
    stack = quantize_weight_micro(w, tiles=True, transposed=True)
    assert stack.codes.numel() > 1 << 32
    ids = torch.full((40, 1), 129, device="cuda")
    x = random((40, 8192), 1, "bf16")
    one = quantize_weight_micro(w[129:], tiles=True, transposed=True)
    del w
    for many, single in ((stack, one), (stack.transposed(), one.transposed())):
        got = X.linear_experts(x, many, X.sort_experts(ids, 130))
        want = X.linear_experts(x, single, X.sort_experts(ids - 129, 1))
        assert torch.equal(got, want) or (got.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()


def test_rows_past_32_bits(room):  # noqa: F811
    """Gathered rows of more than 2^32 bytes, there and back."""
    from tcc_spmm_amd import experts as X
    room(120)
    tokens, each, width = 300_000, 8, 2048
    ids = choices(tokens, each, 64, 1)
    plan = X.sort_experts(ids, 64)
    x = torch.randn((tokens, width), device="cuda", dtype=torch.bfloat16)
    rows = X.gather_experts(x, plan)
    assert rows.numel() > 1 << 32
    for r in (0, rows.shape[0] // 2, rows.shape[0] - 1):
        assert torch.equal(rows[r], x[plan.order[r].long() // each])
    w = torch.rand((tokens, each), device="cuda")
    y = X.combine_experts(rows, plan, w / w.sum(1, keepdim=True))
    assert (y.float() - x.float()).abs().max() <= 2.0 ** -7 * x.float().abs().max()
    drows, dw = X.combine_experts_backward(x, rows, plan, w)
    last = plan.places[-each:].long()
    assert torch.equal(drows[last], (w[-1, :, None] * x[-1].float()).to(torch.bfloat16))
    dot = (x[-1].double() * x[-1].double()).sum()
    assert ((dw[-1].double() - dot).abs() <= 1e-5 * dot).all()


def test_tokens_whose_codes_pass_31_bits(room):  # noqa: F811
    """By token, more bytes of codes than the kernels reach by 32 bits: the rows are gathered first."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import quantize_weight_micro
    room(60)
    tokens, inner = 270_000, 8192
    x = torch.randn((tokens, inner), device="cuda", dtype=torch.bfloat16)
    weight = quantize_weight_micro(random((2, 24, inner), 1, spread=0.02))
    ids = (torch.arange(tokens, device="cuda") % 2)[:, None]
    plan = X.sort_experts(ids, 2)
    y = X.linear_experts(x, weight, plan, by_token=True)
    want = X.linear_experts(X.gather_experts(x, plan), weight, plan)
    assert torch.equal(y, want)
