"""The experts' products of tokens that are codes already, of more bytes than the kernels reach by 32 bits: in the library's C
entry refused, here gathered first."""
import pytest
import torch

from test_gpu_blocks import random
from test_gpu_blocks_large import room  # noqa: F401  (a fixture)
from test_gpu_experts import choices
from test_gpu_micro import FORMATS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes,lead", [("e4m3", (3, 90_000)), ("e2m1", (530_000,))])
def test_codes_of_tokens_past_31_bits(room, codes, lead):  # noqa: F811
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.blocks import quantize_blocks
    from tcc_spmm_amd.micro import quantize_micro, quantize_weight_micro
    room(80)
    inner = 8192
    x = torch.randn((*lead, inner), device="cuda", dtype=torch.bfloat16)
    weight = quantize_weight_micro(random((3, 24, inner), 1, spread=0.02))
    plan = X.sort_experts(choices(x.numel() // inner, 1, 3, 2, 0.1).reshape(*lead, 1), 3)
    coded = (quantize_blocks if codes == "e4m3" else quantize_micro)(x)
    assert coded.codes.numel() >= 1 << 31
    y = X.matmul_experts(coded, weight, plan, by_token=True)
    assert torch.equal(y, X.linear_experts(x, weight, plan, by_token=True, codes=FORMATS[codes]))
    assert not y[plan.offsets[-1]:].any() and y[:plan.offsets[-1]].any(1).all()


@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
def test_gathered_codes_are_the_rows_codes(gpu, codes):
    """Every byte, NaN patterns of bf16 among them, of rows with an odd number of blocks."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.blocks import BlockTensor
    from tcc_spmm_amd.micro import MicroTensor
    plan = X.sort_experts(choices(50, 3, 6, 1, 0.2).reshape(5, 10, 3), 6)
    pitch, exponent_pitch, kind = (384, 4, BlockTensor) if codes == "e4m3" else (192, 16, MicroTensor)
    gen = torch.Generator(device="cuda").manual_seed(0)
    parts = [torch.randint(0, 256, (50, n), generator=gen, device="cuda", dtype=torch.uint8) for n in (pitch, exponent_pitch)]
    moved = X._gather_codes(kind(parts[0].view(FORMATS[codes]), parts[1], 300), plan)
    assert type(moved) is kind and moved.columns == 300 and moved.codes.dtype == FORMATS[codes]
    here, token = plan.offsets[-1], plan.order.long() // 3
    for got, given in zip((moved.codes.view(torch.uint8), moved.exponents), parts):
        assert torch.equal(got[:here], given[token][:here]) and not got[here:].any()
