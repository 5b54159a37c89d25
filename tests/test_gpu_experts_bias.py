"""A bias of the experts under autograd: of any type and layout, as micro_linear's."""
import pytest
import torch

from test_gpu_blocks import random
from test_gpu_experts import choices

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("context", [torch.enable_grad, torch.no_grad])
def test_bias_of_any_type_and_layout(gpu, context):
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd.micro import quantize_weight_micro
    plan = X.sort_experts(choices(20, 2, 4), 4)
    stack = quantize_weight_micro(random((4, 40, 64), 1), tiles=True, transposed=True)
    x, full = random((20, 64), 2).requires_grad_(), random((4, 40), 3)
    with context():
        for bias in (full, full.bfloat16(), full.half(), full.t().contiguous().t(), full[:1].expand(4, 40), full.double()):
            got = X.expert_linear(x, stack, plan, bias, by_token=True)
            want = X.linear_experts(x.detach(), stack, plan, bias.float().contiguous(), by_token=True)
            assert torch.equal(got, want) and got.requires_grad == torch.is_grad_enabled()
        with pytest.raises(ValueError, match="bias must be"):
            X.expert_linear(x, stack, plan, full[:, :39], by_token=True)
