"""What a backward pass of the experts' layers reads besides saved tensors, the plan and the frozen weights: as it was in the
forward pass, or the error that autograd gives for its own."""
import pytest
import torch

from test_gpu_blocks import random
from test_gpu_experts import choices

pytestmark = pytest.mark.gpu


def layers(X, M, inference=False):
    with torch.inference_mode(inference):
        plan = X.sort_experts(choices(20, 2, 4), 4)
        stack = M.quantize_weight_micro(random((4, 40, 64), 3), tiles=True, transposed=True)
    weights = random((20, 2), 4)
    return plan, stack, {"gather": (lambda x: X.expert_gather(x, plan), (20, 64)),
                         "combine": (lambda x: X.expert_combine(x, plan, weights), (40, 64)),
                         "linear": (lambda x: X.expert_linear(x, stack, plan), (40, 64)),
                         "linear by token": (lambda x: X.expert_linear(x, stack, plan, by_token=True), (20, 64))}


@pytest.mark.parametrize("name,changed", [
    *((name, part) for name in ("gather", "combine", "linear", "linear by token") for part in ("offsets", "order", "places")),
    *((name, part) for name in ("linear", "linear by token") for part in ("codes_t", "exponents_t"))])
def test_changed_in_place(gpu, name, changed):
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd import micro as M
    plan, stack, functions = layers(X, M)
    layer, shape = functions[name]
    x = random(shape, 5).requires_grad_()
    y = layer(x)
    target = getattr(stack if changed.endswith("_t") else plan, changed)
    target.copy_(target.clone())
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward(torch.ones_like(y))
    y = layer(x)  # and again, with them as they are now
    y.backward(torch.ones_like(y))


@pytest.mark.parametrize("name", ["gather", "combine", "linear", "linear by token"])
@pytest.mark.parametrize("inference", [False, True])
def test_replaced_and_not_changed(gpu, name, inference):
    """Tensors that a plan or weight object is given later are not the forward pass's; inference tensors are taken."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd import micro as M
    plan, stack, functions = layers(X, M, inference)
    layer, shape = functions[name]
    x = random(shape, 5).requires_grad_()
    y = layer(x)
    dy = random(y.shape, 6)
    want, = torch.autograd.grad(y, x, dy, retain_graph=True)
    other = X.sort_experts(choices(20, 2, 4, 9), 4)
    plan.offsets, plan.order, plan.places = other.offsets, other.order, other.places
    stack.codes_t, stack.exponents_t = stack.codes_t.clone(), torch.zeros_like(stack.exponents_t)
    again, = torch.autograd.grad(y, x, dy)
    assert torch.equal(want, again)


def test_a_stack_without_a_transposed_copy(gpu):
    """Serves tensors that need no gradient, with gradients on."""
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd import micro as M
    plan = X.sort_experts(choices(20, 2, 4), 4)
    stack = M.quantize_weight_micro(random((4, 40, 64), 3))
    y = X.expert_linear(random((40, 64), 1), stack, plan)
    assert not y.requires_grad
