"""The differentiable layers where no_grad leaves something on: forward mode, which they do not have and have to refuse, and
tracing, whose graph has to hold the layer."""
import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_blocks import random
from test_gpu_experts import choices

pytestmark = pytest.mark.gpu


def layers():
    """Functions of one tensor, with its shape."""
    from tcc_spmm_amd import blocks as B
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd import micro as M
    w, bias = random((40, 64), 1).requires_grad_(), random((40,), 2)
    plan = X.sort_experts(choices(20, 2, 4), 4)
    stack = M.quantize_weight_micro(random((4, 40, 64), 3))
    weights = random((20, 2), 4)
    held = w.detach()
    return {"micro_linear": (lambda x: M.micro_linear(x, held, bias), (20, 64)),
            "block_linear": (lambda x: B.block_linear(x, held, bias), (20, 64)),
            "block_activation": (lambda x: B.block_activation(x, gated=True), (20, 64)),
            "block_activation, nothing kept": (lambda x: B.block_activation(x, codes=None), (20, 64)),
            "expert_gather": (lambda x: X.expert_gather(x, plan), (20, 64)),
            "expert_combine": (lambda x: X.expert_combine(x, plan, weights), (40, 64)),
            "expert_linear": (lambda x: X.expert_linear(x, stack, plan, by_token=True), (20, 64)),
            # parameters that require a gradient, whose layers keep nothing without one
            "micro_linear, w": (lambda x: M.micro_linear(x, w, bias), (20, 64)),
            "block_linear, w": (lambda x: B.block_linear(x, w, bias), (20, 64))}


NAMES = ["micro_linear", "block_linear", "block_activation", "block_activation, nothing kept", "expert_gather",
         "expert_combine", "expert_linear", "micro_linear, w", "block_linear, w"]


def test_every_layer_is_below(gpu):
    assert list(layers()) == NAMES


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(gpu, name):
    layer, shape = layers()[name]
    x, tangent = random(shape, 5), random(shape, 6)
    with torch.no_grad():
        want = layer(x)
    for context in (torch.enable_grad, torch.no_grad):
        with forward_ad.dual_level(), context():
            with pytest.raises(NotImplementedError, match="forward mode"):
                layer(forward_ad.make_dual(x, tangent))
            assert torch.equal(layer(x), want)  # a tensor without a tangent is any other
    with torch.no_grad(), forward_ad.dual_level():
        # what requires a gradient is refused nothing that it is given outside
        assert torch.equal(layer(x.clone().requires_grad_()), want)


@pytest.mark.parametrize("name", [n for n in NAMES if not n.endswith(", w")])
def test_a_trace_holds_the_layer(gpu, name):
    layer, shape = layers()[name]
    with torch.no_grad():
        traced = torch.jit.trace(layer, (random(shape, 5),), check_trace=False)
        for seed in (7, 8):
            x = random(shape, seed)
            assert torch.equal(traced(x), layer(x))
