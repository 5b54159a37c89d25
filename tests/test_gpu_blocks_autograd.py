"""What block_linear, block_activation and BlockLinear do, and leave out, in the modes that torch calls them in."""
import numpy as np
import pytest
import torch

from blocks_oracle import DTYPES, f64
from test_gpu_blocks import U, cut, near, random

pytestmark = pytest.mark.gpu


@pytest.fixture
def calls(monkeypatch):
    """(function, what it keeps or makes besides the result) of each call that the layers make."""
    from tcc_spmm_amd import blocks as B
    seen = []
    linear, activation, quantize = B.linear_blocks, B.activation_blocks, B.quantize_weight_blocks

    def see_linear(*args, keep=False, **more):
        seen.append(("linear", keep))
        return linear(*args, keep=keep, **more)

    def see_activation(*args, codes=B.INT8, **more):
        seen.append(("activation", codes is not None))
        return activation(*args, codes=codes, **more)

    def see_quantize(w, transposed=True, **more):
        seen.append(("weight", transposed))
        return quantize(w, transposed, **more)

    monkeypatch.setattr(B, "linear_blocks", see_linear)
    monkeypatch.setattr(B, "activation_blocks", see_activation)
    monkeypatch.setattr(B, "quantize_weight_blocks", see_quantize)
    return seen


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_nothing_is_kept_without_gradients(gpu, calls, mode):
    from tcc_spmm_amd import blocks as B
    layer, x = B.BlockLinear(100, 64).cuda(), random((300, 100), 1).requires_grad_()
    want = layer(x)
    act = B.block_activation(want, "silu")
    assert calls == [("weight", True), ("linear", True), ("activation", True)]
    calls.clear()
    with mode():
        y = layer(x)
        a = B.block_activation(y.clone().requires_grad_() if mode is torch.no_grad else y, "silu")
    assert torch.equal(y, want) and torch.equal(a, act)
    assert calls == [("weight", False), ("linear", False), ("activation", False)]


def test_an_activation_without_gradient_may_keep_nothing(gpu):
    from tcc_spmm_amd import blocks as B
    x = random((20, 64), 1)
    assert torch.equal(B.block_activation(x, "gelu", codes=None), B.activation_blocks(x, "gelu")[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bias_of_any_layout(gpu, dtype):
    """A column of a wider tensor and one number for all, with their gradients."""
    from tcc_spmm_amd import blocks as B
    x, w, dy = random((30, 70), 1), random((40, 70), 2), random((30, 40), 3)
    for make in (lambda t: t[:, 1], lambda t: t[0, :1].expand(40)):
        base = random((40, 3), 4, dtype).requires_grad_()
        plain = make(base.detach().clone()).contiguous().requires_grad_()
        want, got = B.block_linear(x, w, plain), B.block_linear(x, w, make(base))
        assert torch.equal(got, want)
        with torch.no_grad():
            assert torch.equal(B.block_linear(x, w, make(base)), want)
        got.backward(dy)
        want.backward(dy)
        grad = torch.zeros_like(base)
        if make(base).stride(0):
            grad[:, 1] = plain.grad
        else:
            grad[0, 0] = plain.grad.sum()
        assert torch.equal(base.grad, grad)


@pytest.mark.parametrize("rows,outer", [(0, 40), (1, 1), (7, 5), (300, 47), (65, 128), (1000, 129), (5003, 520), (40000, 64),
                                        (9000, 4104)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_bias_gradient_alone(gpu, rows, outer, dtype):
    """Sums of n numbers through the MFMA, which adds at least four at once, in a few splits: (n / 4 + 64) roundings of
    2^-24 of the magnitudes' sum. NaN beside a slice and in the other columns stays there."""
    from tcc_spmm_amd.blocks import linear_blocks_backward, weight_grad_blocks
    dy = random((rows, outer), 1, dtype)
    want, terms = f64(dy).sum(0), np.abs(f64(dy)).sum(0)
    for d in (dy, cut(dy)):
        dw, db = weight_grad_blocks(d, None)
        assert dw is None
        near(db, want, (rows / 4 + 64) * U * terms, "db")
        assert torch.equal(db, weight_grad_blocks(d, None)[1]), "repeated calls give the same bits"
        assert torch.equal(linear_blocks_backward(d, None, None, need=(False, False, True))[2], db)
    if rows and outer > 1:
        dy[0, 1] = float("nan")
        bad = weight_grad_blocks(dy, None)[1]
        assert bad[1].isnan() and bad.isnan().sum() == 1


def test_a_frozen_weight_keeps_nothing_of_its_input(gpu, calls):
    from tcc_spmm_amd import blocks as B
    layer, x, dy = B.BlockLinear(100, 64).cuda(), random((300, 100), 1), random((300, 64), 2)
    layer(x).backward(dy)
    want = layer.bias.grad.clone()
    layer.zero_grad()
    layer.weight.requires_grad_(False)
    calls.clear()
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        y = layer(x)
    assert calls == [("weight", False), ("linear", False)] and not saved
    y.backward(dy)
    # Both are FP32 sums of the same 300 numbers, in an order of their own.
    assert layer.weight.grad is None
    assert ((layer.bias.grad - want).abs() <= 2 * (300 / 4 + 64) * U * dy.abs().sum(0)).all()


@pytest.mark.parametrize("autocast", ["bf16", "f16"])
def test_under_autocast(gpu, autocast):
    """FP32 rows go through the layers in autocast's type, there and back; parameters and x have gradients of their own
    type; within a disabled region nothing is cast."""
    from tcc_spmm_amd import blocks as B
    layer, x = B.BlockLinear(100, 128).cuda(), random((300, 100), 1).requires_grad_()
    dy = random((300, 64), 2, autocast)

    def step(x):
        y = B.block_activation(layer(x), "silu", gated=True)
        assert y.dtype == DTYPES[autocast]
        y.backward(dy)
        grads = [p.grad.clone() for p in layer.parameters()]
        layer.zero_grad()
        return y, grads

    half = x.detach().to(DTYPES[autocast]).requires_grad_()
    want, want_grads = step(half)
    with torch.autocast("cuda", DTYPES[autocast]):
        got, grads = step(x)
        with torch.no_grad():
            assert layer(x).dtype == DTYPES[autocast]
        with torch.autocast("cuda", enabled=False):
            assert layer(x).dtype == torch.float32
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))
    assert x.grad.dtype == torch.float32 and torch.equal(x.grad, half.grad.float())
    assert layer(x).dtype == torch.float32
