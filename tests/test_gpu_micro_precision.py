"""What include/micro.h says about the range of the products, at both ends of it, through every kernel: one product a sum, so that
it shows what a code and its exponent stand for. The value in every output, but in an FP32 one of E4M3 rows the value as bf16
has it: that is the same for exponents of E4M3 blocks of 3 to 246 and of microscaled ones of 0 to 252, and for those of 253 up
to the code 3, which is as far as quantizing goes."""
import numpy as np
import pytest
import torch

import micro_oracle as O
from blocks_oracle import CODES, DTYPES, f64
from test_gpu_blocks_precision import in_bf16
from test_micro_forms import expert_form, product_form

pytestmark = pytest.mark.gpu

EIGHT = np.array([2.0 ** -9, 3 * 2.0 ** -9, 7 * 2.0 ** -9, 2.0 ** -6, 1.0, 1.875, 240.0, 448.0])
FOUR = np.array([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -6.0])
ENDS = [0, 1, 2, 3, 4, 127, 245, 246, 247, 251, 252, 253, 254]


def rows_of(first, e, codes, rows, inner=128):
    """Rows whose last element's code is that of `first`, in turn, and whose others are zeros; all exponents e."""
    from tcc_spmm_amd.blocks import BlockTensor
    from tcc_spmm_amd.micro import E2M1, MicroTensor
    v = np.resize(first, rows)
    steps, at = -(-inner // 128), inner - 1
    if codes == "e4m3":
        code = torch.from_numpy(v.astype(np.float32)).cuda().to(CODES["e4m3"])
        assert np.array_equal(f64(code.float()), v)
        q = torch.zeros((rows, 128 * steps), device="cuda").to(code.dtype)
        q[:, at] = code
        return BlockTensor(q, torch.full((rows, -(-steps // 4) * 4), e, dtype=torch.uint8, device="cuda"), inner)
    code = O.to_codes(v)
    assert np.array_equal(O.of_codes(code), v)
    q = torch.zeros((rows, 64 * steps), device="cuda", dtype=torch.uint8)
    q[:, at // 2] = torch.from_numpy(code << 4 * (at % 2)).cuda()
    return MicroTensor(q.view(E2M1), torch.full((rows, -(-steps // 4) * 16), e, dtype=torch.uint8, device="cuda"), inner)


def weight_of(first, e, outer, inner=128, experts=None):
    from tcc_spmm_amd.micro import MicroWeight
    t = rows_of(first, e, "e2m1", outer, inner)
    if experts is None:
        return MicroWeight(t.codes, t.exponents, inner)
    return MicroWeight(t.codes.view(torch.uint8).expand(experts, -1, -1).contiguous().view(t.codes.dtype),
                       t.exponents.expand(experts, -1, -1).contiguous(), inner)


def check(y, kinds, ones, e, f, exact):
    """y [rows, outer] of rows `kinds` at exponent e and columns `ones` at f."""
    with np.errstate(over="ignore"):
        value = kinds * 2.0 ** (e - 127)
        value = in_bf16(value) if exact else value
        want = np.resize(value, y.shape[0])[:, None] * (np.resize(ones, y.shape[1]) * 2.0 ** (f - 127))[None]
    assert np.array_equal(f64(y), want)


# rows, inner, outer: each kernel of the product
SIZES = {"microTiles32": (16, 4096, 1000), "microTiles64x32": (500, 2900, 1001), "microTiles64": (777, 1001, 1437),
         "microTiles128": (4091, 300, 4099), "microWide": (3900, 600, 4000)}
TAKEN = [("f32", "e4m3", n) for n in list(SIZES)[:3]] + [("bf16", "e4m3", n) for n in SIZES] + \
        [(t, "e2m1", n) for t in ("f32", "bf16") for n in SIZES]


def test_the_sizes_above_take_every_kernel(gpu):
    for dtype, codes, form in TAKEN:
        assert product_form(*SIZES[form], dtype, codes, "matmul") == form


@pytest.mark.parametrize("e", ENDS)
@pytest.mark.parametrize("dtype,codes,form", TAKEN)
def test_values_at_the_ends_of_the_range(gpu, dtype, codes, form, e):
    from tcc_spmm_amd.micro import matmul_micro
    rows, inner, outer = SIZES[form]
    f = min(max(254 - e, 30), 220)  # brings the products back to the middle of the range
    exact = dtype == "f32" and codes == "e4m3"
    # the ends in x
    kinds = EIGHT if codes == "e4m3" else FOUR
    y = matmul_micro(rows_of(kinds, e, codes, rows, inner), weight_of([1.0], f, outer, inner), dtype=DTYPES[dtype])
    check(y, kinds, [1.0], e, f, exact)
    # the ends in the weight
    y = matmul_micro(rows_of([1.0], f, codes, rows, inner), weight_of(FOUR, e, outer, inner), dtype=DTYPES[dtype])
    check(y.t(), FOUR, [1.0], e, f, exact)


@pytest.mark.parametrize("e", ENDS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
def test_a_few_dense_rows(gpu, dtype, codes, e):
    """Through microTokens, which codes x itself: the weight's ends, and FP32 rows near FP32's."""
    from tcc_spmm_amd.micro import E2M1, linear_micro
    assert product_form(4, 128, 64, dtype, codes) == "microTokens"
    kind = CODES["e4m3"] if codes == "e4m3" else E2M1
    f = min(max(254 - e, 30), 220)
    exact = dtype == "f32" and codes == "e4m3"
    x = torch.zeros((4, 128), device="cuda", dtype=DTYPES[dtype])
    x[:, 127] = 2.0 ** (f - 127)  # against the rows' last elements
    check(linear_micro(x, weight_of(FOUR, e, 64), codes=kind).t(), FOUR, [1.0], e, f, exact)
    if 1 <= e <= 253:
        x[:, 127] = 2.0 ** (e - 127)  # a power of two, which both formats hold
        check(linear_micro(x, weight_of([1.0], f, 64), codes=kind), np.array([1.0]), [1.0], e, f, False)


@pytest.mark.parametrize("e", [0, 3, 246, 252, 253])
@pytest.mark.parametrize("tokens,count,inner,outer,dtype,codes,form", [
    (24, 32, 2048, 400, "f32", "e4m3", "microTiles64"), (24, 32, 2048, 400, "bf16", "e4m3", "microTiles64"),
    (6002, 8, 2048, 1000, "f32", "e2m1", "microTiles128"), (6002, 8, 1000, 2048, "bf16", "e4m3", "microWide")])
def test_experts_at_the_ends_of_the_range(gpu, tokens, count, inner, outer, dtype, codes, form, e):
    from tcc_spmm_amd import experts as X
    assert expert_form(tokens, count, inner, outer, dtype, codes) == form
    f = min(max(254 - e, 30), 220)
    plan = X.sort_experts((torch.arange(tokens, device="cuda") % count)[:, None], count)
    weight = weight_of(FOUR, e, outer, inner, count)
    y = X.matmul_experts(rows_of([1.0], f, codes, tokens, inner), weight, plan, by_token=True, dtype=DTYPES[dtype])
    check(y.t(), FOUR, [1.0], e, f, dtype == "f32" and codes == "e4m3")


def test_values_of_weights_that_were_quantized(gpu):
    """FP32 weights whose blocks reach FP32's ends: their products with a one are the values that they stand for."""
    from tcc_spmm_amd.micro import E2M1, linear_micro, quantize_weight_micro
    peaks = np.array([2.0 ** -149, 2.0 ** -130, 6 * 2.0 ** -126, 7 * 2.0 ** -126, 1.5 * 2.0 ** 127, 1.9 * 2.0 ** 127,
                      float(np.finfo(np.float32).max)], np.float32)
    w = torch.zeros((len(peaks), 128))
    w[:, 0] = torch.from_numpy(peaks)
    weight = quantize_weight_micro(w.cuda())
    want = f64(weight.dequantize())[:, 0]
    assert np.array_equal(want, O.quantize(f64(w))[2][:, 0]) and np.isfinite(want).all()
    for rows in (3, 200):
        x = torch.zeros((rows, 128), device="cuda")
        x[:, 0] = 2.0 ** -10
        for kind in (CODES["e4m3"], E2M1):
            y = f64(linear_micro(x, weight, codes=kind))
            scaled, normal = want * 2.0 ** -10, want * 2.0 ** -10 >= 2.0 ** -126
            assert np.array_equal(y[:, normal], np.broadcast_to(scaled[normal], y[:, normal].shape)) and normal.sum() == 3
            assert np.isfinite(y).all()
