"""The block kernels at sizes that pass 32 bits somewhere."""
import pytest
import torch

from blocks_oracle import CODES, DTYPES
from test_blocks_forms import GRADIENTS, PRODUCTS, TYPES, gradient_form, product_form
from test_gpu_blocks import random

pytestmark = pytest.mark.gpu


@pytest.fixture
def room(gpu):
    """Skips where the card has less free memory than the test asks for, in GB; frees what it took."""
    def need(gigabytes):
        torch.cuda.empty_cache()
        if torch.cuda.mem_get_info()[0] < gigabytes * 1e9:
            pytest.skip(f"needs {gigabytes} GB of GPU memory")
    yield need
    torch.cuda.empty_cache()


def test_more_blocks_than_a_launch_takes_threads_for(room):
    """2^28 + 1000 rows of one block, of 16 threads each: more than 2^32 threads. Some rows from each part of the range
    are those of a call on them alone."""
    from tcc_spmm_amd import blocks as B
    room(120)
    rows = (1 << 28) + 1000
    x = torch.randn((rows, 4), device="cuda", dtype=torch.bfloat16)
    parts = [slice(at, at + 500) for at in (0, (1 << 27) - 250, (1 << 28) - 250, rows - 500)]
    kept = B.quantize_blocks(x)
    values = kept.dequantize(torch.bfloat16)
    for p in parts:
        want = B.quantize_blocks(x[p])
        assert torch.equal(kept.codes[p].view(torch.uint8), want.codes.view(torch.uint8))
        assert torch.equal(kept.exponents[p], want.exponents) and torch.equal(values[p], want.dequantize(torch.bfloat16))
    del kept, values
    y, act = B.activation_blocks(x, "silu")
    dx = B.activation_blocks_backward(y, act, "silu")
    for p in parts:
        want, want_act = B.activation_blocks(x[p], "silu")
        assert torch.equal(y[p], want) and torch.equal(act.codes[p], want_act.codes)
        assert torch.equal(dx[p], B.activation_blocks_backward(y[p], want_act, "silu"))


def test_product_of_more_rows_than_small_tiles_have_threads_for(room):
    """2^30 + 300 rows are too many tiles of 64 rows for a launch. Most rows are zeros; the others are those of a product
    of them alone."""
    from tcc_spmm_amd import blocks as B
    room(190)
    rows, outer = (1 << 30) + 300, 8
    codes = torch.zeros((rows, 128), device="cuda", dtype=torch.uint8).view(B.E4M3)
    exponents = torch.full((rows, 4), 127, device="cuda", dtype=torch.uint8)
    weight = B.quantize_weight_blocks(random((outer, 128), 1))
    parts = [slice(at, at + 300) for at in (0, (1 << 29) - 100, rows - 300)]
    for i, p in enumerate(parts):
        some = B.quantize_blocks(random((300, 128), 2 + i))
        codes[p], exponents[p] = some.codes, some.exponents
    y = B.matmul_blocks(B.BlockTensor(codes, exponents, 128), weight)
    for p in parts:
        alone = B.BlockTensor(codes[p].contiguous(), exponents[p].contiguous(), 128)
        # One block is one instruction's sum in every form of the product.
        assert torch.equal(y[p], B.matmul_blocks(alone, weight))
    assert not y[1000:100000].any()


def far(rows, columns, dtype, step=1):
    """Rows so far apart that the last one starts past 2^32 elements, a multiple of `step` from each other."""
    stride = max(columns, -(-(1 << 32) // (rows - 1)) + 8)
    stride = -(-stride // step) * step
    flat = torch.empty((rows - 1) * stride + columns, dtype=DTYPES[dtype], device="cuda")
    return flat.as_strided((rows, columns), (stride, 1))


def moved(t, dtype, step=1):
    """t's values in rows far apart."""
    out = far(*t.shape, dtype, step)
    return out.copy_(t)


ONE_OF_EACH = [p for i, p in enumerate(PRODUCTS) if p[:2] not in {q[:2] for q in PRODUCTS[:i]}
               and (p[1] != "f16" or "Wide" in p[0]) and p[2] > 1]


@pytest.mark.parametrize("form,dtype,rows,inner,outer", ONE_OF_EACH)
def test_rows_far_apart_through_the_layer(room, form, dtype, rows, inner, outer):
    """Row starts of x and y past 2^32 elements: the same bits as from rows side by side."""
    from tcc_spmm_amd import blocks as B
    from tcc_spmm_amd._lib import check, lib
    room(60)
    x, weight, kind = random((rows, inner), 1, dtype), B.quantize_weight_blocks(random((outer, inner), 2)), TYPES[dtype]
    assert product_form(rows, inner, outer, dtype) == form
    y, kept = B.linear_blocks(x, weight, keep=True)
    got, got_kept = B.linear_blocks(moved(x, dtype), weight, keep=True)
    assert torch.equal(got, y) and torch.equal(got_kept.codes.view(torch.uint8), kept.codes.view(torch.uint8))
    to, args = far(rows, outer, dtype), (weight.codes.data_ptr(), weight.exponents.data_ptr(), None)
    stream = torch.cuda.current_stream().cuda_stream
    check(lib().tcc_linear_blocks(x.data_ptr(), inner, kind, *args, to.data_ptr(), to.stride(0), got_kept.codes.data_ptr(),
                                  got_kept.exponents.data_ptr(), rows, inner, outer, None, 0, stream))
    assert torch.equal(to, y)
    want = B.matmul_blocks(kept, weight, dtype=DTYPES[dtype])
    to.zero_()
    check(lib().tcc_matmul_blocks(kept.codes.data_ptr(), kept.exponents.data_ptr(), *args, to.data_ptr(), to.stride(0), kind,
                                  rows, inner, outer, stream))
    assert torch.equal(to, want)


@pytest.mark.parametrize("form,splits,dtype,rows,inner,outer", [g for g in GRADIENTS if g[3] > 520 and g[2] != "f16"] +
                         [g for g in GRADIENTS if g[3] <= 520][:3])
def test_rows_far_apart_through_the_gradient(room, form, splits, dtype, rows, inner, outer):
    from tcc_spmm_amd import blocks as B
    room(40)
    kept, dy = B.quantize_blocks(random((rows, inner), 1, dtype)), random((rows, outer), 2, dtype)
    apart = moved(dy, dtype, 8)
    assert gradient_form(apart.data_ptr(), apart.stride(0), dtype, rows, inner, outer) == (form, splits)
    for got, want in zip(B.weight_grad_blocks(apart, kept), B.weight_grad_blocks(dy, kept)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,codes", [("f32", "int8"), ("bf16", "e4m3")])
def test_rows_far_apart_through_blocks_and_activations(room, dtype, codes):
    from tcc_spmm_amd import blocks as B
    from tcc_spmm_amd._lib import check, lib
    room(60)
    rows, width, kind, code = 1003, 300, TYPES[dtype], B._CODES[CODES[codes]]
    stream = torch.cuda.current_stream().cuda_stream
    x, dy = random((rows, 2 * width), 1, dtype), random((rows, width), 2, dtype)
    kept = B.quantize_blocks(x, CODES[codes])
    got = B.quantize_blocks(moved(x, dtype), CODES[codes])
    assert torch.equal(got.codes.view(torch.uint8), kept.codes.view(torch.uint8))
    to = far(rows, 2 * width, dtype)
    check(lib().tcc_dequantize_blocks(kept.codes.data_ptr(), kept.exponents.data_ptr(), code, to.data_ptr(), to.stride(0),
                                      kind, rows, 2 * width, stream))
    assert torch.equal(to, kept.dequantize(DTYPES[dtype]))
    for gated, x in ((True, x), (False, x[:, :width])):
        y, act = B.activation_blocks(x, "silu", gated=gated, codes=CODES[codes])
        dx = B.activation_blocks_backward(dy, act, "silu", gated=gated)
        apart = moved(x, dtype)
        got, got_act = B.activation_blocks(apart, "silu", gated=gated, codes=CODES[codes])
        assert torch.equal(got, y) and torch.equal(got_act.codes.view(torch.uint8), act.codes.view(torch.uint8))
        assert torch.equal(B.activation_blocks_backward(moved(dy, dtype), act, "silu", gated=gated), dx)
        to = far(rows, width, dtype)
        check(lib().tcc_activation_blocks(apart.data_ptr(), apart.stride(0), kind, 0, gated, to.data_ptr(), to.stride(0), None,
                                          None, code, rows, width, stream))
        assert torch.equal(to, y)
        del apart, to
        to = far(*dx.shape, dtype)
        check(lib().tcc_activation_blocks_backward(dy.data_ptr(), width, kind, act.codes.data_ptr(), act.exponents.data_ptr(),
                                                   code, 0, gated, to.data_ptr(), to.stride(0), rows, width, stream))
        assert torch.equal(to, dx)
        del to


def test_codes_past_32_bits(room):
    """17,000,000 rows of 256: codes, kept ones among them, and the elements of x and y pass 2^32. The last rows are
    those of calls on them alone."""
    from tcc_spmm_amd import blocks as B
    room(90)
    rows, tail = 17_000_000, 20_000
    assert (rows - tail) * 256 > 1 << 32
    x = torch.randn((rows, 256), device="cuda", dtype=torch.bfloat16)
    weight = B.quantize_weight_blocks(random((256, 256), 2))
    assert product_form(rows, 256, 256, "bf16") == product_form(tail, 256, 256, "bf16") == "multiplyRows"
    y, kept = B.linear_blocks(x, weight, keep=True)
    want, want_kept = B.linear_blocks(x[-tail:], weight, keep=True)
    same = lambda a, b: torch.equal(a.codes[-tail:].view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(  # noqa: E731
        a.exponents[-tail:], b.exponents)
    assert torch.equal(y[-tail:], want) and same(kept, want_kept) and same(B.quantize_blocks(x), want_kept)
    assert torch.equal(kept.dequantize(torch.bfloat16)[-tail:], want_kept.dequantize(torch.bfloat16))
    # Two blocks are two instructions' sums in the same order, whatever the tile.
    for dtype in (torch.bfloat16, torch.float32):
        assert torch.equal(B.matmul_blocks(kept, weight, dtype=dtype)[-tail:], B.matmul_blocks(want_kept, weight, dtype=dtype))
    # A gradient that is zero but for the last rows is theirs, but for the order of the sums.
    dy = torch.zeros((rows, 40), device="cuda", dtype=torch.bfloat16)
    dy[-tail:] = random((tail, 40), 3, "bf16")
    got, alone = B.weight_grad_blocks(dy, kept), B.weight_grad_blocks(dy[-tail:], want_kept)
    terms = dy[-tail:].float().abs().t() @ want_kept.dequantize().abs(), dy[-tail:].float().abs().sum(0)
    for a, b, t in zip(got, alone, terms):
        assert ((a - b).abs() <= 2 * (tail / 4 + 64) * 2.0 ** -24 * t * 1.01).all()
    del y, dy, kept
    for gated in (False, True):
        given = x.view(rows // 2, 512) if gated else x
        a, act = B.activation_blocks(given, "silu", gated=gated)
        dx = B.activation_blocks_backward(a, act, "silu", gated=gated)
        some = tail // 2 if gated else tail
        b, want_act = B.activation_blocks(given[-some:], "silu", gated=gated)
        assert torch.equal(a[-some:], b) and same(act, want_act)
        assert torch.equal(dx[-some:], B.activation_blocks_backward(b, want_act, "silu", gated=gated))
        del a, act, dx


def test_weight_past_32_bits(room):
    """A weight of 66,000 x 65,536, whose elements, codes and gradient pass 2^32: its last columns of y and rows of the
    gradient are those of its last rows alone. Whole numbers, so that sums are exact in any order."""
    from tcc_spmm_amd import blocks as B
    room(120)
    outer, inner, rows, last = 66_000, 65_536, 70, 128 * 515
    assert last * inner > 1 << 32
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randint(-2, 3, (outer, inner), generator=gen, device="cuda", dtype=torch.int8).float()
    x = torch.randint(-1, 2, (rows, inner), generator=gen, device="cuda").float()
    weight, end = B.quantize_weight_blocks(w), B.quantize_weight_blocks(w[last:])
    assert torch.equal(weight.codes[last:].view(torch.uint8), end.codes.view(torch.uint8))
    assert torch.equal(weight.codes_t[:, last:].float()[:, :outer - last], end.codes_t.float()[:, :outer - last])
    for dtype in (torch.float32, torch.bfloat16):
        y = B.linear_blocks(x.to(dtype), weight)
        assert torch.equal(y[:, last:], B.linear_blocks(x.to(dtype), end))
    del w, y
    dy, kept = torch.zeros((rows, outer), device="cuda"), B.quantize_blocks(x)
    dy[:, last:] = torch.randint(-3, 4, (rows, outer - last), generator=gen, device="cuda").float()
    assert torch.equal(B.linear_blocks(dy, weight.transposed()), B.linear_blocks(dy[:, last:], end.transposed()))
    for d in (dy, dy.bfloat16()):
        dw, db = B.weight_grad_blocks(d, kept)
        want, want_db = B.weight_grad_blocks(d[:, last:], kept)
        assert torch.equal(dw[last:], want) and torch.equal(db[last:], want_db) and not dw[:last].any()
        del dw
