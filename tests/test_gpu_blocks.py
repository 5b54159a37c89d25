"""The 8-bit block kernels against their definitions in 64 bits (tests/blocks_oracle.py).

Codes and exponents have to be equal. What the other tolerances allow for:
- an FP32 sum of n terms through the MFMA, which adds at least four products at once: (n / 4 + 16) roundings
  of 2^-24 of the sum of the terms' magnitudes;
- the 8-bit MFMA, which adds the 128 products of a block with at least 17 bits below the largest:
  128 * 2^-17 of it for each block;
- the exponential: 2 roundings, and one of its argument, 1.5 * 2^-24 of it in the result;
- one rounding to the output's type.
"""
import numpy as np
import pytest
import torch

import blocks_oracle as O
from blocks_oracle import CODES, DTYPES, ROUNDING, f64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def random(shape, seed, dtype="f32", spread=1.0, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * spread).to(DTYPES[dtype]).to(device)


def cut(t, left=3, right=2):
    """The same values as a slice of wider rows that hold NaN beside it."""
    wide = torch.full((t.shape[0], t.shape[1] + left + right), float("nan"), dtype=t.dtype, device=t.device)
    wide[:, left:left + t.shape[1]] = t
    return wide[:, left:left + t.shape[1]]


def near(got, want, allowed, what):
    got = f64(got)
    assert got.shape == want.shape, what
    finite = np.isfinite(want)
    assert np.array_equal(finite, np.isfinite(got)), f"{what}: finite elsewhere"
    off = np.abs(got - want)[finite]
    room = np.broadcast_to(allowed, want.shape)[finite]
    assert (off <= room).all(), f"{what}: off by {off.max()} where {room[off.argmax()]} is allowed"


def rounded(want, dtype):
    """Room for one rounding to the type, subnormals of f16 included."""
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0
    return ROUNDING[dtype] * np.abs(want) + tiny


# --------------------------------------------------------------------------------------------------
# The format


def check_blocks(blocks, x, codes):
    q, e, values = O.quantize(f64(x), codes)
    assert np.array_equal(blocks.exponents.cpu().numpy()[:, :e.shape[1]], e)
    assert (blocks.exponents.cpu().numpy()[:, e.shape[1]:] == 127).all()
    assert np.array_equal(f64(blocks.codes.float()), q)
    assert np.array_equal(f64(blocks.dequantize()), values, equal_nan=True)


@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 384), (64, 640), (130, 1001),
                                          (1000, 100), (2, 4100)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_quantize_rows(gpu, rows, columns, dtype, codes):
    from tcc_spmm_amd.blocks import quantize_blocks
    x = random((rows, columns), rows + columns, dtype, 3.0)
    check_blocks(quantize_blocks(x, CODES[codes]), x, codes)
    check_blocks(quantize_blocks(cut(x), CODES[codes]), x, codes)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_quantize_scales(gpu, codes):
    """Peaks at, just below and just above the largest code times a power of two, over the FP32 range; zeros;
    subnormals; ties."""
    from tcc_spmm_amd.blocks import quantize_blocks
    top = O.TOP[codes]
    peaks = []
    for p in (-149, -140, -127, -126, -120, -20, -1, 0, 1, 60, 100, 119):
        for m in (top, np.nextafter(np.float32(top), np.float32(0)), np.nextafter(np.float32(top), np.float32(1e9)), 1.0, 1.5):
            peaks.append(np.float32(m * 2.0 ** p))
    x = np.random.default_rng(0).uniform(-1, 1, (len(peaks) + 2, 128)).astype(np.float32) * 0.9
    x[:len(peaks)] *= np.array(peaks, np.float32)[:, None]
    x[:len(peaks), 5] = peaks
    x[len(peaks)] = 0.0
    x[len(peaks) + 1] = np.arange(128) * 0.5 if codes == "int8" else np.arange(128) * 1.0
    x[len(peaks) + 1, -1] = top
    t = torch.from_numpy(x[np.isfinite(x).all(1)]).cuda()
    check_blocks(quantize_blocks(t, CODES[codes]), t, codes)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinities_and_nan_stay_in_their_block(gpu, codes, dtype):
    from tcc_spmm_amd.blocks import quantize_blocks
    x = random((6, 300), 1, dtype)
    x[0, 3], x[1, 130], x[2, 299], x[3, 0] = float("inf"), float("-inf"), float("nan"), torch.finfo(x.dtype).min
    blocks = quantize_blocks(x, CODES[codes])
    check_blocks(blocks, x, codes)
    values = f64(blocks.dequantize())
    assert np.isnan(values[0, :128]).all() and np.isfinite(values[0, 128:]).all()
    assert np.isfinite(values[3:]).all()


@pytest.mark.parametrize("outer,inner", [(1, 1), (128, 128), (127, 129), (300, 1001), (513, 64), (64, 1100)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantize_weight(gpu, outer, inner, dtype):
    from tcc_spmm_amd.blocks import quantize_weight_blocks
    w = random((outer, inner), outer, dtype)
    if outer > 200:
        w[:128, :128] = 0.0
        w[130, 5] = float("nan")
    q, e, _ = O.quantize_tiles(f64(w))
    for weight in (quantize_weight_blocks(w), quantize_weight_blocks(cut(w), transposed=True)):
        assert np.array_equal(f64(weight.codes.float()), q)
        assert np.array_equal(weight.exponents.cpu().numpy()[:, :e.shape[1]], e)
        t = np.zeros((inner, -(-outer // 128) * 128))
        t[:, :outer] = q[:, :inner].T
        assert np.array_equal(f64(weight.codes_t.float()), t)
        assert np.array_equal(weight.exponents_t.cpu().numpy()[:, :e.shape[0]], e.T)
    assert quantize_weight_blocks(w, transposed=False).codes_t is None


# --------------------------------------------------------------------------------------------------
# The product


def product_room(x, w, dtype):
    """Room for the sums of x w^T before the rounding to the output's type."""
    terms = np.abs(x) @ np.abs(w).T
    room = (x.shape[1] / 4 + 16) * U * terms
    if dtype != "f32":
        for k in range(0, x.shape[1], 128):
            room = room + 128 * 2.0 ** -17 * np.abs(x[:, k:k + 128]).max(1)[:, None] * np.abs(w[:, k:k + 128]).max(1)[None]
    return room


SHAPES = [(1, 1, 1), (1, 128, 16), (1, 4096, 130), (3, 100, 77), (16, 512, 64), (17, 1001, 200), (40, 640, 129),
          (64, 256, 300), (65, 128, 128), (129, 129, 127), (200, 1300, 257), (300, 384, 513), (513, 1024, 640),
          (700, 2048, 1000), (1111, 96, 47), (5000, 128, 256), (24, 4096, 1000), (32, 2900, 513), (5, 2048, 2050)]


@pytest.mark.parametrize("rows,inner,outer,dtype", [(4090, 200, 4100, "bf16"), (4091, 300, 4099, "f16"),
                                                    (3900, 600, 4000, "bf16"), (4096, 1024, 4096, "bf16")])
def test_linear_wide(gpu, rows, inner, outer, dtype):
    """Products of many tiles, which the largest tile takes: one block more than its pairs, ragged edges."""
    test_linear(gpu, rows, inner, outer, dtype)


@pytest.mark.parametrize("rows,inner,outer", [(65, 4500, 100), (130, 1500, 200), (200, 8300, 33), (511, 1024, 65)])
def test_linear_f32_few_tiles(gpu, rows, inner, outer):
    """FP32 products of more than 64 rows that are too few tiles: 64 rows at a time, the last ones ragged."""
    test_linear(gpu, rows, inner, outer, "f32")


@pytest.mark.parametrize("rows,inner,outer", [(8192, 128, 256), (20011, 47, 256), (10007, 256, 47), (9001, 300, 100),
                                              (8200, 512, 130), (16385, 129, 3), (8199, 7, 40), (16391, 300, 100),
                                              (16390, 509, 47), (16401, 512, 130), (17000, 250, 256)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_linear_narrow(gpu, rows, inner, outer, dtype):
    """Many rows through a layer whose weight fits in LDS, and the same layer where blocks are given."""
    test_linear(gpu, rows, inner, outer, dtype)


@pytest.mark.parametrize("rows,inner,outer", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_linear(gpu, rows, inner, outer, dtype):
    from tcc_spmm_amd.blocks import linear_blocks, matmul_blocks, quantize_blocks, quantize_weight_blocks
    x = random((rows, inner), 5, dtype) * random((rows, 1), 6).exp().to(DTYPES[dtype])
    w, bias = random((outer, inner), 7, spread=inner ** -0.5), random((outer,), 8)
    weight = quantize_weight_blocks(w)
    xv, wv = O.quantize(f64(x))[2], O.quantize_tiles(f64(w))[2]
    room = product_room(xv, wv, dtype)
    for b in (None, bias):
        want = xv @ wv.T + (0 if b is None else f64(b))
        allowed = (room + 4 * U * np.abs(want)) * 1.01 + rounded(want, dtype)
        near(linear_blocks(x, weight, b), want, allowed, "y")
    y, kept = linear_blocks(cut(x), weight, bias, keep=True)
    near(y, want, allowed, "y of a slice")
    check_blocks(kept, x, "e4m3")
    again = matmul_blocks(quantize_blocks(x), weight, bias, dtype=DTYPES[dtype])
    near(again, want, allowed, "y of blocks")


def test_linear_leading_dimensions_and_layouts(gpu):
    from tcc_spmm_amd.blocks import linear_blocks, quantize_weight_blocks
    x, w = random((4, 5, 70), 1, "bf16"), random((33, 70), 2)
    weight = quantize_weight_blocks(w, transposed=False)
    y = linear_blocks(x, weight)
    assert y.shape == (4, 5, 33)
    flat = x.reshape(20, 70)
    assert torch.equal(y.reshape(20, 33), linear_blocks(flat, weight))
    assert torch.equal(linear_blocks(flat.t().contiguous().t(), weight), y.reshape(20, 33))
    one = flat[:1].expand(20, 70)
    assert torch.equal(linear_blocks(one, weight), linear_blocks(one.contiguous(), weight))
    assert linear_blocks(x[:0], weight).shape == (0, 5, 33)
    assert torch.equal(quantize_weight_blocks(w.t().contiguous().t()).codes.float(), weight.codes.float())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [5, 200])
def test_linear_with_nan_rows(gpu, rows, dtype):
    """A row with an infinity or a NaN gives a row of NaN and leaves the others alone."""
    from tcc_spmm_amd.blocks import linear_blocks, quantize_weight_blocks
    x, w = random((rows, 300), 1, dtype), random((150, 300), 2)
    weight = quantize_weight_blocks(w)
    clean = linear_blocks(x, weight)
    x[1, 7], x[3, 299] = float("nan"), float("inf")
    y = linear_blocks(x, weight)
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[[1, 3]] = True
    assert y[bad].isnan().all() and torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 150])
def test_given_exponents_over_their_range(gpu, rows, dtype):
    """Blocks that a caller made: scales from 2^-60 to 2^60, and NaN."""
    from tcc_spmm_amd.blocks import BlockTensor, BlockWeight, matmul_blocks
    rng = np.random.default_rng(0)
    q = torch.from_numpy(rng.integers(-8, 9, (rows, 512)).astype(np.float32)).cuda().to(CODES["e4m3"])
    w = torch.from_numpy(rng.integers(-8, 9, (200, 512)).astype(np.float32)).cuda().to(CODES["e4m3"])
    e = torch.from_numpy(rng.integers(67, 188, (rows, 4)).astype(np.uint8)).cuda()
    f = torch.from_numpy(rng.integers(97, 158, (2, 4)).astype(np.uint8)).cuda()
    e[1, 2] = 255
    xv = f64(q.float()) * np.repeat(O.scale(e.cpu().numpy()), 128, 1)
    wv = f64(w.float()) * np.repeat(np.repeat(O.scale(f.cpu().numpy()), 128, 0)[:200], 128, 1)
    want = xv @ wv.T
    y = matmul_blocks(BlockTensor(q, e, 512), BlockWeight(w, f, 512), dtype=DTYPES[dtype])
    near(y, want, product_room(xv, wv, dtype) + 4 * U * np.abs(want) + rounded(want, dtype), "y")


@pytest.mark.parametrize("rows,outer", [(3, 40), (20, 300), (100, 200), (600, 500), (4096, 4100)])
@pytest.mark.parametrize("columns", [128, 640, 1153])
def test_exponents_past_the_last_block_do_not_count(gpu, rows, outer, columns):
    """Bytes that fill up a row of exponents may be anything, 255 among them."""
    from tcc_spmm_amd.blocks import matmul_blocks, quantize_blocks, quantize_weight_blocks, weight_grad_blocks
    x, weight = quantize_blocks(random((rows, columns), 1)), quantize_weight_blocks(random((outer, columns), 2))
    dy = random((rows, outer), 3, "bf16")
    want = matmul_blocks(x, weight), weight_grad_blocks(dy, x)[0]
    blocks = -(-columns // 128)
    x.exponents[:, blocks:] = 255
    weight.exponents[:, blocks:] = 255
    assert torch.equal(matmul_blocks(x, weight), want[0]) and torch.equal(weight_grad_blocks(dy, x)[0], want[1])
    assert matmul_blocks(x, weight, dtype=torch.float32).isfinite().all()


def test_offsets_past_32_bits(gpu):
    """Nine million rows of 256: x, y and the kept codes pass 2^31, x 2^32 bytes; the last rows are those of a call
    on them alone."""
    from tcc_spmm_amd import blocks as B
    x = torch.randn((9_000_000, 256), device="cuda", dtype=torch.bfloat16)
    weight = B.quantize_weight_blocks(random((64, 256), 2))
    y, kept = B.linear_blocks(x, weight, keep=True)
    tail, tail_kept = B.linear_blocks(x[-9000:], weight, keep=True)
    assert torch.equal(y[-9000:], tail) and torch.equal(kept.codes[-9000:].float(), tail_kept.codes.float())
    assert torch.equal(B.matmul_blocks(kept, weight)[-9000:], tail)
    a, act = B.activation_blocks(x, "silu", gated=True)
    b, tail_act = B.activation_blocks(x[-9000:], "silu", gated=True)
    assert torch.equal(a[-9000:], b) and torch.equal(act.codes[-18000:], tail_act.codes)
    assert torch.equal(B.activation_blocks_backward(a, act, gated=True)[-9000:],
                       B.activation_blocks_backward(b, tail_act, gated=True))
    dy = torch.zeros((9_000_000, 64), device="cuda", dtype=torch.bfloat16)
    dy[-9000:] = random((9000, 64), 3, "bf16")
    dw, _ = B.weight_grad_blocks(dy, kept)
    want, _ = B.weight_grad_blocks(dy[-9000:], tail_kept)
    assert (dw - want).abs().max() <= 1e-4 * want.abs().max()


# --------------------------------------------------------------------------------------------------
# Gradients of the layer


@pytest.mark.parametrize("rows,inner,outer", [(1, 1, 1), (1, 300, 140), (7, 130, 47), (64, 128, 128), (65, 200, 300),
                                              (500, 129, 127), (1000, 512, 384), (5003, 128, 200), (20000, 100, 64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_linear_backward(gpu, rows, inner, outer, dtype):
    from tcc_spmm_amd.blocks import linear_blocks, linear_blocks_backward, quantize_weight_blocks
    x, dy = random((rows, inner), 1, dtype), random((rows, outer), 2, dtype, 1e-2)
    weight = quantize_weight_blocks(random((outer, inner), 3))
    _, kept = linear_blocks(x, weight, keep=True)
    xv, wv = O.quantize(f64(x))[2], O.quantize_tiles(f64(random((outer, inner), 3)))[2]
    gv, g = O.quantize(f64(dy))[2], f64(dy)
    want = {"dx": gv @ wv, "dw": g.T @ xv, "db": g.sum(0)}
    room = {"dx": product_room(gv, wv.T, dtype) + rounded(gv @ wv, dtype),
            "dw": (rows / 4 + 64) * U * (np.abs(g).T @ np.abs(xv)), "db": (rows / 4 + 64) * U * np.abs(g).sum(0)}
    for d in (dy, cut(dy)):
        got = dict(zip(("dx", "dw", "db"), linear_blocks_backward(d, kept, weight)))
        for name in want:
            near(got[name], want[name], room[name] * 1.01 + 1e-30, name)
        again = dict(zip(("dx", "dw", "db"), linear_blocks_backward(d, kept, weight)))
        assert all(torch.equal(got[n], again[n]) for n in want), "repeated calls give the same bits"
    only = linear_blocks_backward(dy, kept, weight, need=(False, True, False))
    assert only[0] is None and only[2] is None and torch.equal(only[1], got["dw"])


@pytest.mark.parametrize("rows,inner,outer", [(1500, 2048, 4096), (1030, 4000, 4104), (4000, 1000, 520)])
def test_weight_gradient_large(gpu, rows, inner, outer):
    """Gradients of many tiles, which the largest tile takes, and of few, over many rows."""
    from tcc_spmm_amd.blocks import quantize_blocks, weight_grad_blocks
    x, dy = random((rows, inner), 1, "bf16"), random((rows, outer), 2, "bf16", 1e-2)
    xv, g = O.quantize(f64(x))[2], f64(dy)
    dw, db = weight_grad_blocks(dy, quantize_blocks(x))
    near(dw, g.T @ xv, (rows / 4 + 64) * U * (np.abs(g).T @ np.abs(xv)) + 1e-30, "dw")
    near(db, g.sum(0), (rows / 4 + 64) * U * np.abs(g).sum(0) + 1e-30, "db")
    assert torch.equal(weight_grad_blocks(dy, quantize_blocks(x), bias=False)[0], dw)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,inner,outer", [(100, 130, 40), (300, 256, 136)])
def test_weight_gradient_of_infinities(gpu, rows, inner, outer, dtype):
    """An infinity or a NaN in dy stays in its column of the gradient, an infinity an infinity where its row of x
    has no zero; the largest finite numbers stay finite."""
    from tcc_spmm_amd.blocks import quantize_blocks, weight_grad_blocks
    x, dy = random((rows, inner), 1, dtype).abs() + 0.5, random((rows, outer), 2, dtype)
    dy[3, 1], dy[5, 2], dy[7, 3] = float("inf"), float("-inf"), float("nan")
    top = torch.finfo(DTYPES[dtype]).max
    dy[:, 4] = 0.0
    dy[9, 4] = top if dtype == "f16" else top / 4
    xv, g = O.quantize(f64(x))[2], f64(dy)
    dw, db = weight_grad_blocks(dy, quantize_blocks(x))
    want = torch.from_numpy(np.nan_to_num(g, nan=0, posinf=0, neginf=0).T @ xv)
    assert (dw[1] == float("inf")).all() and (dw[2] == float("-inf")).all() and dw[3].isnan().all()
    assert db[1] == float("inf") and db[2] == float("-inf") and db[3].isnan()
    rest = [i for i in range(outer) if i not in (1, 2, 3)]
    terms = np.abs(np.nan_to_num(g, nan=0, posinf=0, neginf=0)).T @ xv
    near(dw[rest], want[rest].numpy(), (rows / 4 + 64) * U * terms[rest], "dw")


def test_weight_gradient_of_no_rows(gpu):
    from tcc_spmm_amd.blocks import quantize_blocks, weight_grad_blocks
    dw, db = weight_grad_blocks(torch.empty((0, 30), device="cuda"), quantize_blocks(torch.empty((0, 50), device="cuda")))
    assert dw.shape == (30, 50) and not dw.any() and not db.any()


def test_gradients_against_differences(gpu):
    """The layer is linear in the values of its blocks, so differences of the loss sum(dy * y) along a direction
    are the gradients' products with it."""
    from tcc_spmm_amd.blocks import linear_blocks, linear_blocks_backward, quantize_weight_blocks
    x, w, dy = random((200, 150), 1), random((90, 150), 2), random((200, 90), 3)
    weight = quantize_weight_blocks(w)
    _, kept = linear_blocks(x, weight, keep=True)
    dx, dw, db = map(f64, linear_blocks_backward(dy, kept, weight))
    xv, wv, g, gv = O.quantize(f64(x))[2], O.quantize_tiles(f64(w))[2], f64(dy), O.quantize(f64(dy))[2]
    rng = np.random.default_rng(4)
    loss = lambda a, b, c, d: (d * (a @ b.T + c)).sum()  # noqa: E731
    for grad, at in ((dx, 0), (dw, 1), (db, 2)):
        v = rng.standard_normal(grad.shape)
        step = [np.zeros_like(xv), np.zeros_like(wv), np.zeros(90)]
        step[at] = v
        d = gv if at == 0 else g  # the input gradient is that of the quantized output gradient
        diff = (loss(xv + step[0], wv + step[1], step[2], d) - loss(xv - step[0], wv - step[1], -step[2], d)) / 2
        assert abs((grad * v).sum() - diff) <= 1e-5 * np.abs(grad * v).sum()


# --------------------------------------------------------------------------------------------------
# Activations


def value_room(kind, x, y):
    room = (10 + 3 * O.argument(kind, x)) * U * np.abs(y)
    return room + 4 * U * np.abs(x) if kind == "gelu" else room


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (3, 127), (50, 129), (7, 1000), (260, 384)])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype,codes", [("f32", "int8"), ("f32", "e4m3"), ("bf16", "int8"), ("f16", "e4m3")])
def test_activation(gpu, rows, width, kind, gated, dtype, codes):
    from tcc_spmm_amd.blocks import activation_blocks, activation_blocks_backward
    x = random((rows, 2 * width if gated else width), 1, dtype, 2.0)
    dy = random((rows, width), 2, dtype)
    xd, g = f64(x), f64(dy)
    value = O.activation(kind, xd[:, :width])[0]
    factor = xd[:, width:] if gated else 1.0
    for given in (x, cut(x)):
        y, kept = activation_blocks(given, kind, gated=gated, codes=CODES[codes])
        want = value * factor
        near(y, want, value_room(kind, xd[:, :width], value) * np.abs(factor) + 2 * U * np.abs(want) +
             rounded(want, dtype) + 1e-37, "y")
        check_blocks(kept, x.reshape(-1, width), codes)
    values = O.quantize(xd.reshape(-1, width), codes)[2].reshape(rows, -1)
    gate = values[:, :width]
    value, slope, terms = O.activation(kind, gate)
    slope_room = (16 + 4 * O.argument(kind, gate)) * U * terms
    if gated:
        up = values[:, width:]
        want = np.concatenate([g * up * slope, g * value], 1)
        room = np.concatenate([np.abs(g * up) * slope_room, np.abs(g) * value_room(kind, gate, value)], 1)
    else:
        want, room = g * slope, np.abs(g) * slope_room
    for given in (dy, cut(dy)):
        dx = activation_blocks_backward(given, kept, kind, gated=gated)
        near(dx, want, room + 4 * U * np.abs(want) + rounded(want, dtype) + 1e-37, "dx")
    assert activation_blocks(x, kind, gated=gated, codes=None)[1] is None


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_activation_far_from_zero_and_empty(gpu, kind):
    """Large magnitudes neither overflow nor lose the limits f(x) = x and f(x) = 0; rows of none."""
    from tcc_spmm_amd.blocks import activation_blocks, activation_blocks_backward
    x = torch.tensor([[-1e30, -1e4, -200.0, -88.0, -0.0, 0.0, 88.0, 200.0, 1e4, 1e30]], device="cuda")
    y, kept = activation_blocks(x, kind)
    want = np.where(f64(x) > 0, f64(x), 0.0)
    near(y, want, 1e-6 * want + 1e-30, "y")
    dx = f64(activation_blocks_backward(torch.ones_like(x), kept, kind))
    assert np.isfinite(dx).all()
    y, kept = activation_blocks(x[:0], kind)
    assert y.shape == (0, 10) and activation_blocks_backward(y, kept, kind).shape == (0, 10)


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_slopes_against_differences(gpu, kind):
    from tcc_spmm_amd.blocks import activation_blocks, activation_blocks_backward
    x = torch.linspace(-6, 6, 256, device="cuda")[None]
    _, kept = activation_blocks(x, kind)
    at, h = f64(kept.dequantize()), 1e-4
    slope = (O.activation(kind, at + h)[0] - O.activation(kind, at - h)[0]) / (2 * h)
    dx = f64(activation_blocks_backward(torch.ones_like(x), kept, kind))
    # the difference's own error is h^2 / 6 times a third derivative below 2; the kernel's a few roundings
    assert np.abs(dx - slope).max() <= h * h + 64 * U


# --------------------------------------------------------------------------------------------------
# Streams, autograd, training


def test_calls_on_another_stream(gpu):
    from tcc_spmm_amd import blocks as B
    x, w, dy = random((300, 256), 1, "bf16"), random((128, 256), 2), random((300, 128), 3, "bf16")
    weight = B.quantize_weight_blocks(w)
    y, kept = B.linear_blocks(x, weight, keep=True)
    grads = B.linear_blocks_backward(dy, kept, weight)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    weight2 = B.quantize_weight_blocks(w, stream=side)
    y2, kept2 = B.linear_blocks(x, weight2, keep=True, stream=side)
    grads2 = B.linear_blocks_backward(dy, kept2, weight2, stream=side)
    side.synchronize()
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_graph_capture_replays(gpu):
    from tcc_spmm_amd import blocks as B
    x, w = random((777, 300), 1, "bf16"), random((200, 300), 2)
    dy = random((777, 200), 3, "bf16")
    weight = B.quantize_weight_blocks(w)

    def step():
        y, kept = B.linear_blocks(x, weight, keep=True)
        a, act = B.activation_blocks(y, "silu")
        return (y, a, *B.linear_blocks_backward(B.activation_blocks_backward(dy, act, "silu"), kept, weight))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (11, 12, 13):
        x.copy_(random((777, 300), seed, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_layer_under_autograd(gpu):
    """BlockLinear and block_activation give the gradients of the calls that they are made of."""
    from tcc_spmm_amd import blocks as B
    torch.manual_seed(0)
    layer = B.BlockLinear(96, 2 * 80).cuda()
    x = random((3, 50, 96), 1).requires_grad_()
    y = B.block_activation(layer(x), "gelu", gated=True)
    y.sum().backward()
    weight = B.quantize_weight_blocks(layer.weight.detach())
    h, kept = B.linear_blocks(x.detach(), weight, layer.bias.detach(), keep=True)
    want, act = B.activation_blocks(h, "gelu", gated=True)
    dh = B.activation_blocks_backward(torch.ones_like(want), act, "gelu", gated=True)
    dx, dw, db = B.linear_blocks_backward(dh, kept, weight)
    assert torch.equal(y, want) and torch.equal(x.grad, dx)
    assert torch.equal(layer.weight.grad, dw) and torch.equal(layer.bias.grad, db)
    frozen, bias = layer.serving()
    assert torch.equal(B.linear_blocks(x.detach(), frozen, bias), h)


def test_what_autograd_keeps(gpu):
    """Of a layer and a gated activation, autograd holds a byte an element and the exponents, not x."""
    from tcc_spmm_amd import blocks as B
    layer = B.BlockLinear(256, 512).cuda()
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        B.block_activation(layer(random((1000, 256), 1).requires_grad_()), "silu", gated=True)
    assert all(t.element_size() == 1 for t in saved)
    # the layer's input, the activation's input of 2 x 256, and the transposed weight
    assert sum(t.numel() for t in saved) == 1000 * (256 + 4) + 2000 * (256 + 4) + 256 * 512 + 2 * 4


# --------------------------------------------------------------------------------------------------
# Refusals


def test_refusals(gpu):
    from tcc_spmm_amd import blocks as B
    x, w = random((8, 64), 1), random((32, 64), 2)
    weight = B.quantize_weight_blocks(w)
    kept = B.quantize_blocks(x)
    for call in (lambda: B.linear_blocks(random((8, 65), 1), weight), lambda: B.linear_blocks(x.double(), weight),
                 lambda: B.linear_blocks(x.cpu(), weight), lambda: B.linear_blocks(x, weight, torch.zeros(31, device="cuda")),
                 lambda: B.linear_blocks(x, weight, torch.zeros(32, device="cuda", dtype=torch.bfloat16)),
                 lambda: B.matmul_blocks(B.quantize_blocks(x, torch.int8), weight),
                 lambda: B.matmul_blocks(kept, B.quantize_weight_blocks(random((32, 63), 1))),
                 lambda: B.weight_grad_blocks(random((7, 32), 1), kept),
                 lambda: B.weight_grad_blocks(random((8, 32), 1), B.quantize_blocks(x, torch.int8)),
                 lambda: B.linear_blocks_backward(random((8, 32), 1), kept, B.quantize_weight_blocks(w, transposed=False)),
                 lambda: B.activation_blocks(x, "relu"), lambda: B.activation_blocks(x[:, :63], gated=True),
                 lambda: B.activation_blocks(x, codes=torch.uint8),
                 lambda: B.activation_blocks_backward(x, B.quantize_blocks(x[:7])),
                 lambda: B.quantize_blocks(x, torch.float16), lambda: B.dequantize_blocks(kept, torch.float64)):
        with pytest.raises(ValueError):
            call()
