"""The kernels of microscaled 4-bit layers against their definitions in 64 bits (tests/micro_oracle.py).

Codes and exponents have to be equal. What the other tolerances allow for:
- an FP32 sum of n terms through the MFMA, which adds at least four products at once: (n / 4 + 16) roundings of 2^-24 of
  the sum of the terms' magnitudes. That holds for products of two 4-bit codes in every type, since they are multiples of
  a quarter and at most 36, eight bits that the MFMA adds whole;
- E4M3 rows in 16-bit types: the 8-bit MFMA cuts each of 8 products off 13 bits below the power of two of the largest, less
  than 2^-13 of the magnitude of the largest for each of the other 7;
- one rounding to the output's type.
"""
import numpy as np
import pytest
import torch

import blocks_oracle as B8
import micro_oracle as O
from blocks_oracle import DTYPES, f64
from test_gpu_blocks import U, cut, near, random, rounded

pytestmark = pytest.mark.gpu

FORMATS = {"e4m3": torch.float8_e4m3fn, "e2m1": torch.float4_e2m1fn_x2}


def raw(codes) -> np.ndarray:
    return codes.view(torch.uint8).cpu().numpy()


def check_micro(codes, exponents, columns, want):
    q, e, _ = want
    assert np.array_equal(raw(codes), O.pack(q))
    assert np.array_equal(exponents.cpu().numpy(), O.place(e))


def row_values(x, codes):
    return O.quantize(f64(x))[2] if codes == "e2m1" else B8.quantize(f64(x))[2]


def product_room(x, w, dtype, codes):
    """Room for the sums of x w^T before the rounding to the output's type."""
    terms = np.abs(x) @ np.abs(w).T
    room = (x.shape[1] / 4 + 16) * U * terms
    return room + 7 * 2.0 ** -13 * terms if codes == "e4m3" and dtype != "f32" else room


# --------------------------------------------------------------------------------------------------
# The format


@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 32), (3, 31), (5, 33), (17, 128), (64, 129), (130, 1001), (1000, 100),
                                          (2, 4100), (9, 512), (4, 513)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantize_rows(gpu, rows, columns, dtype):
    from tcc_spmm_amd.micro import quantize_micro
    x = random((rows, columns), rows + columns, dtype, 3.0)
    want = O.quantize(f64(x))
    for given in (x, cut(x)):
        got = quantize_micro(given)
        check_micro(got.codes, got.exponents, columns, want)
        assert np.array_equal(f64(got.dequantize()), want[2])
        for out in ("bf16", "f16"):
            assert torch.equal(got.dequantize(DTYPES[out]), got.dequantize().to(DTYPES[out]))


def test_quantize_scales(gpu):
    """Peaks at, just below and just above the largest code times a power of two, over the FP32 range; zeros; subnormals;
    every tie between two codes."""
    from tcc_spmm_amd.micro import quantize_micro
    peaks = []
    for p in (-149, -140, -128, -127, -126, -120, -20, -1, 0, 1, 60, 100, 124, 125):
        for m in (6.0, np.nextafter(np.float32(6), np.float32(0)), np.nextafter(np.float32(6), np.float32(9)), 1.0, 1.5, 7.0,
                  7.99):
            with np.errstate(over="ignore"):
                peaks.append(np.float32(np.float64(m) * 2.0 ** p))
    peaks.append(np.finfo(np.float32).max)
    x = np.random.default_rng(0).uniform(-1, 1, (len(peaks) + 2, 64)).astype(np.float32) * 0.9
    with np.errstate(invalid="ignore", over="ignore"):
        x[:len(peaks)] *= np.array(peaks, np.float32)[:, None]
    x[:len(peaks), 5] = peaks
    x[len(peaks)] = 0.0
    x[len(peaks) + 1] = np.concatenate([np.arange(-31, 1) * 0.25, np.arange(0, 32) * 0.125])
    x[len(peaks) + 1, [0, 63]] = 6.0
    t = torch.from_numpy(x[np.isfinite(x).all(1)]).cuda()
    want = O.quantize(f64(t))
    got = quantize_micro(t)
    check_micro(got.codes, got.exponents, 64, want)
    assert np.array_equal(f64(got.dequantize()), want[2]) and np.isfinite(want[2]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_infinities_and_nan_stay_in_their_block(gpu, dtype):
    from tcc_spmm_amd.micro import quantize_micro
    x = random((6, 300), 1, dtype)
    x[0, 3], x[1, 130], x[2, 299], x[3, 0] = float("inf"), float("-inf"), float("nan"), torch.finfo(x.dtype).min
    want = O.quantize(f64(x))
    got = quantize_micro(x)
    check_micro(got.codes, got.exponents, 300, want)
    values = f64(got.dequantize())
    assert np.array_equal(values, want[2], equal_nan=True)
    assert np.isnan(values[0, :32]).all() and np.isfinite(values[0, 32:]).all() and np.isfinite(values[3:]).all()


@pytest.mark.parametrize("experts,outer,inner", [(None, 1, 1), (None, 32, 32), (None, 31, 33), (None, 128, 128), (None, 300, 1001),
                                                 (None, 513, 64), (None, 64, 1100), (3, 40, 70), (2, 129, 515)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantize_weight(gpu, experts, outer, inner, dtype):
    from tcc_spmm_amd.micro import quantize_weight_micro
    shape = (outer, inner) if experts is None else (experts, outer, inner)
    w = random(shape, outer, dtype)
    if outer > 200:
        w[:32, :64] = 0.0
        w[130, 5] = float("nan")
    stack = f64(w).reshape(-1, outer, inner)
    by_row = quantize_weight_micro(w)
    assert by_row.codes_t is None and by_row.experts == experts and by_row.rows == outer
    for given in (w, cut(w) if experts is None else w.transpose(1, 2).contiguous().transpose(1, 2)):
        tiles, alone = quantize_weight_micro(given, tiles=True, transposed=True), quantize_weight_micro(given, tiles=True)
        assert alone.codes_t is None
        assert np.array_equal(raw(alone.codes), raw(tiles.codes)) and torch.equal(alone.exponents, tiles.exponents)
        parts = [t.reshape(-1, *t.shape[-2:]) for t in (by_row.codes, by_row.exponents, tiles.codes, tiles.exponents,
                                                        tiles.codes_t, tiles.exponents_t)]
        for i, one in enumerate(stack):
            check_micro(parts[0][i], parts[1][i], inner, O.quantize(one))
            q, e, values = O.quantize_tiles(one)
            check_micro(parts[2][i], parts[3][i], inner, (q, e, values))
            blocks = -(-outer // 32)
            t = np.zeros((inner, -(-outer // 128) * 128), np.uint8)
            t[:, :outer] = q[:, :inner].T
            check_micro(parts[4][i], parts[5][i], outer, (t, np.repeat(e[::32].T, 32, 0)[:inner, :blocks], None))
            back = tiles.dequantize().reshape(-1, outer, inner)[i]
            turned = tiles.transposed().dequantize().reshape(-1, inner, outer)[i]
            assert np.array_equal(f64(back), values, equal_nan=True)
            assert np.array_equal(f64(turned), values.T, equal_nan=True)


def test_a_weight_from_elsewhere(gpu):
    """Codes two a byte and exponents in the order of their blocks, as others keep them, reordered on the way in."""
    from tcc_spmm_amd.micro import E2M1, MicroWeight, quantize_weight_micro
    w = random((70, 1024), 1)
    q, e, values = O.quantize(f64(w))
    codes, natural = torch.from_numpy(O.pack(q)).cuda(), torch.from_numpy(e).cuda()
    exponents = natural.reshape(70, -1, 4, 4).transpose(2, 3).reshape(70, -1).contiguous()
    weight = MicroWeight(codes.view(E2M1), exponents, 1024)
    assert np.array_equal(f64(weight.dequantize()), values)
    assert torch.equal(exponents, quantize_weight_micro(w).exponents)


# --------------------------------------------------------------------------------------------------
# The product

SHAPES = [(1, 1, 1), (1, 128, 16), (1, 4096, 130), (3, 100, 77), (4, 1001, 50), (5, 513, 33), (16, 512, 64), (17, 1001, 200),
          (40, 640, 129), (64, 256, 300), (65, 128, 128), (129, 129, 127), (200, 1300, 257), (300, 384, 513), (513, 1024, 640),
          (700, 2048, 1000), (1111, 96, 47), (3000, 128, 256), (24, 4096, 1000), (32, 2900, 513), (5, 2048, 2050),
          (100, 16, 3000), (1500, 200, 2100), (2049, 1100, 2100), (70, 4500, 100)]


@pytest.mark.parametrize("rows,inner,outer", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
def test_linear(gpu, rows, inner, outer, dtype, codes):
    from tcc_spmm_amd.blocks import quantize_blocks
    from tcc_spmm_amd.micro import linear_micro, matmul_micro, quantize_micro, quantize_weight_micro
    x = random((rows, inner), 5, dtype) * random((rows, 1), 6).exp().to(DTYPES[dtype])
    w, bias = random((outer, inner), 7, spread=inner ** -0.5), random((outer,), 8)
    weight = quantize_weight_micro(w)
    xv, wv = row_values(x, codes), O.quantize(f64(w))[2]
    room = product_room(xv, wv, dtype, codes)
    for b in (None, bias):
        want = xv @ wv.T + (0 if b is None else f64(b))
        allowed = (room + 4 * U * np.abs(want)) * 1.01 + rounded(want, dtype)
        near(linear_micro(x, weight, b, codes=FORMATS[codes]), want, allowed, "y")
    coded = (quantize_blocks if codes == "e4m3" else quantize_micro)(x)
    if codes == "e4m3":
        y, kept = linear_micro(cut(x), weight, bias, keep=True)
        assert torch.equal(kept.codes.float(), coded.codes.float()) and torch.equal(kept.exponents, coded.exponents)
    else:
        y = linear_micro(cut(x), weight, bias, codes=FORMATS[codes])
    near(y, want, allowed, "y of a slice")
    near(matmul_micro(coded, weight, bias, dtype=DTYPES[dtype]), want, allowed, "y of coded rows")


@pytest.mark.parametrize("rows,inner,outer", [(4090, 200, 4100), (4091, 300, 4099), (3900, 600, 4300), (4097, 1153, 4000)])
@pytest.mark.parametrize("dtype,codes", [("bf16", "e4m3"), ("f16", "e4m3"), ("f32", "e2m1"), ("bf16", "e2m1"), ("f16", "e2m1")])
def test_linear_wide(gpu, rows, inner, outer, dtype, codes):
    """Products of many tiles, which the largest tile takes: odd and even numbers of its steps, ragged edges."""
    test_linear(gpu, rows, inner, outer, dtype, codes)


@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
def test_linear_leading_dimensions_and_layouts(gpu, codes):
    from tcc_spmm_amd.micro import linear_micro, quantize_weight_micro
    x, w, kind = random((4, 5, 70), 1, "bf16"), random((33, 70), 2), FORMATS[codes]
    weight = quantize_weight_micro(w)
    y = linear_micro(x, weight, codes=kind)
    assert y.shape == (4, 5, 33)
    flat = x.reshape(20, 70)
    assert torch.equal(y.reshape(20, 33), linear_micro(flat, weight, codes=kind))
    assert torch.equal(linear_micro(flat.t().contiguous().t(), weight, codes=kind), y.reshape(20, 33))
    one = flat[:1].expand(20, 70)
    assert torch.equal(linear_micro(one, weight, codes=kind), linear_micro(one.contiguous(), weight, codes=kind))
    assert linear_micro(x[:0], weight, codes=kind).shape == (0, 5, 33)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows", [4, 40, 200, 2500])
def test_linear_with_nan_rows(gpu, rows, dtype, codes):
    """A row with an infinity or a NaN gives a row of NaN and leaves the others alone."""
    from tcc_spmm_amd.micro import linear_micro, quantize_weight_micro
    x, w = random((rows, 300), 1, dtype), random((2000, 300), 2)
    weight = quantize_weight_micro(w)
    clean = linear_micro(x, weight, codes=FORMATS[codes])
    x[1, 7], x[3, 299] = float("nan"), float("inf")
    y = linear_micro(x, weight, codes=FORMATS[codes])
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[[1, 3]] = True
    assert y[bad].isnan().all() and torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("codes", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows,outer", [(2, 200), (150, 200), (1500, 2100)])
def test_given_exponents_over_their_range(gpu, rows, outer, dtype, codes):
    """Blocks that a caller made: scales from 2^-60 to 2^60 and NaN, of rows and of weights, and bytes past the last block,
    which may be anything, 255 among them."""
    from tcc_spmm_amd import blocks, micro
    rng = np.random.default_rng(0)
    columns = 700  # 22 blocks: six steps, the last of two blocks
    def coded(n, low, high):
        q = rng.integers(0, 16, (n, 768)).astype(np.uint8)
        q[:, columns:] = 0
        e = rng.integers(low, high, (n, 22)).astype(np.uint8)
        return q, e
    def kept(q, e, kind):
        return kind(torch.from_numpy(O.pack(q)).cuda().view(micro.E2M1), torch.from_numpy(O.place(e, 255)).cuda(), columns)
    wq, we = coded(outer, 97, 158)
    we[7, 3] = 255
    wv = (O.of_codes(wq[:, :704]) * np.repeat(B8.scale(we), 32, 1))[:, :columns]
    if codes == "e2m1":
        xq, xe = coded(rows, 67, 188)
        xe[1, 21] = 255
        xv = (O.of_codes(xq[:, :704]) * np.repeat(B8.scale(xe), 32, 1))[:, :columns]
        x = kept(xq, xe, micro.MicroTensor)
    else:
        q = torch.from_numpy(rng.integers(-8, 9, (rows, 768)).astype(np.float32)).cuda()
        q[:, columns:] = 0
        xe = rng.integers(67, 188, (rows, 6)).astype(np.uint8)
        xe[1, 2] = 255
        xv = (f64(q) * np.repeat(B8.scale(xe), 128, 1))[:, :columns]
        e = torch.full((rows, 8), 255, dtype=torch.uint8, device="cuda")
        e[:, :6] = torch.from_numpy(xe)
        x = blocks.BlockTensor(q.to(blocks.E4M3), e, columns)
    want = xv @ wv.T
    y = micro.matmul_micro(x, kept(wq, we, micro.MicroWeight), dtype=DTYPES[dtype])
    near(y, want, product_room(xv, wv, dtype, codes) + 4 * U * np.abs(want) + rounded(want, dtype), "y")
    assert y[1].isnan().all() and y[:, 7].isnan().all() and y.isnan().sum() == rows + outer - 1


# --------------------------------------------------------------------------------------------------
# Gradients, autograd, streams


@pytest.mark.parametrize("rows,inner,outer", [(1, 1, 1), (3, 300, 140), (7, 130, 47), (65, 200, 300), (500, 129, 127),
                                              (1000, 512, 384), (5003, 128, 200)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_linear_backward(gpu, rows, inner, outer, dtype):
    from tcc_spmm_amd.micro import linear_micro, linear_micro_backward, quantize_weight_micro
    x, dy, w = random((rows, inner), 1, dtype), random((rows, outer), 2, dtype, 1e-2), random((outer, inner), 3)
    weight = quantize_weight_micro(w, tiles=True, transposed=True)
    _, kept = linear_micro(x, weight, keep=True)
    xv, wv, gv, g = B8.quantize(f64(x))[2], O.quantize_tiles(f64(w))[2], B8.quantize(f64(dy))[2], f64(dy)
    want = {"dx": gv @ wv, "dw": g.T @ xv, "db": g.sum(0)}
    room = {"dx": product_room(gv, wv.T, dtype, "e4m3") + rounded(gv @ wv, dtype),
            "dw": (rows / 4 + 64) * U * (np.abs(g).T @ np.abs(xv)), "db": (rows / 4 + 64) * U * np.abs(g).sum(0)}
    for d in (dy, cut(dy)):
        got = dict(zip(("dx", "dw", "db"), linear_micro_backward(d, kept, weight)))
        for name in want:
            near(got[name], want[name], room[name] * 1.01 + 1e-30, name)
        again = dict(zip(("dx", "dw", "db"), linear_micro_backward(d, kept, weight)))
        assert all(torch.equal(got[n], again[n]) for n in want), "repeated calls give the same bits"
    only = linear_micro_backward(dy, kept, None, need=(False, True, False))
    assert only[0] is None and only[2] is None and torch.equal(only[1], got["dw"])


def test_gradients_against_differences(gpu):
    """The layer is linear in the values of its blocks, so differences of the loss sum(dy * y) along a direction are the
    gradients' products with it. The input gradient is that of the quantized output gradient."""
    from tcc_spmm_amd.micro import linear_micro, linear_micro_backward, quantize_weight_micro
    x, w, dy = random((200, 150), 1), random((90, 150), 2), random((200, 90), 3)
    weight = quantize_weight_micro(w, tiles=True, transposed=True)
    _, kept = linear_micro(x, weight, keep=True)
    grads = [f64(t) for t in linear_micro_backward(dy, kept, weight)]
    xv, wv, g, gv = B8.quantize(f64(x))[2], O.quantize_tiles(f64(w))[2], f64(dy), B8.quantize(f64(dy))[2]
    rng = np.random.default_rng(4)
    loss = lambda a, b, c, d: (d * (a @ b.T + c)).sum()  # noqa: E731
    for at, grad in enumerate(grads):
        v = rng.standard_normal(grad.shape)
        step = [np.zeros_like(xv), np.zeros_like(wv), np.zeros(90)]
        step[at] = v
        d = gv if at == 0 else g
        diff = (loss(xv + step[0], wv + step[1], step[2], d) - loss(xv - step[0], wv - step[1], -step[2], d)) / 2
        assert abs((grad * v).sum() - diff) <= 1e-5 * np.abs(grad * v).sum()


@pytest.mark.parametrize("autocast", [None, "bf16"])
def test_layer_under_autograd(gpu, autocast):
    """MicroLinear gives the gradients of the calls that it is made of, under autocast in its type; what autograd keeps of x
    is a byte an element."""
    from tcc_spmm_amd import micro as M
    torch.manual_seed(0)
    layer = M.MicroLinear(96, 80).cuda()
    x, dy = random((3, 50, 96), 1).requires_grad_(), random((3, 50, 80), 2, autocast or "f32")
    saved = []
    with torch.autocast("cuda", DTYPES[autocast or "bf16"], enabled=autocast is not None):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
            y = layer(x)
        with torch.no_grad():
            assert torch.equal(layer(x), y)
    y.backward(dy)
    weight = M.quantize_weight_micro(layer.weight.detach(), tiles=True, transposed=True)
    given = x.detach().to(dy.dtype)
    want, kept = M.linear_micro(given, weight, layer.bias.detach(), keep=True)
    dx, dw, db = M.linear_micro_backward(dy, kept, weight)
    assert torch.equal(y, want) and torch.equal(x.grad, dx.float())
    assert torch.equal(layer.weight.grad, dw) and torch.equal(layer.bias.grad, db)
    assert all(t.element_size() == 1 for t in saved)
    frozen, bias = layer.serving()
    assert torch.equal(M.linear_micro(given, frozen, bias), want)


def test_calls_on_another_stream(gpu):
    from tcc_spmm_amd import micro as M
    x, w, dy = random((300, 256), 1, "bf16"), random((128, 256), 2), random((300, 128), 3, "bf16")

    def calls(stream):
        weight = M.quantize_weight_micro(w, tiles=True, transposed=True, stream=stream)
        y, kept = M.linear_micro(x, weight, keep=True, stream=stream)
        four = M.linear_micro(x, weight, codes=M.E2M1, stream=stream)
        rows = M.quantize_micro(x, stream=stream)
        return (y, four, M.matmul_micro(rows, weight, stream=stream), rows.dequantize(stream=stream),
                *M.linear_micro_backward(dy, kept, weight, stream=stream))

    want = calls(None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = calls(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_graph_capture_replays(gpu):
    """Two graphs captured one after the other, replayed in turn with eager work between, each with inputs of its own."""
    from tcc_spmm_amd import micro as M
    w = random((200, 300), 2)
    inputs = [(random((777, 300), s, "bf16"), random((777, 200), s + 1, "bf16")) for s in (1, 5)]

    def step(x, dy):
        weight = M.quantize_weight_micro(w, tiles=True, transposed=True)
        y, kept = M.linear_micro(x, weight, keep=True)
        return (y, M.linear_micro(x[:3], weight), M.linear_micro(x, weight, codes=M.E2M1),
                *M.linear_micro_backward(dy, kept, weight))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*inputs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for given in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*given)
        graphs.append((graph, out))
    for seed in (11, 12, 13):
        for (graph, out), (x, dy) in zip(graphs, inputs):
            x.copy_(random((777, 300), seed, "bf16"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step(x, dy)))


def test_refusals(gpu):
    from tcc_spmm_amd import blocks as B
    from tcc_spmm_amd import micro as M
    x, w = random((8, 64), 1), random((32, 64), 2)
    weight, stack = M.quantize_weight_micro(w), M.quantize_weight_micro(w.reshape(4, 8, 64))
    for call in (lambda: M.linear_micro(random((8, 65), 1), weight), lambda: M.linear_micro(x.double(), weight),
                 lambda: M.linear_micro(x.cpu(), weight), lambda: M.linear_micro(x, weight, torch.zeros(31, device="cuda")),
                 lambda: M.linear_micro(x, weight, torch.zeros(32, device="cuda", dtype=torch.bfloat16)),
                 lambda: M.linear_micro(x, weight, codes=torch.int8), lambda: M.linear_micro(x, stack),
                 lambda: M.linear_micro(x, weight, codes=M.E2M1, keep=True),
                 lambda: M.matmul_micro(B.quantize_blocks(x, torch.int8), weight),
                 lambda: M.matmul_micro(M.quantize_micro(x[:, :63]), weight),
                 lambda: M.matmul_micro(M.quantize_micro(x), stack),
                 lambda: M.linear_micro_backward(random((8, 32), 1), B.quantize_blocks(x), weight),
                 lambda: M.quantize_weight_micro(w, transposed=True), lambda: M.quantize_weight_micro(w[0]),
                 lambda: M.dequantize_micro(M.quantize_micro(x), torch.float64), lambda: M.micro_linear(x, w.reshape(4, 8, 64)),
                 lambda: M.quantize_micro(x.to(torch.float64))):
        with pytest.raises(ValueError):
            call()
