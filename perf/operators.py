"""The dense layers behind the sparse product, as measurable cases: a linear layer whose product runs in
8-bit floating point with a scale for each block of 128, its training step, and activations whose
input is kept in 8 bits for the backward pass.

Blocks: 128 consecutive elements of a row (for a weight, a tile of 128 x 128) share one power of two,
held as a byte e that stands for 2^(e - 127): the smallest that brings the block's largest magnitude
to at most 448 (E4M3 codes) or 127 (INT8 codes). Codes are stored with rows padded by zeros to a
multiple of 128, exponents with rows padded to a multiple of 4.

Row counts and widths follow the library's graphs (2,449,029 and 262,144 rows, 128 and 256 features)
and generic dense layers; odd sizes are generic.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"e4m3": E4M3, "int8": INT8}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# --------------------------------------------------------------------------------------------------
# Cases


def listed() -> list[dict]:
    return [
        # One token through a square layer: every weight is read once for it; latency counts.
        linear("linear_token", 1, 4096, 4096, "bf16"),
        # A small batch of requests, one token each, through a wide layer.
        linear("linear_batch_24", 24, 4096, 8192, "f16", bias=True),
        # A mini-batch with no size a multiple of anything, its rows cut out of a wider array.
        linear("linear_odd", 777, 1001, 1437, "bf16", bias=True, cut=True),
        # A prompt, or a training batch's forward pass.
        linear("linear_prompt", 4096, 4096, 8192, "bf16"),
        # The rows that the sparse product gives for the large product graph, through one layer.
        linear("linear_graph_2m", 2449029, 128, 256, "f32", bias=True),
        # One training step of a layer, ordinary sizes.
        step("step_ordinary", 2048, 1024, 4096, "bf16"),
        # The largest: 8,192 tokens through a layer that widens 4,096 to 8,192.
        step("step_large", 8192, 4096, 8192, "bf16"),
        # One training step on the rows of a medium graph, in 32 bits, with an odd class count.
        step("step_graph_262k", 262144, 256, 47, "f32"),
        # A gated activation in a training step: forward, 8-bit checkpoint, backward.
        activation("gated_step", 8192, 8192, "bf16", "silu", True, "int8"),
        # A small odd one, where launches count.
        activation("gelu_step_small", 333, 1001, "f32", "gelu", False, "int8"),
        # The backward pass alone, from a checkpoint in E4M3.
        activation("gelu_backward", 4096, 8192, "bf16", "gelu_tanh", False, "e4m3", op="activation_backward"),
        # The backward pass on the large graph's rows.
        activation("silu_backward_graph_2m", 2449029, 128, "f32", "silu", False, "int8",
                   op="activation_backward"),
    ]


def linear(name, rows, inner, outer, dtype, bias=False, cut=False) -> dict:
    return dict(name=name, op="linear", rows=rows, inner=inner, outer=outer, dtype=dtype, bias=bias, cut=cut)


def step(name, rows, inner, outer, dtype, cut=False) -> dict:
    return dict(name=name, op="step", rows=rows, inner=inner, outer=outer, dtype=dtype, bias=True, cut=cut)


def activation(name, rows, width, dtype, kind, gated, codes, op="activation_step") -> dict:
    return dict(name=name, op=op, rows=rows, width=width, dtype=dtype, kind=kind, gated=gated, codes=codes)


def draw(rng) -> dict:
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    def width_of(low, high):
        width = spread(low, high)
        if rng.random() < 0.5:
            width = -(-width // 128) * 128
        return width if width != 3072 else 2048

    limit = work(step("", 8192, 4096, 8192, "bf16"))
    most_bytes = work(activation("", 2449029, 128, "f32", "silu", False, "int8"))["bytes"] * 2
    while True:
        op = rng.choice(["linear", "linear", "step", "activation_step", "activation_backward"])
        dtype = rng.choice(["f32", "bf16", "f16"])
        graph = rng.random() < 0.3
        rows = spread(100000, 2449029) if graph else spread(1, 16384)
        if op in ("linear", "step"):
            low, high = (16, 512) if graph else (64, 8192)
            inner, outer = width_of(low, high), width_of(low, high)
            make = linear if op == "linear" else step
            case = make("", rows, inner, outer, dtype, cut=rng.random() < 0.25)
            case["bias"] = op == "step" or rng.random() < 0.5
        else:
            width = width_of(16, 512) if graph else width_of(64, 16384)
            case = activation("", rows, width, dtype, rng.choice(["silu", "gelu", "gelu_tanh"]),
                              rng.random() < 0.5, rng.choice(["int8", "e4m3"]), op=op)
        need = work(case)
        if need["flops"] <= limit["flops"] and need["bytes"] <= most_bytes:
            del case["name"]
            return case


def work(case) -> dict:
    m, s = case["rows"], BYTES[case["dtype"]]
    if case["op"] in ("linear", "step"):
        k, n = case["inner"], case["outer"]
        tiles = -(-k // 128) * -(-n // 128)
        bias = 4 * n if case["bias"] else 0
        if case["op"] == "linear":
            return {"bytes": m * k * s + n * k + tiles + bias + m * n * s, "flops": 2 * m * n * k}
        # x, dy and the weight in; y, dx and the weight's and the bias's gradients out
        return {"bytes": 2 * m * k * s + 2 * m * n * s + 8 * n * k + 2 * bias, "flops": 6 * m * n * k + m * n}
    f = case["width"]
    wide = 2 * f if case["gated"] else f
    if case["op"] == "activation_step":
        # x and dy in, y and dx out
        return {"bytes": 2 * m * wide * s + 2 * m * f * s, "flops": 30 * m * f}
    blocks = -(-f // 128) * (2 if case["gated"] else 1)
    return {"bytes": m * f * s + m * (wide + blocks) + m * wide * s, "flops": 16 * m * f}


# --------------------------------------------------------------------------------------------------
# Inputs


def _random(shape, gen, dtype, spread=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE) * spread).to(dtype)


def _cut(t, cut):
    """The same values as a view into rows that hold 5 elements more."""
    if not cut:
        return t
    wide = torch.zeros((t.shape[0], t.shape[1] + 5), dtype=t.dtype, device=t.device)
    wide[:, 3:3 + t.shape[1]] = t
    return wide[:, 3:3 + t.shape[1]]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype, m = DTYPES[case["dtype"]], case["rows"]
    state = {"case": case}
    if case["op"] in ("linear", "step"):
        k, n = case["inner"], case["outer"]
        # Rows of different size, as rows of different degree have after an aggregation.
        rows = torch.exp(torch.randn((m, 1), generator=gen, device=DEVICE))
        state["x"] = _cut((_random((m, k), gen, torch.float32) * rows).to(dtype), case["cut"])
        w = _random((n, k), gen, torch.float32, k ** -0.5)
        state["bias"] = _random((n,), gen, torch.float32, 0.1) if case["bias"] else None
        if case["op"] == "linear":
            # A served layer keeps its weight in 8 bits.
            state["codes"], state["exponents"] = _store(*_tile_codes(w), k)
        else:
            state["w"] = w
            state["dy"] = _cut(_random((m, n), gen, dtype, 1e-2), case["cut"])
        return state
    f = case["width"]
    x = _random((m, 2 * f if case["gated"] else f), gen, dtype, 1.5)
    state["dy"] = _random((m, f), gen, dtype, 1e-2)
    if case["op"] == "activation_step":
        state["x"] = x
    else:
        # What the forward pass kept: a gated row is two rows of its width, the gate and the factor.
        kept = x.reshape(-1, f).float()
        state["codes"], state["exponents"] = _store(*_row_codes(kept, CODES[case["codes"]]), f)
    return state


# --------------------------------------------------------------------------------------------------
# The plain form: 32 bits, elementary operations


def _exponents(peak, codes):
    """The byte of each block's power of two, from the bits of the block's largest magnitude."""
    bits = peak.view(torch.int32)
    lead, past = (8, 0x600000) if codes == E4M3 else (6, 0x7E0000)
    e = (bits >> 23) - lead + ((bits & 0x7FFFFF) > past).int()
    return torch.where(peak == 0, 127, e.clamp(min=1))


def _power(e):
    return (e.int() << 23).view(torch.float32)


def _round(scaled, codes):
    return scaled.to(E4M3) if codes == E4M3 else scaled.round().to(INT8)


def _padded(x, rows, columns):
    return torch.nn.functional.pad(x, (0, columns - x.shape[1], 0, rows - x.shape[0]))


def _row_codes(x, codes=E4M3):
    """Codes [rows, blocks, 128] and exponents [rows, blocks] of an FP32 matrix."""
    m, k = x.shape
    blocks = -(-k // 128)
    b = _padded(x, m, blocks * 128).reshape(m, blocks, 128)
    e = _exponents(b.abs().amax(2), codes)
    return _round(b * _power(254 - e)[:, :, None], codes), e


def _tile_codes(w):
    """Codes [rows, blocks, 128] and exponents [row tiles, blocks] of an FP32 weight."""
    n, k = w.shape
    up, across = -(-n // 128), -(-k // 128)
    t = _padded(w, up * 128, across * 128).reshape(up, 128, across, 128)
    e = _exponents(t.abs().amax((1, 3)), E4M3)
    q = _round(t * _power(254 - e)[:, None, :, None], E4M3)
    return q.reshape(up * 128, across, 128)[:n], e


def _store(q, e, columns):
    """Codes and exponents as they are kept: rows of whole blocks, exponents in fours."""
    kept = torch.full((e.shape[0], -(-e.shape[1] // 4) * 4), 127, dtype=torch.uint8, device=e.device)
    kept[:, :e.shape[1]] = e.to(torch.uint8)
    return q.reshape(q.shape[0], -1).contiguous(), kept


def _row_values(q, e, columns):
    m = q.shape[0]
    return (q.float() * _power(e)[:, :, None]).reshape(m, -1)[:, :columns]


def _tile_values(q, e, columns):
    n = q.shape[0]
    s = _power(e).repeat_interleave(128, 0)[:n]
    return (q.float() * s[:, :, None]).reshape(n, -1)[:, :columns]


def _function(kind, x):
    """f(x) and f'(x)."""
    if kind == "silu":
        s = 1 / (1 + torch.exp(-x))
        return x * s, s * (1 + x * (1 - s))
    if kind == "gelu":
        p = 0.5 * (1 + torch.erf(x * 0.5 ** 0.5))
        return x * p, p + x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
    c = (2 / math.pi) ** 0.5
    t = torch.tanh(c * (x + 0.044715 * x * x * x))
    return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x)


def _act_backward(case, dy, kept):
    f, (m, width) = case["kind"], dy.shape
    if not case["gated"]:
        return dy * _function(f, kept)[1]
    g, u = kept.reshape(m, 2, width).unbind(1)
    value, slope = _function(f, g)
    return torch.cat((dy * u * slope, dy * value), 1)


def _plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        k, n = case["inner"], case["outer"]
        x = _row_values(*_row_codes(state["x"].float()), k)
        blocks = -(-k // 128)
        w = _tile_values(state["codes"].reshape(n, blocks, 128), state["exponents"][:, :blocks], k)
        y = x @ w.T
        return (y if state["bias"] is None else y + state["bias"]).to(dtype)
    if case["op"] == "step":
        x, dy = state["x"].float(), state["dy"].float()
        k, n = case["inner"], case["outer"]
        xv = _row_values(*_row_codes(x), k)
        wv = _tile_values(*_tile_codes(state["w"]), k)
        y = xv @ wv.T + state["bias"]
        dx = _row_values(*_row_codes(dy), n) @ wv
        return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dy.T @ xv, "db": dy.sum(0)}
    codes, width = CODES[case["codes"]], case["width"]
    dy = state["dy"].float()
    if case["op"] == "activation_step":
        x = state["x"].float()
        if case["gated"]:
            g, u = x[:, :width], x[:, width:]
            y = _function(case["kind"], g)[0] * u
        else:
            y = _function(case["kind"], x)[0]
        kept = _row_values(*_row_codes(x.reshape(-1, width), codes), width)
        return {"y": y.to(dtype), "dx": _act_backward(case, dy, kept).to(dtype)}
    q, blocks = state["codes"], -(-width // 128)
    kept = _row_values(q.reshape(q.shape[0], blocks, 128), state["exponents"][:, :blocks], width)
    return _act_backward(case, dy, kept).to(dtype)


# --------------------------------------------------------------------------------------------------
# One pass


def run(state):
    if not own:
        return _plain(state)
    from tcc_spmm_amd import blocks as B
    case = state["case"]
    if case["op"] == "linear":
        weight = B.BlockWeight(state["codes"], state["exponents"], case["inner"])
        return B.linear_blocks(state["x"], weight, state["bias"])
    if case["op"] == "step":
        weight = B.quantize_weight_blocks(state["w"], transposed=True)
        y, kept = B.linear_blocks(state["x"], weight, state["bias"], keep=True)
        dx, dw, db = B.linear_blocks_backward(state["dy"], kept, weight)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    kind, gated = case["kind"], case["gated"]
    if case["op"] == "activation_step":
        y, kept = B.activation_blocks(state["x"], kind, gated=gated, codes=CODES[case["codes"]])
        return {"y": y, "dx": B.activation_blocks_backward(state["dy"], kept, kind, gated=gated)}
    kept = B.BlockTensor(state["codes"], state["exponents"], case["width"])
    return B.activation_blocks_backward(state["dy"], kept, kind, gated=gated)


# --------------------------------------------------------------------------------------------------
# The definition in 64 bits, written apart from the plain form


def _two_to(e):
    """2^e in 64 bits, from its bits: the GPU's pow and exp2 may be a last bit off."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest(v, peak, top):
    """v [.., with its block's peak broadcast] on the grid that the block's power of two gives."""
    fraction, power = torch.frexp(peak)  # peak = fraction * 2^power, 0.5 <= fraction < 1
    limit, high = math.frexp(top)
    e = torch.clamp(power - high + (fraction > limit).int(), min=-126)
    e = torch.where(peak == 0, torch.zeros_like(e), e)
    scale = _two_to(e)
    v = v / scale
    if top == 127.0:
        return torch.round(v) * scale
    # E4M3: three bits after the leading one, the smallest normal 2^-6
    at = torch.frexp(v)[1] - 1
    unit = _two_to(torch.clamp(at, min=-6) - 3)
    return torch.round(v / unit) * unit * scale


def _grid_rows(x, top=448.0):
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], 128):
        part = x[:, c:c + 128]
        out[:, c:c + 128] = _nearest(part, part.abs().amax(1, keepdim=True), top)
    return out


def _grid_tiles(w):
    out = torch.empty_like(w)
    for r in range(0, w.shape[0], 128):
        for c in range(0, w.shape[1], 128):
            part = w[r:r + 128, c:c + 128]
            out[r:r + 128, c:c + 128] = _nearest(part, part.abs().amax(), 448.0)
    return out


def _kept_values(codes, exponents, columns, group):
    """The numbers that stored codes stand for; one row of exponents for each `group` rows."""
    v = codes.double()
    scale = _two_to(exponents.int() - 127)
    for b in range(v.shape[1] // 128):
        v[:, 128 * b:128 * b + 128] *= scale[:, b].repeat_interleave(group)[:v.shape[0], None]
    return v[:, :columns]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "linear":
        x = _grid_rows(state["x"].double())
        w = _kept_values(state["codes"], state["exponents"], case["inner"], 128)
        y = torch.matmul(x, w.t())
        if case["bias"]:
            y += state["bias"].double()
        return y
    if case["op"] == "step":
        x, dy = _grid_rows(state["x"].double()), state["dy"].double()
        w = _grid_tiles(state["w"].double())
        return {"y": torch.matmul(x, w.t()) + state["bias"].double(), "dx": torch.matmul(_grid_rows(dy), w),
                "dw": torch.matmul(dy.t(), x), "db": dy.sum(0)}
    width, top = case["width"], 448.0 if case["codes"] == "e4m3" else 127.0
    dy, out = state["dy"].double(), {}

    def value(v):
        if case["kind"] == "silu":
            return v * torch.sigmoid(v)
        if case["kind"] == "gelu":
            return 0.5 * v * torch.erfc(-v / math.sqrt(2.0))
        return v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))

    def slope(v):
        if case["kind"] == "silu":
            s = torch.sigmoid(v)
            return s + v * s * torch.sigmoid(-v)
        if case["kind"] == "gelu":
            return 0.5 * torch.erfc(-v / math.sqrt(2.0)) + v * torch.exp(-v * v / 2.0) / math.sqrt(2.0 * math.pi)
        a = 2.0 * math.sqrt(2.0 / math.pi)
        s = torch.sigmoid(a * (v + 0.044715 * v ** 3))
        return s + v * s * (1.0 - s) * a * (1.0 + 0.134145 * v * v)

    if case["op"] == "activation_step":
        x = state["x"].double()
        out["y"] = value(x[:, :width]) * x[:, width:] if case["gated"] else value(x)
        kept = torch.cat([_grid_rows(x[:, c:c + width], top) for c in range(0, x.shape[1], width)], 1)
    else:
        kept = _kept_values(state["codes"], state["exponents"], width, 1).reshape(case["rows"], -1)
    if case["gated"]:
        g, u = kept[:, :width], kept[:, width:]
        out["dx"] = torch.cat([dy * u * slope(g), dy * value(g)], 1)
    else:
        out["dx"] = dy * slope(kept)
    return out if case["op"] == "activation_step" else out["dx"]
