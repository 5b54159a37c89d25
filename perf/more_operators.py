"""Microscaled 4-bit layers and their routing, as measurable cases: rows and weights in E2M1 blocks of 32, a linear
layer whose weight is held in them, its training step, and a layer of many experts: tokens sorted by expert and
back, and the experts' products.

Microscaled blocks: 32 consecutive elements of a row share one power of two, a byte e that stands for 2^(e - 127): the
smallest that brings the block's largest magnitude to at most 6, the largest E2M1 code. A weight that is trained has
one power for each tile of 32 x 32, so that its transpose holds the same values. Two codes are a byte, the first in
the low half; rows of codes are padded by zeros to a multiple of 128 elements. Exponents: the byte of block b of a row
lies at 16 (b / 16) + 4 (b % 4) + b / 4 % 4, rows being padded to a multiple of 16 with 127.

What a layer multiplies the weight with is x in E4M3 blocks of 128 (the format of the 8-bit layers: codes up to 448)
or in microscaled blocks of its own.

Row counts and widths follow the library's graphs (2,449,029 and 262,144 rows, 128 and 256 features) and generic dense
layers and routers; odd sizes are generic.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
E4M3, E2M1 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"e4m3": E4M3, "e2m1": E2M1}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# --------------------------------------------------------------------------------------------------
# Cases


def listed() -> list[dict]:
    return [
        # Rows of a batch's activations into microscaled blocks, and the values back, as a 4-bit cache or checkpoint does.
        rows("micro_rows", 8192, 8192, "bf16"),
        # A small odd one, where launches count.
        rows("micro_rows_small", 333, 1001, "f32"),
        # One token through a square layer: every weight is read once for it; latency counts.
        linear("micro_token", 1, 4096, 4096, "bf16", "e4m3"),
        # A batch of requests, one token each, with a bias, its rows cut out of a wider array.
        linear("micro_batch_48", 48, 4096, 8191, "f16", "e4m3", bias=True, cut=True),
        # A prompt whose activations keep 8 bits.
        linear("micro_prompt", 4096, 4096, 8192, "bf16", "e4m3"),
        # The largest: 8,192 tokens with both operands in 4 bits.
        linear("micro_both_4", 8192, 4096, 8192, "bf16", "e2m1"),
        # One training step of a layer whose weight is held in 4 bits, odd rows and classes, in 32 bits.
        step("micro_step", 2001, 1024, 4097, "f32"),
        # One new token of each of 24 requests, to 4 of 32 experts and back.
        routed("routed_token", 24, 4, 32, 2048, "bf16", False),
        # A training batch to 8 of 64 experts and back, with all gradients.
        routed("routed_step", 8192, 8, 64, 2048, "bf16", True),
        # One new token of each of 24 requests through the experts' first layer: most experts get a row or a few.
        experts("experts_token", 24, 4, 32, 2048, 4096, "bf16", "e4m3"),
        # A prompt through it, with both operands in 4 bits.
        experts("experts_prompt", 8192, 4, 32, 2048, 4096, "bf16", "e2m1"),
        # The experts' second layer, forward and the gradient of its rows, the experts themselves being frozen.
        experts("experts_step", 3001, 2, 8, 2048, 1000, "bf16", "e4m3", True),
    ]


def rows(name, count, width, dtype) -> dict:
    return dict(name=name, op="rows", rows=count, width=width, dtype=dtype)


def linear(name, count, inner, outer, dtype, codes, bias=False, cut=False) -> dict:
    return dict(name=name, op="linear", rows=count, inner=inner, outer=outer, dtype=dtype, codes=codes, bias=bias, cut=cut)


def step(name, count, inner, outer, dtype) -> dict:
    return dict(name=name, op="step", rows=count, inner=inner, outer=outer, dtype=dtype)


def routed(name, tokens, each, count, width, dtype, gradients, away=0.0) -> dict:
    """Tokens to `each` of `count` experts; a share `away` of the choices is for experts that are not here."""
    return dict(name=name, op="routed", tokens=tokens, each=each, experts=count, width=width, dtype=dtype,
                gradients=gradients, away=away)


def experts(name, tokens, each, count, inner, outer, dtype, codes, gradients=False, away=0.0) -> dict:
    """The experts' layer of tokens; with gradients, of rows in the experts' order."""
    return dict(name=name, op="experts", tokens=tokens, each=each, experts=count, inner=inner, outer=outer, dtype=dtype,
                codes=codes, gradients=gradients, away=away)


def draw(rng) -> dict:
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    def width_of(low, high):
        width = spread(low, high)
        return -(-width // 128) * 128 if rng.random() < 0.5 else width

    most_flops = work(linear("", 8192, 4096, 8192, "bf16", "e2m1"))["flops"]
    most_bytes = 2.5e9
    while True:
        op = rng.choice(["rows", "linear", "linear", "step", "routed", "experts", "experts"])
        dtype, codes = rng.choice(["f32", "bf16", "f16"]), rng.choice(["e4m3", "e2m1"])
        graph = rng.random() < 0.2
        count = spread(100000, 2449029) if graph else spread(1, 16384)
        inner, outer = (width_of(16, 512), width_of(16, 512)) if graph else (width_of(64, 8192), width_of(64, 8192))
        chosen = spread(1, 128)
        each, away = rng.randint(1, min(8, chosen)), rng.choice([0.0, 0.0, 0.0, 0.1, 0.5])
        tokens = spread(1, 16384)
        if op == "rows":
            case = rows("", count, inner, dtype)
        elif op == "linear":
            case = linear("", count, inner, outer, dtype, codes, rng.random() < 0.5, rng.random() < 0.25)
        elif op == "step":
            case = step("", count, inner, outer, dtype)
        elif op == "routed":
            case = routed("", tokens, each, chosen, min(inner, 8192), dtype, rng.random() < 0.6, away)
        else:
            case = experts("", tokens, each, chosen, inner, outer, dtype, codes, rng.random() < 0.3, away)
        need = work(case)
        weights = chosen * inner * outer if op == "experts" else 0
        if need["flops"] <= most_flops and need["bytes"] <= most_bytes and weights <= 1 << 29:
            del case["name"]
            return case


def work(case) -> dict:
    s = BYTES[case["dtype"]]
    if case["op"] == "rows":
        m, w = case["rows"], case["width"]
        # x in, codes and exponents out, and the values
        return {"bytes": 2 * m * w * s + m * (w // 2 + -(-w // 32)), "flops": 4 * m * w}
    if case["op"] in ("linear", "step"):
        m, k, n = case["rows"], case["inner"], case["outer"]
        if case["op"] == "linear":
            weight = n * k // 2 + n * -(-k // 32) + (4 * n if case["bias"] else 0)
            return {"bytes": m * k * s + weight + m * n * s, "flops": 2 * m * n * k}
        # x, dy and the weight in; y, dx and the weight's and the bias's gradients out
        return {"bytes": 2 * m * k * s + 2 * m * n * s + 8 * n * k + 8 * n, "flops": 6 * m * n * k + m * n}
    t, j, slots = case["tokens"], case["each"], case["tokens"] * case["each"]
    lists = 8 * slots + 4 * slots + 4 * (case["experts"] + 1)  # choices in, the order and the offsets out
    if case["op"] == "routed":
        w = case["width"] * s
        # x in and its rows out; the experts' rows and weights in and their sums out
        forward = lists + t * w + slots * w + slots * w + 4 * slots + t * w
        if not case["gradients"]:
            return {"bytes": forward, "flops": 2 * slots * case["width"]}
        # dy in, the rows' and the weights' gradients out; the gradient of x's rows in, x's out
        return {"bytes": forward + t * w + slots * w + 4 * slots + slots * w + t * w, "flops": 7 * slots * case["width"]}
    k, n = case["inner"], case["outer"]
    used = min(case["experts"], slots)
    weight = used * (n * k // 2 + n * -(-k // 32))
    if not case["gradients"]:
        return {"bytes": 8 * slots + t * k * s + weight + slots * n * s, "flops": 2 * slots * n * k}
    return {"bytes": 8 * slots + 2 * slots * (k + n) * s + 2 * weight, "flops": 4 * slots * n * k}


# --------------------------------------------------------------------------------------------------
# Inputs


def _random(shape, gen, dtype, spread=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE) * spread).to(dtype)


def _rows_of_sizes(shape, gen, dtype):
    """Rows of different size, as activations have."""
    return (_random(shape, gen, torch.float32) * torch.exp(_random((shape[0], 1), gen, torch.float32))).to(dtype)


def _cut(t, cut):
    """The same values as a view into rows that hold 5 elements more."""
    if not cut:
        return t
    wide = torch.zeros((t.shape[0], t.shape[1] + 5), dtype=t.dtype, device=t.device)
    wide[:, 3:3 + t.shape[1]] = t
    return wide[:, 3:3 + t.shape[1]]


def _choices(case, gen):
    """Experts and weights of each token, as a router gives them: some experts are chosen more than others."""
    t, j, e = case["tokens"], case["each"], case["experts"]
    scores = torch.randn((t, e), generator=gen, device=DEVICE) + torch.randn((1, e), generator=gen, device=DEVICE)
    top, ids = scores.topk(j, dim=1)
    here = torch.rand((t, j), generator=gen, device=DEVICE) >= case["away"]
    return torch.where(here, ids, -1), torch.softmax(top, 1)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype, state = DTYPES[case["dtype"]], {"case": case}
    if case["op"] == "rows":
        state["x"] = _rows_of_sizes((case["rows"], case["width"]), gen, dtype)
        return state
    if case["op"] in ("linear", "step"):
        m, k, n = case["rows"], case["inner"], case["outer"]
        w = _random((n, k), gen, torch.float32, k ** -0.5)
        if case["op"] == "linear":
            state["x"] = _cut(_rows_of_sizes((m, k), gen, dtype), case["cut"])
            # A served layer keeps its weight in 4 bits.
            state["codes"], state["exponents"] = _store(*_micro_codes(w))
            state["bias"] = _random((n,), gen, torch.float32, 0.1) if case["bias"] else None
        else:
            state["x"], state["w"] = _rows_of_sizes((m, k), gen, dtype), w
            state["bias"] = _random((n,), gen, torch.float32, 0.1)
            state["dy"] = _random((m, n), gen, dtype, 1e-2)
        return state
    state["ids"], weights = _choices(case, gen)
    t, slots = case["tokens"], case["tokens"] * case["each"]
    if case["op"] == "routed":
        state["x"], state["weights"] = _random((t, case["width"]), gen, dtype), weights
        state["out"] = _random((slots, case["width"]), gen, dtype)
        if case["gradients"]:
            state["dy"] = _random((t, case["width"]), gen, dtype, 1e-2)
            state["drows"] = _random((slots, case["width"]), gen, dtype, 1e-2)
        return state
    e, k, n = case["experts"], case["inner"], case["outer"]
    state["x"] = _rows_of_sizes((slots if case["gradients"] else t, k), gen, dtype)
    stacks = [[], [], [], []]
    for _ in range(e):
        w = _random((n, k), gen, torch.float32, k ** -0.5)
        if case["gradients"]:
            q, b = _tile_codes(w)
            parts = (*_store(q[:n, :-(-k // 32)], b[:n, :-(-k // 32)]), *_store(*_turned(q, b, n, k)))
        else:
            parts = _store(*_micro_codes(w))
        for stack, part in zip(stacks, parts):
            stack.append(part)
    names = ("codes", "exponents", "codes_t", "exponents_t")
    state.update({name: torch.stack(stack) for name, stack in zip(names, stacks) if stack})
    if case["gradients"]:
        state["dy"] = _random((slots, n), gen, dtype, 1e-2)
    return state


# --------------------------------------------------------------------------------------------------
# The plain form: 32 bits, elementary operations


def _exponents(peak, lead, past):
    """The byte of each block's power of two, from the bits of the block's largest magnitude."""
    bits = peak.view(torch.int32)
    e = (bits >> 23) - lead + ((bits & 0x7FFFFF) > past).int()
    return torch.where(peak == 0, 127, e.clamp(min=1))


def _power(e):
    return (e.int() << 23).view(torch.float32)


def _padded(x, count, columns):
    return torch.nn.functional.pad(x, (0, columns - x.shape[1], 0, count - x.shape[0]))


def _e2m1(v):
    """Codes of |v| <= 6, rounded half to even: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and the same with the sign's bit."""
    a = v.abs()
    half = torch.where(a < 2, (2 * a).round(), torch.where(a < 4, a.round() + 2, (a / 2).round() + 4))
    return half.to(torch.uint8) + torch.signbit(v).to(torch.uint8) * 8


def _micro_codes(x):
    """Codes [rows, blocks, 32] and exponents [rows, blocks] of an FP32 matrix."""
    m, k = x.shape
    blocks = -(-k // 32)
    b = _padded(x, m, blocks * 32).reshape(m, blocks, 32)
    e = _exponents(b.abs().amax(2), 2, 0x400000)
    return _e2m1(b * _power(254 - e)[:, :, None]), e


def _tile_codes(w):
    """The same of a weight in tiles of 32 x 32, both sides padded to whole tiles."""
    n, k = w.shape
    up, across = -(-n // 32), -(-k // 32)
    t = _padded(w, up * 32, across * 32).reshape(up, 32, across, 32)
    e = _exponents(t.abs().amax((1, 3)), 2, 0x400000)
    q = _e2m1(t * _power(254 - e)[:, None, :, None])
    return q.reshape(up * 32, across, 32), e.repeat_interleave(32, 0)


def _turned(q, e, n, k):
    """Codes and exponents of the transposed weight, from its tiles."""
    up, across = q.shape[0] // 32, q.shape[1]
    qt = q.reshape(up * 32, across * 32).t().reshape(across * 32, up, 32)[:k]
    return qt, e[::32].t().repeat_interleave(32, 0)[:k]


def _store(q, e):
    """Codes and exponents as they are kept."""
    m, blocks = e.shape
    whole = _padded(q.reshape(m, -1), m, -(-blocks // 4) * 128)
    kept = torch.full((m, -(-blocks // 16) * 16), 127, dtype=torch.uint8, device=e.device)
    kept[:, :blocks] = e.to(torch.uint8)
    kept = kept.reshape(m, -1, 4, 4).transpose(2, 3).reshape(m, -1)
    return (whole[:, 0::2] | whole[:, 1::2] << 4).contiguous(), kept.contiguous()


def _micro_values(q, e):
    """The values of codes [rows, blocks, 32]."""
    half = (q & 7).float()
    a = torch.where(half < 4, half * 0.5, torch.where(half < 6, half - 2, half * 2 - 8))
    return torch.where(q >= 8, -a, a) * _power(e)[:, :, None]


def _load(codes, exponents, columns):
    """The values that kept codes and exponents stand for."""
    m = codes.shape[0]
    q = torch.stack((codes & 15, codes >> 4), 2).reshape(m, -1, 32)
    e = exponents.reshape(m, -1, 4, 4).transpose(2, 3).reshape(m, -1)[:, :q.shape[1]].int()
    return _micro_values(q, e).reshape(m, -1)[:, :columns]


def _e4m3_values(x):
    """FP32 rows rounded to E4M3 blocks of 128."""
    m, k = x.shape
    blocks = -(-k // 128)
    b = _padded(x, m, blocks * 128).reshape(m, blocks, 128)
    e = _exponents(b.abs().amax(2), 8, 0x600000)
    q = (b * _power(254 - e)[:, :, None]).to(E4M3).float()
    return (q * _power(e)[:, :, None]).reshape(m, -1)[:, :k]


def _row_values(x, codes):
    if codes == "e4m3":
        return _e4m3_values(x)
    return _micro_values(*_micro_codes(x)).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _sort(ids, count):
    """(offsets of each expert's rows, the choice that each row holds, the row of each choice)."""
    flat = ids.reshape(-1)
    flat = torch.where((flat >= 0) & (flat < count), flat, count)
    order = torch.sort(flat, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(order.numel(), device=order.device)
    offsets = torch.zeros(count + 1, dtype=torch.int64, device=order.device)
    offsets[1:] = (flat[:, None] == torch.arange(count, device=order.device)).sum(0).cumsum(0)
    return offsets, order, places


def _plain_routed(state):
    case, dtype = state["case"], DTYPES[state["case"]["dtype"]]
    t, j = state["ids"].shape
    offsets, order, places = _sort(state["ids"], case["experts"])
    here = (torch.arange(t * j, device=order.device) < offsets[-1])[:, None]
    rows_ = torch.where(here, state["x"].float()[order // j], 0.0).to(dtype)
    used = (places < offsets[-1]).reshape(t, j)
    w = torch.where(used, state["weights"], 0.0)
    y = torch.zeros((t, case["width"]), device=order.device)
    dx = torch.zeros_like(y)
    for i in range(j):
        at = places.reshape(t, j)[:, i]
        y += w[:, i:i + 1] * state["out"].float()[at]
        if case["gradients"]:
            dx += torch.where(used[:, i:i + 1], state["drows"].float()[at], 0.0)
    out = {"offsets": offsets.int(), "order": order.int(), "rows": rows_, "y": y.to(dtype)}
    if case["gradients"]:
        dy = state["dy"].float()
        out["dx"] = dx.to(dtype)
        out["dout"] = torch.where(here, w.reshape(-1)[order][:, None] * dy[order // j], 0.0).to(dtype)
        dots = [(dy * state["out"].float()[places.reshape(t, j)[:, i]]).sum(1) for i in range(j)]
        out["dweights"] = torch.where(used, torch.stack(dots, 1), 0.0)
    return out


def _plain_experts(state):
    case, dtype = state["case"], DTYPES[state["case"]["dtype"]]
    k, n, j = case["inner"], case["outer"], case["each"]
    offsets, order, _ = _sort(state["ids"], case["experts"])
    x = _row_values(state["x"].float(), case["codes"])
    if not case["gradients"]:
        x = x[order // j]
    y = torch.zeros((order.numel(), n), device=order.device)
    bounds = offsets.tolist()
    spans = [(e, slice(bounds[e], bounds[e + 1])) for e in range(case["experts"]) if bounds[e] < bounds[e + 1]]
    for e, span in spans:
        y[span] = x[span] @ _load(state["codes"][e], state["exponents"][e], k).T
    if not case["gradients"]:
        return y.to(dtype)
    dy = _row_values(state["dy"].float(), case["codes"])
    dx = torch.zeros((order.numel(), k), device=order.device)
    for e, span in spans:
        dx[span] = dy[span] @ _load(state["codes_t"][e], state["exponents_t"][e], n).T
    return {"y": y.to(dtype), "dx": dx.to(dtype)}


def _plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rows":
        return _row_values(state["x"].float(), "e2m1").to(dtype)
    if case["op"] == "linear":
        x = _row_values(state["x"].float(), case["codes"])
        y = x @ _load(state["codes"], state["exponents"], case["inner"]).T
        return (y if state["bias"] is None else y + state["bias"]).to(dtype)
    if case["op"] == "step":
        n, k = case["outer"], case["inner"]
        x, dy = _e4m3_values(state["x"].float()), state["dy"].float()
        w = _micro_values(*_tile_codes(state["w"])).reshape(-(-n // 32) * 32, -1)[:n, :k]
        y = x @ w.T + state["bias"]
        return {"y": y.to(dtype), "dx": (_e4m3_values(dy) @ w).to(dtype), "dw": dy.T @ x, "db": dy.sum(0)}
    return _plain_routed(state) if case["op"] == "routed" else _plain_experts(state)


# --------------------------------------------------------------------------------------------------
# One pass


def run(state):
    if not own:
        return _plain(state)
    from tcc_spmm_amd import experts as X
    from tcc_spmm_amd import micro as M
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rows":
        return M.quantize_micro(state["x"]).dequantize(dtype)
    if case["op"] == "linear":
        weight = M.MicroWeight(state["codes"].view(E2M1), state["exponents"], case["inner"])
        return M.linear_micro(state["x"], weight, state["bias"], codes=CODES[case["codes"]])
    if case["op"] == "step":
        weight = M.quantize_weight_micro(state["w"], tiles=True, transposed=True)
        y, kept = M.linear_micro(state["x"], weight, state["bias"], keep=True)
        dx, dw, db = M.linear_micro_backward(state["dy"], kept, weight)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    plan = X.sort_experts(state["ids"], case["experts"])
    if case["op"] == "routed":
        out = {"offsets": plan.offsets, "order": plan.order, "rows": X.gather_experts(state["x"], plan),
               "y": X.combine_experts(state["out"], plan, state["weights"])}
        if case["gradients"]:
            out["dx"] = X.combine_experts(state["drows"], plan)
            out["dout"], out["dweights"] = X.combine_experts_backward(state["dy"], state["out"], plan, state["weights"])
        return out
    codes = CODES[case["codes"]]
    if not case["gradients"]:
        weight = M.MicroWeight(state["codes"].view(E2M1), state["exponents"], case["inner"])
        return X.linear_experts(state["x"], weight, plan, by_token=True, codes=codes)
    weight = M.MicroWeight(state["codes"].view(E2M1), state["exponents"], case["inner"],
                           state["codes_t"].view(E2M1), state["exponents_t"])
    return {"y": X.linear_experts(state["x"], weight, plan, codes=codes),
            "dx": X.linear_experts(state["dy"], weight.transposed(), plan, codes=codes)}


# --------------------------------------------------------------------------------------------------
# The definition in 64 bits, written apart from the plain form


def _two_to(e):
    """2^e in 64 bits, from its bits: the GPU's pow and exp2 may be a last bit off."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _to_grid(v, peak, top, bits, low):
    """v [.., with its block's peak broadcast] on the grid that the block's power of two gives: codes up to `top`, with
    `bits` after the leading one and 2^low the smallest normal."""
    fraction, power = torch.frexp(peak)  # peak = fraction * 2^power, 0.5 <= fraction < 1
    limit, high = math.frexp(top)
    e = torch.clamp(power - high + (fraction > limit).int(), min=-126)
    e = torch.where(peak == 0, torch.zeros_like(e), e)
    v = v / _two_to(e)
    unit = _two_to(torch.clamp(torch.frexp(v)[1] - 1, min=low) - bits)
    return torch.round(v / unit) * unit * _two_to(e)


def _grid_rows(x, codes):
    size, top, bits, low = (128, 448.0, 3, -6) if codes == "e4m3" else (32, 6.0, 1, 0)
    out = torch.empty_like(x)
    whole = x.shape[1] // size * size
    if whole:
        part = x[:, :whole].reshape(x.shape[0], -1, size)
        out[:, :whole] = _to_grid(part, part.abs().amax(2, keepdim=True), top, bits, low).reshape(x.shape[0], -1)
    if whole < x.shape[1]:
        part = x[:, whole:]
        out[:, whole:] = _to_grid(part, part.abs().amax(1, keepdim=True), top, bits, low)
    return out


def _grid_tiles(w):
    out = torch.empty_like(w)
    for r in range(0, w.shape[0], 32):
        band = w[r:r + 32]
        peak = band.abs().amax(0)
        for_block = torch.nn.functional.pad(peak, (0, -peak.numel() % 32)).reshape(-1, 32).amax(1)
        out[r:r + 32] = _to_grid(band, for_block.repeat_interleave(32)[:w.shape[1]], 6.0, 1, 0)
    return out


def _kept_values(codes, exponents, columns):
    """The numbers that kept 4-bit codes stand for."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64,
                         device=codes.device)
    v = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.float64, device=codes.device)
    v[:, 0::2], v[:, 1::2] = table[(codes % 16).long()], table[(codes // 16).long()]
    for b in range(-(-columns // 32)):
        at = 16 * (b // 16) + 4 * (b % 4) + b // 4 % 4
        v[:, 32 * b:32 * b + 32] *= _two_to(exponents[:, at:at + 1].int() - 127)
    return v[:, :columns]


def _lists(ids, count):
    """Expert by expert, the choices that go to it, in their order; those that go nowhere; and all of them."""
    flat = ids.reshape(-1)
    lists = [torch.nonzero(flat == e).reshape(-1) for e in range(count)]
    rest = torch.nonzero((flat < 0) | (flat >= count)).reshape(-1)
    return lists, rest, torch.cat([*lists, rest])


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rows":
        return _grid_rows(state["x"].double(), "e2m1")
    if case["op"] == "linear":
        w = _kept_values(state["codes"], state["exponents"], case["inner"])
        y = torch.matmul(_grid_rows(state["x"].double(), case["codes"]), w.t())
        if case["bias"]:
            y += state["bias"].double()
        return y
    if case["op"] == "step":
        x, dy, w = _grid_rows(state["x"].double(), "e4m3"), state["dy"].double(), _grid_tiles(state["w"].double())
        return {"y": torch.matmul(x, w.t()) + state["bias"].double(), "dx": torch.matmul(_grid_rows(dy, "e4m3"), w),
                "dw": torch.matmul(dy.t(), x), "db": dy.sum(0)}
    lists, rest, order = _lists(state["ids"], case["experts"])
    token, here = order // case["each"], order.numel() - rest.numel()
    starts = torch.tensor([0] + [part.numel() for part in lists], device=DEVICE).cumsum(0)
    if case["op"] == "routed":
        gathered = state["x"].double()[token]
        gathered[here:] = 0
        w = state["weights"].double().reshape(-1)[order]
        w[here:] = 0
        y = torch.zeros(state["x"].shape, dtype=torch.float64, device=DEVICE)
        # the same token's rows of one expert are one row, so that an expert's sums touch each token once
        for e, part in enumerate(lists):
            span = slice(int(starts[e]), int(starts[e + 1]))
            y[token[span]] += w[span, None] * state["out"][span].double()
        out = {"offsets": starts.int(), "order": order.int(), "rows": gathered, "y": y}
        if case["gradients"]:
            dx, dy = torch.zeros_like(y), state["dy"].double()[token]
            for e, part in enumerate(lists):
                span = slice(int(starts[e]), int(starts[e + 1]))
                dx[token[span]] += state["drows"][span].double()
            dots = torch.zeros(order.numel(), dtype=torch.float64, device=DEVICE)
            dots[order[:here]] = (dy[:here] * state["out"][:here].double()).sum(1)
            out.update(dx=dx, dout=w[:, None] * dy, dweights=dots.reshape(state["ids"].shape))
        return out
    k, n = case["inner"], case["outer"]
    x = _grid_rows(state["x"].double(), case["codes"])
    x = x if case["gradients"] else x[token]
    y = torch.zeros((order.numel(), n), dtype=torch.float64, device=DEVICE)
    dx = torch.zeros((order.numel(), k), dtype=torch.float64, device=DEVICE)
    dy = _grid_rows(state["dy"].double(), case["codes"]) if case["gradients"] else None
    for e, part in enumerate(lists):
        if not part.numel():
            continue
        span = slice(int(starts[e]), int(starts[e + 1]))
        w = _kept_values(state["codes"][e], state["exponents"][e], k)
        y[span] = torch.matmul(x[span], w.t())
        if case["gradients"]:
            dx[span] = torch.matmul(dy[span], w)
    return {"y": y, "dx": dx} if case["gradients"] else y
