"""Layers of many experts on torch tensors (Python mirror of include/experts.h): tokens sorted by expert and back, and the
experts' products with weights in microscaled 4-bit blocks (tcc_spmm_amd.micro).

A router chooses some of the experts for each token. sort_experts makes a plan of the choices: rows in the experts' order.
gather_experts brings tokens into that order, combine_experts brings rows back and adds each token's, by their
weights; linear_experts multiplies each row with its expert's weight, and can take the tokens as they are. expert_gather,
expert_combine and expert_linear put the three under autograd; the experts' weights are frozen there, what is
trained is the router and what lies in front.

Every computation runs in the HIP kernels of libtcc_spmm.so; there is no fallback. Streams, layouts and types are taken as
tcc_spmm_amd.blocks takes them. Nothing waits for the device: how many rows an expert has stays there.
"""
from __future__ import annotations

import torch

from ._lib import check, lib
from .blocks import (_TYPES, E4M3, BlockTensor, _away, _dense, _float_bias, _recorded, _rows, _same_device, _stream,
                     _stride)
from .micro import _FORMATS, MicroTensor, MicroWeight, _code_pitch, _format, _laid, _workspace

MAX_EXPERTS = 1024
MAX_EACH = 1024


class ExpertPlan:
    """Choices of tokens sorted by expert, int32 tensors: `order` [choices] holds the choice of each sorted row (of token
    order // each), those of one expert in their own order and those for none of 0 .. experts - 1 last; `places` [choices] the
    row of each choice; expert e's rows are offsets[e] to offsets[e + 1]. `lead` is the tokens' shape."""

    __slots__ = ("offsets", "order", "places", "lead", "each", "choices", "experts", "device")

    def __init__(self, offsets: torch.Tensor, order: torch.Tensor, places: torch.Tensor, lead, each: int):
        lead = tuple(lead)
        tokens = 1
        for n in lead:
            tokens *= n
        for t, name in ((offsets, "offsets"), (order, "order"), (places, "places")):
            if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 vector")
            _same_device(offsets.device, t)
        if not 2 <= offsets.numel() <= MAX_EXPERTS + 1:
            raise ValueError(f"experts must be 1 to {MAX_EXPERTS}")
        if not 1 <= each <= MAX_EACH:
            raise ValueError(f"choices of a token must be 1 to {MAX_EACH}")
        if order.numel() != tokens * each or places.numel() != tokens * each:
            raise ValueError(f"order and places must have {tokens * each} elements")
        _fill(self, offsets, order, places, lead, each)

    @property
    def tokens(self) -> int:
        return self.choices // self.each


def _fill(plan, offsets, order, places, lead, each) -> ExpertPlan:
    plan.offsets, plan.order, plan.places, plan.lead, plan.each = offsets, order, places, lead, each
    plan.choices, plan.experts, plan.device = order.numel(), offsets.numel() - 1, offsets.device
    return plan


def _plan(offsets, order, places, lead, each) -> ExpertPlan:
    """An ExpertPlan of tensors that are laid out as its constructor would check."""
    return _fill(ExpertPlan.__new__(ExpertPlan), offsets, order, places, lead, each)


def _here(device, plan: ExpertPlan) -> None:
    if device != plan.device:
        raise ValueError(f"tensor on {device}, expected {plan.device}")


def _sorted_rows(t: torch.Tensor, plan: ExpertPlan, name: str, columns: int | None = None) -> None:
    _dense(t, name, columns)
    if t.dim() != 2 or t.shape[0] != plan.choices:
        raise ValueError(f"{name} must be [{plan.choices}, columns], got {list(t.shape)}")
    _here(t.device, plan)


def _token_rows(t: torch.Tensor, plan: ExpertPlan, name: str, columns: int | None = None) -> None:
    _dense(t, name, columns)
    if t.shape[:-1] != plan.lead:
        raise ValueError(f"{name} must be {[*plan.lead, 'columns']}, got {list(t.shape)}")
    _here(t.device, plan)


def _weights(weights, plan: ExpertPlan) -> None:
    if weights is None:
        return
    if weights.dtype not in _TYPES:
        raise ValueError(f"weights must be float32, bfloat16 or float16, got {weights.dtype}")
    if weights.shape != (*plan.lead, plan.each):
        raise ValueError(f"weights must be {[*plan.lead, plan.each]}, got {list(weights.shape)}")
    _here(weights.device, plan)


def sort_experts(experts: torch.Tensor, count: int, stream=None) -> ExpertPlan:
    """sortExperts: the plan of choices [..., each], int32 or int64 numbers of `count` experts; others than 0 .. count - 1
    are for experts that are not here (their rows are zeros, and add nothing). Repeated calls give the same plan."""
    if experts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"experts must be int32 or int64, got {experts.dtype}")
    if experts.dim() < 1 or not 1 <= experts.shape[-1] <= MAX_EACH:
        raise ValueError(f"experts must be [..., choices], of 1 to {MAX_EACH} choices each")
    if not 1 <= count <= MAX_EXPERTS:
        raise ValueError(f"experts must be 1 to {MAX_EXPERTS}, got {count}")
    device = experts.device
    away = _away(device, stream)
    if away:
        with away:
            return sort_experts(experts, count)
    ids = experts.contiguous()
    choices = ids.numel()
    # One allocation: the lists of a plan live and end together.
    lists = torch.empty(2 * choices + count + 1, dtype=torch.int32, device=device)
    offsets, order, places = lists.split_with_sizes((count + 1, choices, choices))
    _space, at, size = _workspace("tcc_sort_experts_workspace", (choices, count), device)
    check(lib().tcc_sort_experts(ids.data_ptr(), ids.element_size(), offsets.data_ptr(), order.data_ptr(), places.data_ptr(),
                                 choices, count, at, size, _stream(device.index)))
    return _plan(offsets, order, places, tuple(ids.shape[:-1]), ids.shape[-1])


def gather_experts(x: torch.Tensor, plan: ExpertPlan, stream=None) -> torch.Tensor:
    """gatherExperts: rows [choices, width] in the experts' order, of tokens x [..., width]; rows of no expert are zeros.
    Its gradient is combine_experts without weights."""
    _token_rows(x, plan, "x")
    device, width = x.device, x.shape[-1]
    away = _away(device, stream)
    if away:
        with away:
            return gather_experts(x, plan)
    flat, _, _, stride = _laid(x)
    rows = torch.empty((plan.choices, width), dtype=x.dtype, device=device)
    check(lib().tcc_gather_experts(flat.data_ptr(), stride, _TYPES[x.dtype], plan.offsets.data_ptr(),
                                   plan.places.data_ptr(), plan.choices, plan.each, plan.experts, rows.data_ptr(), width,
                                   width, _stream(device.index)))
    return rows


def combine_experts(rows: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor | None = None,
                    stream=None) -> torch.Tensor:
    """combineExperts: for each token the sum of its choices' rows by their weights [..., each] (None: ones), added in
    float32 in the choices' order; choices for no expert here add nothing. [..., width] in the rows' type."""
    _sorted_rows(rows, plan, "rows")
    _weights(weights, plan)
    device, width = rows.device, rows.shape[-1]
    away = _away(device, stream)
    if away:
        with away:
            return combine_experts(rows, plan, weights)
    flat, _, _, stride = _laid(rows)
    weights = None if weights is None else weights.contiguous()
    y = torch.empty((*plan.lead, width), dtype=rows.dtype, device=device)
    check(lib().tcc_combine_experts(flat.data_ptr(), stride, _TYPES[rows.dtype], plan.offsets.data_ptr(),
                                    plan.places.data_ptr(), plan.choices, plan.each, plan.experts,
                                    0 if weights is None else weights.data_ptr(),
                                    0 if weights is None else _TYPES[weights.dtype], y.data_ptr(), width, width,
                                    _stream(device.index)))
    return y


def combine_experts_backward(dy: torch.Tensor, rows: torch.Tensor | None, plan: ExpertPlan,
                             weights: torch.Tensor | None = None, *, need=(True, True), stream=None):
    """combineExpertsBackward: (drows [choices, width] in dy's type, dweights in the weights' type and shape) of
    combine_experts, None for what `need` leaves out; rows are read for dweights alone."""
    _token_rows(dy, plan, "dy")
    _weights(weights, plan)
    device, width = dy.device, dy.shape[-1]
    if not (need[0] or need[1]):
        raise ValueError("neither the rows' nor the weights' gradient is asked for")
    if need[1]:
        if weights is None or rows is None:
            raise ValueError("the weights' gradient needs the weights and the rows")
        _sorted_rows(rows, plan, "rows", width)
        _same_device(device, rows)
        if rows.dtype != dy.dtype:
            raise ValueError(f"rows are {rows.dtype}, dy {dy.dtype}")
    away = _away(device, stream)
    if away:
        with away:
            return combine_experts_backward(dy, rows, plan, weights, need=need)
    flat, _, _, stride = _laid(dy)
    rows = _rows(rows) if need[1] else None
    weights = None if weights is None else weights.contiguous()
    drows = torch.empty((plan.choices, width), dtype=dy.dtype, device=device) if need[0] else None
    dweights = torch.empty_like(weights) if need[1] else None
    check(lib().tcc_combine_experts_backward(
        flat.data_ptr(), stride, rows.data_ptr() if need[1] else 0, _stride(rows) if need[1] else 0,
        _TYPES[dy.dtype], plan.offsets.data_ptr(), plan.places.data_ptr(), plan.choices, plan.each, plan.experts,
        0 if weights is None else weights.data_ptr(), 0 if weights is None else _TYPES[weights.dtype],
        drows.data_ptr() if need[0] else 0, width, dweights.data_ptr() if need[1] else 0, width, _stream(device.index)))
    return drows, dweights


def _stack(weight: MicroWeight, plan: ExpertPlan) -> None:
    if weight.experts != plan.experts:
        raise ValueError(f"weight must be a stack of {plan.experts} experts' weights")


def _gather_codes(x: BlockTensor | MicroTensor, plan: ExpertPlan) -> BlockTensor | MicroTensor:
    """Tokens' codes and exponents as rows in the experts' order: both are whole numbers of pairs of bytes, which a gather
    moves as they are."""
    moved = type(x).__new__(type(x))  # laid out as x is
    moved.columns = x.columns
    for name in ("codes", "exponents"):
        t = getattr(x, name)
        pairs = t.view(torch.uint8).view(torch.bfloat16).reshape(*plan.lead, -1)
        setattr(moved, name, gather_experts(pairs, plan).view(torch.uint8).view(t.dtype))
    return moved


def _stack_bias(bias, experts: int, outer: int, device) -> int:
    if bias is None:
        return 0
    if bias.dtype != torch.float32 or tuple(bias.shape) != (experts, outer) or not bias.is_contiguous():
        raise ValueError(f"bias must be a contiguous float32 [{experts}, {outer}] tensor")
    _same_device(device, bias)
    return bias.data_ptr()


def matmul_experts(x: BlockTensor | MicroTensor, weight: MicroWeight, plan: ExpertPlan,
                   bias: torch.Tensor | None = None, *, by_token: bool = False, dtype=torch.bfloat16,
                   stream=None) -> torch.Tensor:
    """matmulExperts: the rows of linear_experts for x already in E4M3 blocks or in microscaled ones, a row for each sorted row
    or, by_token, for each token. dtype is that of the result, with the sums of matmul_micro."""
    if x.codes.dtype not in _FORMATS:
        raise ValueError("x must have float8_e4m3fn or float4_e2m1fn_x2 codes")
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    _stack(weight, plan)
    if x.columns != weight.columns:
        raise ValueError(f"x has rows of {x.columns} elements, expected {weight.columns}")
    if x.rows != (plan.tokens if by_token else plan.choices):
        raise ValueError(f"x must have {plan.tokens if by_token else plan.choices} rows, got {x.rows}")
    device, outer = x.codes.device, weight.rows
    _here(device, plan)
    _same_device(device, weight.codes)
    at_bias = _stack_bias(bias, plan.experts, outer, device)
    away = _away(device, stream)
    if away:
        with away:
            return matmul_experts(x, weight, plan, bias, by_token=by_token, dtype=dtype)
    if by_token and x.codes.numel() >= 1 << 31:
        # The kernels reach a token's codes by 32 bits.
        x, by_token = _gather_codes(x, plan), False
    y = torch.empty((plan.choices, outer), dtype=dtype, device=device)
    check(lib().tcc_matmul_experts(x.codes.data_ptr(), x.exponents.data_ptr(), _FORMATS[x.codes.dtype], by_token,
                                   weight.codes.data_ptr(), weight.exponents.data_ptr(), at_bias, y.data_ptr(), outer,
                                   _TYPES[dtype], plan.offsets.data_ptr(), plan.order.data_ptr(), plan.choices, plan.each,
                                   plan.experts, x.columns, outer, _stream(device.index)))
    return y


def linear_experts(x: torch.Tensor, weight: MicroWeight, plan: ExpertPlan, bias: torch.Tensor | None = None, *,
                   by_token: bool = False, codes=E4M3, stream=None) -> torch.Tensor:
    """linearExperts: rows [choices, outer] in x's type, each Q(x) times its expert's weight of the stack, plus that
    expert's bias of [experts, outer]; rows of no expert are zeros. x is [choices, inner] in the experts' order or, by_token, the
    tokens [..., inner] themselves, which are then never copied. Codes and sums are those of linear_micro."""
    kind = _format(codes)
    _stack(weight, plan)
    inner, outer = weight.columns, weight.rows
    (_token_rows if by_token else _sorted_rows)(x, plan, "x", inner)
    device = x.device
    _same_device(device, weight.codes)
    at_bias = _stack_bias(bias, plan.experts, outer, device)
    away = _away(device, stream)
    if away:
        with away:
            return linear_experts(x, weight, plan, bias, by_token=by_token, codes=codes)
    if by_token and plan.choices // plan.each * _code_pitch(inner) * (2 - kind) >= 1 << 31:
        # The kernels reach a token's codes by 32 bits.
        x, by_token = gather_experts(x, plan), False
    flat, _, _, stride = _laid(x)
    dtype = _TYPES[x.dtype]
    y = torch.empty((plan.choices, outer), dtype=x.dtype, device=device)
    _space, at, size = _workspace("tcc_linear_experts_workspace",
                                  (plan.choices, plan.each, plan.experts, by_token, inner, outer, dtype, kind), device)
    check(lib().tcc_linear_experts(flat.data_ptr(), stride, dtype, kind, by_token, weight.codes.data_ptr(),
                                   weight.exponents.data_ptr(), at_bias, y.data_ptr(), outer, plan.offsets.data_ptr(),
                                   plan.order.data_ptr(), plan.choices, plan.each, plan.experts, inner, outer, at, size,
                                   _stream(device.index)))
    return y


# --------------------------------------------------------------------------------------------------
# Under autograd


# Plans and frozen weights are not saved as autograd saves tensors, whose hooks may move or copy what they are given: a
# Function holds them, and their versions, itself.


def _hold(ctx, plan: ExpertPlan, *weights: torch.Tensor) -> None:
    ctx.plan = _plan(plan.offsets, plan.order, plan.places, plan.lead, plan.each)
    ctx.versions = _versions(ctx.plan, weights)


def _versions(plan: ExpertPlan, weights):
    """Inference tensors, which have no versions, count as unchanged."""
    return [None if t.is_inference() else t._version for t in (plan.offsets, plan.order, plan.places, *weights)]


def _held(ctx, *weights: torch.Tensor) -> ExpertPlan:
    if _versions(ctx.plan, weights) != ctx.versions:
        raise RuntimeError("the experts' plan or weight has been modified by an inplace operation since the forward pass, "
                           "whose gradient needs it as it was")
    return ctx.plan


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        _hold(ctx, plan)
        return gather_experts(x, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drows):
        return combine_experts(drows, _held(ctx)), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, plan, weights):
        _hold(ctx, plan)
        # rows are what the weights' gradient needs, weights what both do.
        ctx.save_for_backward(rows if ctx.needs_input_grad[2] else None, weights)
        return combine_experts(rows, plan, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rows, weights = ctx.saved_tensors
        need = (ctx.needs_input_grad[0], ctx.needs_input_grad[2])
        drows, dweights = combine_experts_backward(dy, rows, _held(ctx), weights, need=need)
        return drows, None, dweights


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, plan, bias, by_token, codes):
        # Without a gradient of x there is no backward pass.
        back = weight.transposed() if ctx.needs_input_grad[0] and weight.codes_t is not None else None
        if back is not None:
            _hold(ctx, plan, back.codes, back.exponents)
        ctx.call = (back, by_token, codes)
        return linear_experts(x, weight, plan, bias, by_token=by_token, codes=codes)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        back, by_token, codes = ctx.call
        plan = _held(ctx, back.codes, back.exponents)
        dx = linear_experts(dy, back, plan, codes=codes)
        return (combine_experts(dx, plan) if by_token else dx), None, None, None, None, None


def expert_gather(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """gather_experts, differentiable."""
    return _Gather.apply(x, plan) if _recorded() else gather_experts(x, plan)


def expert_combine(rows: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor | None = None) -> torch.Tensor:
    """combine_experts, differentiable in the rows and the weights."""
    return _Combine.apply(rows, plan, weights) if _recorded() else combine_experts(rows, plan, weights)


def expert_linear(x: torch.Tensor, weight: MicroWeight, plan: ExpertPlan, bias: torch.Tensor | None = None, *,
                  by_token: bool = False, codes=E4M3) -> torch.Tensor:
    """linear_experts, differentiable in x; the experts are frozen, their bias is of any type and layout. The gradient goes
    through the output gradient's codes and the weight's transposed copy; by_token each row's is rounded to x's type before a
    token's are added. Under autocast x is cast to its type first."""
    if x.is_cuda and x.dtype in _TYPES and torch.is_autocast_enabled("cuda"):
        x = x.to(torch.get_autocast_dtype("cuda"))
    if not _recorded():
        return linear_experts(x, weight, plan, _float_bias(bias), by_token=by_token, codes=codes)
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("the experts are frozen: their bias has no gradient")
    if x.requires_grad and weight.codes_t is None and torch.is_grad_enabled():
        raise ValueError("x requires a gradient, which needs the weight's transposed copy")
    return _Linear.apply(x, weight, plan, _float_bias(bias), by_token, codes)
