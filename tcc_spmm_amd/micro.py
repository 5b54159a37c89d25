"""Dense layers with weights in microscaled 4-bit blocks on torch tensors (Python mirror of include/micro.h).

32 consecutive elements of a row share one power of two and are held as E2M1 codes, two a byte. A weight is held so, either
by its rows, as it is served, or in tiles of 32 x 32 that share a power, as it is trained, so that its transposed copy holds
the same values. What it is multiplied with is x in E4M3 blocks of 128 (tcc_spmm_amd.blocks), or in microscaled blocks
of its own, at half the bytes and twice the matrix instructions' rate. MicroLinear and micro_linear put the layer under
autograd; its weight gradient is that of the 8-bit layers.

Sums are float32, but for E4M3 rows in 16-bit types, which have the 8-bit matrix instruction's (tcc_spmm_amd.blocks).

Every computation runs in the HIP kernels of libtcc_spmm.so; there is no fallback. Streams, layouts and types are taken as
tcc_spmm_amd.blocks takes them.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from ._lib import check, lib
from .blocks import (_TYPES, E4M3, BlockTensor, _away, _bias, _dense, _float_bias, _new_blocks, _recorded, _rows,
                     _same_device, _stream, _stride, weight_grad_blocks)

BLOCK = 32
E2M1 = torch.float4_e2m1fn_x2

_FORMATS = {E4M3: 0, E2M1: 1}


def _code_pitch(columns: int) -> int:
    return -(-columns // 128) * 64


def _exponent_pitch(columns: int) -> int:
    return -(-columns // 512) * 16


def _check_micro(codes, exponents, columns: int, dims, name: str) -> None:
    if codes.dtype != E2M1:
        raise ValueError(f"{name} codes must be {E2M1}, got {codes.dtype}")
    if exponents.dtype != torch.uint8:
        raise ValueError(f"{name} exponents must be torch.uint8, got {exponents.dtype}")
    if columns < 1:
        raise ValueError(f"{name} needs at least one column")
    pitch, exponent_pitch = _code_pitch(columns), _exponent_pitch(columns)
    if codes.dim() not in dims or codes.shape[-1] != pitch or not codes.is_contiguous():
        raise ValueError(f"{name} codes must be contiguous [{'.., ' if 3 in dims else ''}rows, {pitch}]")
    if exponents.shape != (*codes.shape[:-1], exponent_pitch) or not exponents.is_contiguous():
        raise ValueError(f"{name} exponents must be contiguous {[*codes.shape[:-1], exponent_pitch]}")
    if exponents.device != codes.device:
        raise ValueError(f"tensor on {exponents.device}, expected {codes.device}")


class MicroTensor:
    """Rows of `columns` elements in microscaled blocks: codes float4_e2m1fn_x2 [rows, 64 * ceil(columns / 128)], zero past
    the row's end, and exponents uint8 [rows, 16 * ceil(columns / 512)], 127 past it. Byte e scales its block by 2^(e -
    127), 255 makes it NaN; block b's is byte 16 * (b // 16) + 4 * (b % 4) + b // 4 % 4 of its row."""

    __slots__ = ("codes", "exponents", "columns")

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, columns: int):
        _check_micro(codes, exponents, columns, (2,), "micro")
        self.codes, self.exponents, self.columns = codes, exponents, columns

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    def dequantize(self, dtype=torch.float32, stream=None) -> torch.Tensor:
        return dequantize_micro(self, dtype, stream)


class MicroWeight:
    """A weight [outer, inner], or a stack of them [experts, outer, inner], in microscaled blocks along `inner`: codes and
    exponents of its rows as a MicroTensor's, and for the input gradient the transposed weight's, if it is in tiles. `rows` is
    outer, of one weight; `experts` the number of a stack, None for one weight."""

    __slots__ = ("codes", "exponents", "columns", "codes_t", "exponents_t", "rows", "experts")

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, columns: int,
                 codes_t: torch.Tensor | None = None, exponents_t: torch.Tensor | None = None):
        _check_micro(codes, exponents, columns, (2, 3), "weight")
        if not codes.numel():
            raise ValueError("a weight needs at least one row")
        if (codes_t is None) != (exponents_t is None):
            raise ValueError("transposed codes and exponents come together")
        if codes_t is not None:
            _check_micro(codes_t, exponents_t, codes.shape[-2], (codes.dim(),), "transposed weight")
            if codes_t.shape[:-1] != (*codes.shape[:-2], columns):
                raise ValueError(f"transposed weight must have {[*codes.shape[:-2], columns]} rows, "
                                 f"got {list(codes_t.shape[:-1])}")
            if codes_t.device != codes.device:
                raise ValueError(f"tensor on {codes_t.device}, expected {codes.device}")
        _fill(self, codes, exponents, columns, codes_t, exponents_t)

    def transposed(self) -> "MicroWeight":
        """The transposed weight's view of the same codes."""
        if self.codes_t is None:
            raise ValueError("the weight was quantized without its transposed copy")
        return _weight(self.codes_t, self.exponents_t, self.rows, self.codes, self.exponents)

    def dequantize(self, dtype=torch.float32, stream=None) -> torch.Tensor:
        rows = MicroTensor(self.codes.flatten(0, -2), self.exponents.flatten(0, -2), self.columns)
        return dequantize_micro(rows, dtype, stream).reshape(*self.codes.shape[:-1], self.columns)


def _fill(weight, codes, exponents, columns, codes_t, exponents_t) -> MicroWeight:
    weight.codes, weight.exponents, weight.columns = codes, exponents, columns
    weight.codes_t, weight.exponents_t = codes_t, exponents_t
    weight.rows, weight.experts = codes.shape[-2], codes.shape[0] if codes.dim() == 3 else None
    return weight


def _weight(codes, exponents, columns, codes_t, exponents_t) -> MicroWeight:
    """A MicroWeight of tensors that are laid out as its constructor would check."""
    return _fill(MicroWeight.__new__(MicroWeight), codes, exponents, columns, codes_t, exponents_t)


def _new_micro(shape, columns: int, device):
    """Codes and exponents of rows [*shape]."""
    return (torch.empty((*shape, _code_pitch(columns)), dtype=E2M1, device=device),
            torch.empty((*shape, _exponent_pitch(columns)), dtype=torch.uint8, device=device))


def _laid(t: torch.Tensor):
    """t as rows (_rows), their number, their columns and their stride."""
    if t.dim() == 2 and t.is_contiguous():
        rows, columns = t.shape
        return t, rows, columns, columns
    t = _rows(t)
    return t, t.shape[0], t.shape[1], _stride(t)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(query: str, *sizes) -> int:
    """What the library's query says for these sizes, of which it is a function; asking costs 2 us."""
    size = C.c_size_t()
    check(getattr(lib(), query)(*sizes, C.byref(size)))
    return size.value


def _workspace(query: str, sizes, device):
    size = _workspace_bytes(query, *sizes)
    if not size:
        return None, 0, 0
    space = torch.empty(size, dtype=torch.uint8, device=device)
    return space, space.data_ptr(), size


def _format(codes) -> int:
    if codes not in _FORMATS:
        raise ValueError(f"codes must be float8_e4m3fn or float4_e2m1fn_x2, got {codes}")
    return _FORMATS[codes]


def _single(weight: MicroWeight) -> None:
    if weight.experts is not None:
        raise ValueError("the weight is a stack of experts' weights")


def quantize_micro(x: torch.Tensor, stream=None) -> MicroTensor:
    """quantizeMicro: x's rows (all leading dimensions) in microscaled blocks along the last one."""
    _dense(x, "x")
    device = x.device
    away = _away(device, stream)
    if away:
        with away:
            return quantize_micro(x)
    x, rows, columns, stride = _laid(x)
    out = MicroTensor.__new__(MicroTensor)  # laid out as its constructor would check
    out.codes = codes = torch.empty((rows, -(-columns // 128) * 64), dtype=E2M1, device=device)
    out.exponents = exponents = torch.empty((rows, -(-columns // 512) * 16), dtype=torch.uint8, device=device)
    out.columns = columns
    check(lib().tcc_quantize_micro(x.data_ptr(), stride, _TYPES[x.dtype], codes.data_ptr(), exponents.data_ptr(), rows, columns,
                                   _stream(device.index)))
    return out


def dequantize_micro(x: MicroTensor, dtype=torch.float32, stream=None) -> torch.Tensor:
    """dequantizeMicro: the values [rows, columns] that the blocks stand for."""
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    device = x.codes.device
    away = _away(device, stream)
    if away:
        with away:
            return dequantize_micro(x, dtype)
    rows, columns = x.rows, x.columns
    out = torch.empty((rows, columns), dtype=dtype, device=device)
    check(lib().tcc_dequantize_micro(x.codes.data_ptr(), x.exponents.data_ptr(), out.data_ptr(), columns, _TYPES[dtype],
                                     rows, columns, _stream(device.index)))
    return out


def quantize_weight_micro(w: torch.Tensor, *, tiles: bool = False, transposed: bool = False, stream=None) -> MicroWeight:
    """w [outer, inner] or [experts, outer, inner] in microscaled blocks along `inner`: of its rows (quantizeMicro), the
    closer ones, or in tiles of 32 x 32 (quantizeWeightMicro). `transposed` adds the copy that the input gradient needs,
    which only tiles can hold with the same values."""
    _dense(w, "w")
    if w.dim() not in (2, 3) or not w.numel():
        raise ValueError("w must be [outer, inner] or [experts, outer, inner]")
    if transposed and not tiles:
        raise ValueError("a transposed copy holds the same values only of a weight in tiles")
    outer, inner = w.shape[-2:]
    device = w.device
    away = _away(device, stream)
    if away:
        with away:
            return quantize_weight_micro(w, tiles=tiles, transposed=transposed)
    stack = w.shape[:-2]
    if not tiles:
        rows = quantize_micro(w)
        return _weight(rows.codes.reshape(*stack, outer, -1), rows.exponents.reshape(*stack, outer, -1), inner, None, None)
    w = _rows(w)
    codes, exponents = _new_micro((*stack, outer), inner, device)
    codes_t, exponents_t = _new_micro((*stack, inner), outer, device) if transposed else (None, None)
    check(lib().tcc_quantize_weight_micro(
        w.data_ptr(), _stride(w), _TYPES[w.dtype], codes.data_ptr(), exponents.data_ptr(),
        codes_t.data_ptr() if transposed else 0, exponents_t.data_ptr() if transposed else 0,
        stack[0] if stack else 1, outer, inner, _stream(device.index)))
    return _weight(codes, exponents, inner, codes_t, exponents_t)


def matmul_micro(x: BlockTensor | MicroTensor, weight: MicroWeight, bias: torch.Tensor | None = None,
                 dtype=torch.bfloat16, stream=None) -> torch.Tensor:
    """matmulMicro: x weight^T + bias [rows, outer] for x already in E4M3 blocks or in microscaled ones. dtype is that of the
    result; with E4M3 blocks a 16-bit one has the 8-bit matrix instruction's sums, all others have float32 sums."""
    if x.codes.dtype not in _FORMATS:
        raise ValueError("x must have float8_e4m3fn or float4_e2m1fn_x2 codes")
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    _single(weight)
    if x.columns != weight.columns:
        raise ValueError(f"x has rows of {x.columns} elements, expected {weight.columns}")
    device, outer = x.codes.device, weight.rows
    _same_device(device, weight.codes)
    at_bias = _bias(bias, outer, device)
    away = _away(device, stream)
    if away:
        with away:
            return matmul_micro(x, weight, bias, dtype)
    y = torch.empty((x.rows, outer), dtype=dtype, device=device)
    check(lib().tcc_matmul_micro(x.codes.data_ptr(), x.exponents.data_ptr(), _FORMATS[x.codes.dtype],
                                 weight.codes.data_ptr(), weight.exponents.data_ptr(), at_bias, y.data_ptr(), outer,
                                 _TYPES[dtype], x.rows, x.columns, outer, _stream(device.index)))
    return y


def linear_micro(x: torch.Tensor, weight: MicroWeight, bias: torch.Tensor | None = None, *, codes=E4M3,
                 keep: bool = False, stream=None):
    """linearMicro: y = Q(x) weight^T + bias in x's type, for x [..., inner] quantized on the way, into E4M3 blocks or, with
    codes=E2M1, into microscaled ones; sums are those of matmul_micro with x's type. With keep=True returns (y, x's
    BlockTensor): what the weight gradient needs of x, in 8 bits."""
    kind = _format(codes)
    if keep and codes != E4M3:
        raise ValueError("the weight gradient takes float8_e4m3fn codes of x: no others are kept")
    _single(weight)
    inner, outer = weight.columns, weight.rows
    _dense(x, "x", inner)
    device = x.device
    _same_device(device, weight.codes)
    at_bias = _bias(bias, outer, device)
    dtype = _TYPES[x.dtype]
    away = _away(device, stream)
    if away:
        with away:
            return linear_micro(x, weight, bias, codes=codes, keep=keep)
    flat, rows, _, stride = _laid(x)
    y = torch.empty((rows, outer) if x.dim() == 2 else (*x.shape[:-1], outer), dtype=x.dtype, device=device)
    kept = _new_blocks(rows, inner, E4M3, device) if keep else None
    _space, at, size = _workspace("tcc_linear_micro_workspace", (rows, inner, outer, dtype, kind, keep), device)
    check(lib().tcc_linear_micro(flat.data_ptr(), stride, dtype, kind, weight.codes.data_ptr(),
                                 weight.exponents.data_ptr(), at_bias, y.data_ptr(), outer,
                                 kept.codes.data_ptr() if keep else 0, kept.exponents.data_ptr() if keep else 0,
                                 rows, inner, outer, at, size, _stream(device.index)))
    return (y, kept) if keep else y


def linear_micro_backward(dy: torch.Tensor, kept: BlockTensor | None, weight: MicroWeight | None, *,
                          need=(True, True, True), stream=None):
    """(dx, dw, db) of linear_micro, None for what `need` leaves out. dx = Q(dy) weight in dy's type, with dy in E4M3 blocks,
    from the weight's transposed copy; dw and db are float32, dw from the kept blocks and dy in full, db from dy."""
    dx = dw = db = None
    if need[0]:
        dx = linear_micro(dy, weight.transposed(), stream=stream)
    if need[1] or need[2]:
        dw, db = weight_grad_blocks(dy, kept if need[1] else None, bias=bool(need[2]), stream=stream)
    return dx, dw, db


# --------------------------------------------------------------------------------------------------
# Under autograd


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias):
        grad_x, grad_w, _ = ctx.needs_input_grad
        weight = quantize_weight_micro(w, tiles=True, transposed=grad_x)
        out = linear_micro(x, weight, _float_bias(bias), keep=grad_w)
        y, kept = out if grad_w else (out, None)
        ctx.save_for_backward(*((kept.codes, kept.exponents) if grad_w else (None, None)),
                              *((weight.codes_t, weight.exponents_t) if grad_x else (None, None)))
        ctx.shape, ctx.types = w.shape, (w.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        codes, exponents, codes_t, exponents_t = ctx.saved_tensors
        outer, inner = ctx.shape
        dx = dw = db = None
        if codes_t is not None:
            dx = linear_micro(dy, MicroWeight(codes_t, exponents_t, outer))
        if codes is not None or ctx.needs_input_grad[2]:
            kept = None if codes is None else BlockTensor(codes, exponents, inner)
            dw, db = weight_grad_blocks(dy, kept, bias=ctx.needs_input_grad[2])
            dw = None if dw is None else dw.to(ctx.types[0])
            db = None if db is None else db.to(ctx.types[1])
        return dx, dw, db


def micro_linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """x w^T + bias with x in E4M3 blocks and w in microscaled tiles, differentiable; w is the master weight, quantized
    in every call. Under autocast x is cast to its type first, as torch's linear casts it; w is quantized and the bias
    added at their own precision."""
    if x.is_cuda and x.dtype in _TYPES and torch.is_autocast_enabled("cuda"):
        x = x.to(torch.get_autocast_dtype("cuda"))
    if w.dim() != 2:
        raise ValueError("w must be [outer, inner]")
    if not _recorded():
        # Inside a Function the mode is off and its arguments still say that they require a gradient.
        return linear_micro(x, quantize_weight_micro(w, tiles=True), _float_bias(bias))
    return _Linear.apply(x, w, bias)


class MicroLinear(torch.nn.Linear):
    """torch.nn.Linear whose weight is multiplied in microscaled tiles, autocast included (micro_linear)."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return micro_linear(x, self.weight, self.bias)

    def serving(self):
        """(MicroWeight, float32 bias or None) for linear_micro, quantized once: the values that it is trained with."""
        bias = None if self.bias is None else self.bias.detach()
        return quantize_weight_micro(self.weight.detach(), tiles=True), _float_bias(bias)
