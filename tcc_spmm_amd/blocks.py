"""Dense layers in 8-bit blocks on torch tensors (Python mirror of include/blocks.h).

128 consecutive elements of a row (of a weight: a tile of 128 x 128) share one power of two and are held
as E4M3 or INT8 codes. On them run a linear layer, whose product is made by the 8-bit matrix
instructions, its input and weight gradients, and activations whose input is kept in 8 bits for the
backward pass. BlockLinear and block_activation put them under autograd.

Sums are float32, but for the products of the layers in 16-bit types: there the 8-bit matrix instruction cuts each of 8
consecutive products off 13 bits below the largest, which makes a sum at most 7 * 2^-13 of its terms' magnitudes wrong
and on random numbers 1.2e-5, a twentieth of a float16 rounding. matmul_blocks with dtype=torch.float32 adds in float32.

Every computation runs in the HIP kernels of libtcc_spmm.so; there is no fallback. Calls are
asynchronous on `stream` (default: the tensors' device's current stream), on which their outputs
and workspaces are allocated. Dense operands are float32, bfloat16 or float16 with any leading
dimensions; rows may lie apart (slices) and start at any element, and what is not laid out in
rows is copied first.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import check, lib

BLOCK = 128
E4M3, INT8 = torch.float8_e4m3fn, torch.int8

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_CODES = {E4M3: 0, INT8: 1}
_KINDS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _blocks(columns: int) -> int:
    return -(-columns // BLOCK)


def _exponent_pitch(columns: int) -> int:
    return -(-_blocks(columns) // 4) * 4


def _check_stored(codes, exponents, columns: int, types, exponent_rows: int | None, name: str) -> None:
    if codes.dtype not in types:
        raise ValueError(f"{name} codes must be {' or '.join(map(str, types))}, got {codes.dtype}")
    if exponents.dtype != torch.uint8:
        raise ValueError(f"{name} exponents must be torch.uint8, got {exponents.dtype}")
    if columns < 1:
        raise ValueError(f"{name} needs at least one column")
    blocks = _blocks(columns)
    if codes.dim() != 2 or codes.shape[1] != blocks * BLOCK or not codes.is_contiguous():
        raise ValueError(f"{name} codes must be contiguous [rows, {blocks * BLOCK}]")
    rows, pitch = codes.shape[0] if exponent_rows is None else exponent_rows, -(-blocks // 4) * 4
    if exponents.shape != (rows, pitch) or not exponents.is_contiguous():
        raise ValueError(f"{name} exponents must be contiguous [{rows}, {pitch}]")
    if exponents.device != codes.device:
        raise ValueError(f"tensor on {exponents.device}, expected {codes.device}")


class BlockTensor:
    """Rows of `columns` elements in blocks: codes (float8_e4m3fn or int8) [rows, 128 * ceil(columns /
    128)], zero past the row's end, and exponents uint8 [rows, 4 * ceil(blocks / 4)]; byte e scales its
    block by 2^(e - 127), 255 makes it NaN."""

    __slots__ = ("codes", "exponents", "columns")

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, columns: int):
        _check_stored(codes, exponents, columns, (E4M3, INT8), None, "block")
        self.codes, self.exponents, self.columns = codes, exponents, columns

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    def dequantize(self, dtype=torch.float32, stream=None) -> torch.Tensor:
        return dequantize_blocks(self, dtype, stream)


class BlockWeight:
    """A weight [outer, inner] in E4M3 tiles of 128 x 128: codes as a BlockTensor's, exponents [ceil(outer /
    128), 4 * ceil(inner blocks / 4)], and for the input gradient the same tiles of the transposed
    weight."""

    __slots__ = ("codes", "exponents", "columns", "codes_t", "exponents_t")

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor, columns: int,
                 codes_t: torch.Tensor | None = None, exponents_t: torch.Tensor | None = None):
        outer = codes.shape[0]
        _check_stored(codes, exponents, columns, (E4M3,), _blocks(outer), "weight")
        if (codes_t is None) != (exponents_t is None):
            raise ValueError("transposed codes and exponents come together")
        if codes_t is not None:
            _check_stored(codes_t, exponents_t, outer, (E4M3,), _blocks(columns), "transposed weight")
            if codes_t.shape[0] != columns:
                raise ValueError(f"transposed weight must have {columns} rows, got {codes_t.shape[0]}")
            if codes_t.device != codes.device:
                raise ValueError(f"tensor on {codes_t.device}, expected {codes.device}")
        self.codes, self.exponents, self.columns = codes, exponents, columns
        self.codes_t, self.exponents_t = codes_t, exponents_t

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    def transposed(self) -> "BlockWeight":
        """The transposed weight's view of the same codes."""
        if self.codes_t is None:
            raise ValueError("the weight was quantized without its transposed copy")
        return _weight(self.codes_t, self.exponents_t, self.rows, self.codes, self.exponents)


def _weight(codes, exponents, columns, codes_t, exponents_t) -> BlockWeight:
    """A BlockWeight of tensors that are laid out as its constructor would check."""
    out = BlockWeight.__new__(BlockWeight)
    out.codes, out.exponents, out.columns = codes, exponents, columns
    out.codes_t, out.exponents_t = codes_t, exponents_t
    return out


def _away(device, stream):
    """None if a call's outputs and launches belong where the caller already is, else the context to make it
    in: another stream than the current one, or another device."""
    if device.type != "cuda":
        raise ValueError("device entry points take CUDA (HIP) tensors")
    if stream is None:
        return None if device.index == torch.cuda.current_device() else torch.cuda.device(device)
    if stream.device != device:
        raise ValueError(f"stream on {stream.device}, tensors on {device}")
    return torch.cuda.stream(stream)


# The current stream's handle; making a torch.cuda.Stream of it would cost 3 us a call.
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _dense(t: torch.Tensor, name: str, columns: int | None = None) -> None:
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} needs a last dimension of at least one element")
    if columns is not None and t.shape[-1] != columns:
        raise ValueError(f"{name} has rows of {t.shape[-1]} elements, expected {columns}")


def _same_device(device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensor on {t.device}, expected {device}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as [rows, columns] with adjacent columns and rows at least a row apart."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.new_empty((0, t.shape[-1]))
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _bias(bias, outer: int, device):
    if bias is None:
        return 0
    if bias.dtype != torch.float32 or tuple(bias.shape) != (outer,) or not bias.is_contiguous():
        raise ValueError(f"bias must be a contiguous float32 [{outer}] tensor")
    _same_device(device, bias)
    return bias.data_ptr()


def _new_blocks(rows: int, columns: int, codes, device) -> BlockTensor:
    out = BlockTensor.__new__(BlockTensor)  # laid out as its constructor would check
    out.codes = torch.empty((rows, _blocks(columns) * BLOCK), dtype=codes, device=device)
    out.exponents = torch.empty((rows, _exponent_pitch(columns)), dtype=torch.uint8, device=device)
    out.columns = columns
    return out


def _workspace(query, args, device):
    size = C.c_size_t()
    check(query(*args, C.byref(size)))
    if not size.value:
        return None, 0, 0
    space = torch.empty(size.value, dtype=torch.uint8, device=device)
    return space, space.data_ptr(), size.value


def quantize_blocks(x: torch.Tensor, codes=E4M3, stream=None) -> BlockTensor:
    """quantizeBlocks: x's rows (all leading dimensions) in blocks along the last one."""
    _dense(x, "x")
    if codes not in _CODES:
        raise ValueError(f"codes must be float8_e4m3fn or int8, got {codes}")
    device = x.device
    away = _away(device, stream)
    if away:
        with away:
            return quantize_blocks(x, codes)
    x = _rows(x)
    out = _new_blocks(x.shape[0], x.shape[1], codes, device)
    check(lib().tcc_quantize_blocks(x.data_ptr(), _stride(x), _TYPES[x.dtype], out.codes.data_ptr(),
                                    out.exponents.data_ptr(), _CODES[codes], x.shape[0], x.shape[1],
                                    _stream(device.index)))
    return out


def dequantize_blocks(x: BlockTensor, dtype=torch.float32, stream=None) -> torch.Tensor:
    """dequantizeBlocks: the values [rows, columns] that the blocks stand for."""
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    device = x.codes.device
    away = _away(device, stream)
    if away:
        with away:
            return dequantize_blocks(x, dtype)
    out = torch.empty((x.rows, x.columns), dtype=dtype, device=device)
    check(lib().tcc_dequantize_blocks(x.codes.data_ptr(), x.exponents.data_ptr(), _CODES[x.codes.dtype],
                                      out.data_ptr(), x.columns, _TYPES[dtype], x.rows, x.columns,
                                      _stream(device.index)))
    return out


def quantize_weight_blocks(w: torch.Tensor, transposed: bool = True, stream=None) -> BlockWeight:
    """quantizeWeightBlocks: w [outer, inner] in tiles; `transposed` adds the copy that the input gradient
    needs, in the same pass."""
    _dense(w, "w")
    if w.dim() != 2 or w.shape[0] < 1:
        raise ValueError("w must be [outer, inner]")
    outer, inner = w.shape
    device = w.device
    away = _away(device, stream)
    if away:
        with away:
            return quantize_weight_blocks(w, transposed)
    w = _rows(w)

    def space(rows, columns):
        return (torch.empty((rows, _blocks(columns) * BLOCK), dtype=E4M3, device=device),
                torch.empty((_blocks(rows), _exponent_pitch(columns)), dtype=torch.uint8, device=device))

    codes, exponents = space(outer, inner)
    codes_t, exponents_t = space(inner, outer) if transposed else (None, None)
    check(lib().tcc_quantize_weight_blocks(
        w.data_ptr(), _stride(w), _TYPES[w.dtype], codes.data_ptr(), exponents.data_ptr(),
        codes_t.data_ptr() if transposed else 0, exponents_t.data_ptr() if transposed else 0, outer, inner,
        _stream(device.index)))
    return _weight(codes, exponents, inner, codes_t, exponents_t)


def matmul_blocks(x: BlockTensor, weight: BlockWeight, bias: torch.Tensor | None = None,
                  dtype=torch.bfloat16, stream=None) -> torch.Tensor:
    """matmulBlocks: x weight^T + bias [rows, outer] for x already in E4M3 blocks. dtype is that of the result; a 16-bit
    one has the 8-bit matrix instruction's sums (the module's docstring), float32 has float32 sums."""
    if x.codes.dtype != E4M3:
        raise ValueError("x must have float8_e4m3fn codes")
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    if x.columns != weight.columns:
        raise ValueError(f"x has rows of {x.columns} elements, expected {weight.columns}")
    device, outer = x.codes.device, weight.rows
    _same_device(device, weight.codes)
    at_bias = _bias(bias, outer, device)
    away = _away(device, stream)
    if away:
        with away:
            return matmul_blocks(x, weight, bias, dtype)
    y = torch.empty((x.rows, outer), dtype=dtype, device=device)
    check(lib().tcc_matmul_blocks(x.codes.data_ptr(), x.exponents.data_ptr(), weight.codes.data_ptr(),
                                  weight.exponents.data_ptr(), at_bias, y.data_ptr(), outer, _TYPES[dtype], x.rows,
                                  x.columns, outer, _stream(device.index)))
    return y


def linear_blocks(x: torch.Tensor, weight: BlockWeight, bias: torch.Tensor | None = None, *,
                  keep: bool = False, stream=None):
    """linearBlocks: y = Q(x) weight^T + bias in x's type, for x [..., inner] quantized into E4M3 blocks on
    the way; sums are those of matmul_blocks with x's type. With keep=True returns (y, x's BlockTensor): what the weight
    gradient needs of x, in 8 bits."""
    inner, outer = weight.columns, weight.rows
    _dense(x, "x", inner)
    device = x.device
    _same_device(device, weight.codes)
    at_bias = _bias(bias, outer, device)
    kind = _TYPES[x.dtype]
    away = _away(device, stream)
    if away:
        with away:
            return linear_blocks(x, weight, bias, keep=keep)
    flat = _rows(x)
    rows = flat.shape[0]
    y = torch.empty((*x.shape[:-1], outer), dtype=x.dtype, device=device)
    kept = _new_blocks(rows, inner, E4M3, device) if keep else None
    _space, at, size = _workspace(lib().tcc_linear_blocks_workspace, (rows, inner, outer, kind, keep), device)
    check(lib().tcc_linear_blocks(flat.data_ptr(), _stride(flat), kind, weight.codes.data_ptr(),
                                  weight.exponents.data_ptr(), at_bias, y.data_ptr(), outer,
                                  kept.codes.data_ptr() if keep else 0,
                                  kept.exponents.data_ptr() if keep else 0, rows, inner, outer, at, size,
                                  _stream(device.index)))
    return (y, kept) if keep else y


def weight_grad_blocks(dy: torch.Tensor, x: BlockTensor | None, bias: bool = True, stream=None):
    """weightGradBlocks: (dw float32 [outer, inner], db float32 [outer] or None) from the output gradient
    [..., outer] and the forward pass's kept blocks; without them (None, db)."""
    _dense(dy, "dy")
    device, outer = dy.device, dy.shape[-1]
    rows = dy.numel() // outer
    if x is None:
        if not bias:
            raise ValueError("neither a weight's nor a bias's gradient is asked for")
    else:
        if x.codes.dtype != E4M3:
            raise ValueError("x must have float8_e4m3fn codes")
        _same_device(device, x.codes)
        if rows != x.rows:
            raise ValueError(f"dy has {rows} rows, the kept blocks {x.rows}")
    away = _away(device, stream)
    if away:
        with away:
            return weight_grad_blocks(dy, x, bias)
    dy = _rows(dy)
    inner = 0 if x is None else x.columns
    dw = None if x is None else torch.empty((outer, inner), dtype=torch.float32, device=device)
    db = torch.empty(outer, dtype=torch.float32, device=device) if bias else None
    sizes = (rows, inner, outer, _TYPES[dy.dtype])
    _space, at, size = _workspace(lib().tcc_weight_grad_blocks_workspace, sizes, device)
    check(lib().tcc_weight_grad_blocks(dy.data_ptr(), _stride(dy), sizes[3], x.codes.data_ptr() if x else 0,
                                       x.exponents.data_ptr() if x else 0, dw.data_ptr() if x else 0,
                                       db.data_ptr() if bias else 0, rows, inner, outer, at, size,
                                       _stream(device.index)))
    return dw, db


def linear_blocks_backward(dy: torch.Tensor, kept: BlockTensor | None, weight: BlockWeight | None, *,
                           need=(True, True, True), stream=None):
    """(dx, dw, db) of linear_blocks, None for what `need` leaves out. dx = Q(dy) weight in dy's type, from the
    weight's transposed copy; dw and db are float32, dw from the kept blocks and dy in full, db from dy."""
    dx = dw = db = None
    if need[0]:
        dx = linear_blocks(dy, weight.transposed(), stream=stream)
    if need[1] or need[2]:
        dw, db = weight_grad_blocks(dy, kept if need[1] else None, bias=bool(need[2]), stream=stream)
    return dx, dw, db


def _activation(kind: str) -> int:
    if kind not in _KINDS:
        raise ValueError(f"kind must be one of {', '.join(_KINDS)}, got {kind!r}")
    return _KINDS[kind]


def activation_blocks(x: torch.Tensor, kind: str = "silu", *, gated: bool = False, codes=INT8, stream=None):
    """activationBlocks: (y, kept) for y = f(x), or gated y = f(g) * u of x = (g | u) along the last axis.
    kept is x in blocks of `codes`, all that the backward pass needs (gated: two rows for each of x's, the
    gate's and the factor's); codes=None keeps nothing."""
    _dense(x, "x")
    function = _activation(kind)
    if codes is not None and codes not in _CODES:
        raise ValueError(f"codes must be float8_e4m3fn, int8 or None, got {codes}")
    if gated and x.shape[-1] % 2:
        raise ValueError("a gated activation needs rows of an even number of elements")
    width = x.shape[-1] // 2 if gated else x.shape[-1]
    device = x.device
    away = _away(device, stream)
    if away:
        with away:
            return activation_blocks(x, kind, gated=gated, codes=codes)
    flat = _rows(x)
    rows = flat.shape[0]
    y = torch.empty((*x.shape[:-1], width), dtype=x.dtype, device=device)
    kept = None if codes is None else _new_blocks(2 * rows if gated else rows, width, codes, device)
    check(lib().tcc_activation_blocks(flat.data_ptr(), _stride(flat), _TYPES[x.dtype], function, gated,
                                      y.data_ptr(), width, kept.codes.data_ptr() if kept else 0,
                                      kept.exponents.data_ptr() if kept else 0,
                                      _CODES[codes] if kept else 0, rows, width, _stream(device.index)))
    return y, kept


def activation_blocks_backward(dy: torch.Tensor, kept: BlockTensor, kind: str = "silu", *, gated: bool = False,
                               stream=None) -> torch.Tensor:
    """activationBlocksBackward: dx in dy's type and x's shape, from the kept blocks."""
    width = kept.columns
    _dense(dy, "dy", width)
    function = _activation(kind)
    device = dy.device
    _same_device(device, kept.codes)
    if dy.numel() // width * (2 if gated else 1) != kept.rows:
        raise ValueError(f"dy has {dy.numel() // width} rows, the kept blocks {kept.rows}")
    wide = 2 * width if gated else width
    away = _away(device, stream)
    if away:
        with away:
            return activation_blocks_backward(dy, kept, kind, gated=gated)
    flat = _rows(dy)
    dx = torch.empty((*dy.shape[:-1], wide), dtype=dy.dtype, device=device)
    check(lib().tcc_activation_blocks_backward(flat.data_ptr(), _stride(flat), _TYPES[dy.dtype],
                                               kept.codes.data_ptr(), kept.exponents.data_ptr(),
                                               _CODES[kept.codes.dtype], function, gated, dx.data_ptr(), wide,
                                               flat.shape[0], width, _stream(device.index)))
    return dx


# --------------------------------------------------------------------------------------------------
# Under autograd


def _float_bias(bias):
    """A bias of any type and layout as the products take it."""
    return None if bias is None else bias.float().contiguous()


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias):
        grad_x, grad_w, _ = ctx.needs_input_grad
        weight = quantize_weight_blocks(w, transposed=grad_x)
        out = linear_blocks(x, weight, _float_bias(bias), keep=grad_w)
        y, kept = out if grad_w else (out, None)
        # x itself is not saved: the weight gradient reads its blocks, a byte an element, and nothing else does.
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
            dx = linear_blocks(dy, BlockWeight(codes_t, exponents_t, outer))
        if codes is not None or ctx.needs_input_grad[2]:
            kept = None if codes is None else BlockTensor(codes, exponents, inner)
            dw, db = weight_grad_blocks(dy, kept, bias=ctx.needs_input_grad[2])
            dw = None if dw is None else dw.to(ctx.types[0])
            db = None if db is None else db.to(ctx.types[1])
        return dx, dw, db


class _Activation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind, gated, codes):
        y, kept = activation_blocks(x, kind, gated=gated, codes=codes if ctx.needs_input_grad[0] else None)
        if kept is not None:
            ctx.save_for_backward(kept.codes, kept.exponents)
            ctx.call = (kept.columns, kind, gated)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        width, kind, gated = ctx.call
        kept = BlockTensor(*ctx.saved_tensors, width)
        return activation_blocks_backward(dy, kept, kind, gated=gated), None, None, None


def block_linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """x w^T + bias with both operands in E4M3 blocks, differentiable; w is the master weight, quantized
    in every call. Under autocast x is cast to its type first, as torch's linear casts it; w is quantized and the bias
    added at their own precision."""
    if x.is_cuda and x.dtype in _TYPES and torch.is_autocast_enabled("cuda"):
        x = x.to(torch.get_autocast_dtype("cuda"))
    if not torch.is_grad_enabled():
        # Inside a Function the mode is off and its arguments still say that they require a gradient.
        weight = quantize_weight_blocks(w, transposed=False)
        return linear_blocks(x, weight, _float_bias(bias))
    return _Linear.apply(x, w, bias)


def block_activation(x: torch.Tensor, kind: str = "silu", *, gated: bool = False, codes=INT8) -> torch.Tensor:
    """activation_blocks, differentiable: what autograd keeps of x is its blocks, so codes=None is for inputs that
    need no gradient."""
    if not torch.is_grad_enabled():
        return activation_blocks(x, kind, gated=gated, codes=None)[0]
    if codes is None and x.requires_grad:
        raise ValueError("x requires a gradient, which codes=None keeps nothing for")
    return _Activation.apply(x, kind, gated, codes)


class BlockLinear(torch.nn.Linear):
    """torch.nn.Linear whose product and gradients run on 8-bit blocks, autocast included (block_linear)."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return block_linear(x, self.weight, self.bias)

    def serving(self):
        """(BlockWeight, float32 bias or None) for linear_blocks, quantized once."""
        bias = None if self.bias is None else self.bias.detach()
        return quantize_weight_blocks(self.weight.detach(), transposed=False), _float_bias(bias)
