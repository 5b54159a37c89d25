"""The microscaled 4-bit format, and the way of tokens to experts and back, in 64 bits on the CPU, written from their
definitions.

A block of 32 has the smallest power of two, at least 2^-126, that brings its largest magnitude to at most 6; a block of zeros
has scale 1, one that holds an infinity or a NaN is NaN. Codes are 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives.
"""
import numpy as np

from blocks_oracle import scale

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def exponent(peak: np.ndarray) -> np.ndarray:
    """Exponent bytes of blocks with these largest magnitudes."""
    fine = np.isfinite(peak) & (peak > 0)
    f, p = np.frexp(np.where(fine, peak, 1.0))
    e = np.maximum(p - 3 + (f > 0.75) + 127, 1)
    return np.where(fine, e, np.where(peak == 0, 127, 255)).astype(np.uint8)


def to_codes(v: np.ndarray) -> np.ndarray:
    """Codes of |v| <= 6: the nearest value, of two as near the one with an even code."""
    off = np.abs(np.abs(v)[..., None] - VALUES)
    best = off.min(-1, keepdims=True)
    tied = off == best
    first = tied.argmax(-1)
    code = np.where((tied.sum(-1) > 1) & (first % 2 == 1), first + 1, first)
    return (code + 8 * np.signbit(v)).astype(np.uint8)


def of_codes(q: np.ndarray) -> np.ndarray:
    return np.where(q >= 8, -1.0, 1.0) * VALUES[q % 8]


def _peaks(x):
    with np.errstate(invalid="ignore"):
        return np.where(np.isfinite(x), np.abs(x), np.inf)


def _encode(v, e):
    """Codes of v, whose elements have the exponents e."""
    nan = e == 255
    s = np.where(nan, 1.0, scale(np.where(nan, 127, e)))
    c = np.where(nan, 0.0, np.where(nan, 0.0, v) / s)
    # what would round to 2^128 takes the code below: values are finite in FP32
    c = np.where(e == 253, np.clip(c, -3.0, 3.0), c)
    return to_codes(c)


def quantize(x: np.ndarray):
    """(codes [rows, 128 * steps], exponents [rows, blocks], values [rows, columns])"""
    rows, columns = x.shape
    blocks = -(-columns // 32)
    v = np.zeros((rows, blocks, 32))
    v.reshape(rows, -1)[:, :columns] = x
    e = exponent(_peaks(v).max(2)) if rows else np.zeros((0, blocks), np.uint8)
    q = _encode(v, np.broadcast_to(e[:, :, None], v.shape))
    return _whole(q, e, columns)


def quantize_tiles(w: np.ndarray):
    """The same of a weight in tiles of 32 x 32."""
    rows, columns = w.shape
    up, across = -(-rows // 32), -(-columns // 32)
    v = np.zeros((up, 32, across, 32))
    v.reshape(up * 32, across * 32)[:rows, :columns] = w
    e = exponent(_peaks(v).max((1, 3)))
    q = _encode(v, np.broadcast_to(e[:, None, :, None], v.shape)).reshape(up * 32, across, 32)[:rows]
    return _whole(q, np.repeat(e, 32, 0)[:rows], columns)


def _whole(q, e, columns):
    rows = q.shape[0]
    values = (of_codes(q) * scale(e)[:, :, None]).reshape(rows, -1)[:, :columns]
    codes = np.zeros((rows, -(-columns // 128) * 128), np.uint8)
    codes[:, :q.shape[1] * 32] = q.reshape(rows, -1)
    return codes, e, values


def pack(codes: np.ndarray) -> np.ndarray:
    """Two codes a byte, the first in the low half."""
    return codes[:, 0::2] | codes[:, 1::2] << 4


def place(e: np.ndarray, fill: int = 127) -> np.ndarray:
    """Exponents [rows, blocks] as they are kept."""
    rows, blocks = e.shape
    out = np.full((rows, -(-blocks // 16) * 16), fill, np.uint8)
    for b in range(blocks):
        out[:, 16 * (b // 16) + 4 * (b % 4) + b // 4 % 4] = e[:, b]
    return out


def plan(ids: np.ndarray, experts: int):
    """(offsets, order, places) of choices [tokens, each]."""
    flat = ids.reshape(-1)
    flat = np.where((flat >= 0) & (flat < experts), flat, experts)
    order = np.argsort(flat, kind="stable")
    places = np.empty_like(order)
    places[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=experts + 1)[:experts])])
    return offsets, order, places
