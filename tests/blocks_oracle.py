"""The 8-bit block format and the layers on it, in 64 bits on the CPU, written from their definitions.

A block's scale is the smallest power of two, at least 2^-126, that brings its largest magnitude to at most
448 (E4M3) or 127 (INT8); a block of zeros has scale 1, one that holds an infinity or a NaN is NaN.
"""
import numpy as np
import torch

TOP = {"e4m3": 448.0, "int8": 127.0}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# Half a unit in the last place, relative to the value.
ROUNDING = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def f64(t) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def exponent(peak: np.ndarray, codes: str) -> np.ndarray:
    """Exponent bytes of blocks with these largest magnitudes."""
    fine = np.isfinite(peak) & (peak > 0)
    safe = np.where(fine, peak, 1.0)
    f, p = np.frexp(safe)
    f0, p0 = np.frexp(TOP[codes])
    e = np.maximum(p - p0 + (f > f0) + 127, 1)
    return np.where(fine, e, np.where(peak == 0, 127, 255)).astype(np.uint8)


def scale(e: np.ndarray) -> np.ndarray:
    return np.where(e == 255, np.nan, np.ldexp(1.0, e.astype(int) - 127))


def to_grid(v: np.ndarray, codes: str) -> np.ndarray:
    """v rounded half to even to the values of the codes."""
    if codes == "int8":
        return np.rint(v)
    unit = np.ldexp(1.0, np.maximum(np.frexp(v)[1] - 1, -6) - 3)
    return np.rint(v / unit) * unit


def _peaks(x):
    with np.errstate(invalid="ignore"):
        return np.where(np.isfinite(x), np.abs(x), np.inf)


def quantize(x: np.ndarray, codes: str = "e4m3"):
    """(code values [rows, 128 * blocks], exponents [rows, blocks], values [rows, columns])"""
    rows, columns = x.shape
    blocks = -(-columns // 128)
    v = np.zeros((rows, blocks, 128))
    v.reshape(rows, -1)[:, :columns] = x
    e = exponent(_peaks(v).max(2), codes) if rows else np.zeros((0, blocks), np.uint8)
    q = np.where(e[:, :, None] == 255, 0.0, to_grid(np.where(e[:, :, None] == 255, 0.0, v) / np.where(
        e == 255, 1.0, scale(e))[:, :, None], codes))
    # what would round to 2^128 takes the code below: values are finite in FP32
    below = 240.0 if codes == "e4m3" else 63.0
    with np.errstate(invalid="ignore"):
        q = np.where(np.abs(q * scale(e)[:, :, None]) >= 2.0 ** 128, np.copysign(below, q), q)
    return q.reshape(rows, -1), e, (q * scale(e)[:, :, None]).reshape(rows, -1)[:, :columns]


def quantize_tiles(w: np.ndarray):
    rows, columns = w.shape
    up, across = -(-rows // 128), -(-columns // 128)
    v = np.zeros((up, 128, across, 128))
    v.reshape(up * 128, across * 128)[:rows, :columns] = w
    e = exponent(_peaks(v).max((1, 3)), "e4m3")
    nan = e[:, None, :, None] == 255
    q = np.where(nan, 0.0, to_grid(np.where(nan, 0.0, v) / np.where(e == 255, 1.0, scale(e))[:, None, :, None], "e4m3"))
    values = (q * scale(e)[:, None, :, None]).reshape(up * 128, across * 128)[:rows, :columns]
    return q.reshape(up * 128, across * 128)[:rows], e, values


def activation(kind: str, x: np.ndarray):
    """f(x), f'(x), and the magnitude of the terms in f' whose rounding errors its own has to allow for."""
    from scipy.special import erfc, expit
    if kind == "gelu":
        p = 0.5 * erfc(-x / np.sqrt(2.0))
        d = x * np.exp(-0.5 * x * x) / np.sqrt(2.0 * np.pi)
        return x * p, p + d, 1.0 + np.abs(d)
    a, b = (1.0, 0.0) if kind == "silu" else (np.sqrt(8.0 / np.pi), 0.044715)
    s = expit(a * (x + b * x ** 3))
    inner = a * (1.0 + 3.0 * b * x * x)
    return x * s, s + x * s * expit(-a * (x + b * x ** 3)) * inner, s + np.abs(x * s * inner)


def argument(kind: str, x: np.ndarray) -> np.ndarray:
    """The magnitude that the activation's exponential is taken of: its relative error grows with it."""
    if kind == "gelu_tanh":
        return np.abs(1.6 * (x + 0.044715 * x ** 3))
    return 0.5 * x * x if kind == "gelu" else np.abs(x)
