"""64-bit restatement of the 8-bit operators (csrc/sgemm_i8_*.cuh): what the device has to return, from the definitions.

Matrices are NumPy arrays with a row per token or channel (``[rows, features]``).  Values of q are exact statements (round to
nearest, halves to even, of an exact quotient); scales, products and gradients are 64-bit numbers that the device's are
compared with under derived bounds."""
from __future__ import annotations

import numpy as np

LARGEST = 127.0 * 2.0 ** 121     # rows with larger magnitudes (or NaN, infinity) get scale NaN and q = 0


def round_bf16(x):
    """Nearest bfloat16 (ties to even) of 64-bit values, as 64-bit values.  (Through FP32: exact there for every value the
    tests round — at most 24 significant bits — or a double rounding far below what the comparisons resolve.)"""
    f = np.asarray(x, dtype=np.float32)
    u = f.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(f), np.nan, r).astype(np.float64)


def round_to(x, kind):
    if kind == "bf16":
        return round_bf16(x)
    with np.errstate(over="ignore"):
        return np.asarray(x).astype({"fp32": np.float32, "fp16": np.float16}[kind]).astype(np.float64)


def _exact_quotient(p, peak):
    """round(127 p / peak) for FP32 values: 127 p and (n + 1/2) peak are exact in 64 bits, so the comparison is too."""
    with np.errstate(invalid="ignore", divide="ignore"):
        n = np.floor(np.where(peak > 0, np.abs(127.0 * p) / peak, 0.0))
    n = np.where(np.isfinite(n), n, 0.0)
    a, half = np.abs(127.0 * p), (n + 0.5) * peak
    up = np.where(a > half, 1.0, np.where(a < half, 0.0, n % 2))
    return np.sign(p) * (n + up)


def quantize(x, pow2=False):
    """(q as int8, scale as float64) of FP32-representable rows."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(invalid="ignore"):
        peak = np.max(np.abs(x), axis=1, keepdims=True) if x.shape[1] else np.zeros((x.shape[0], 1))
    bad = ~(peak <= LARGEST)
    safe = np.where(bad, 0.0, peak)
    xs = np.where(bad, 0.0, x)
    if pow2:
        mantissa, exponent = np.frexp(safe)              # safe = mantissa * 2^exponent, mantissa in [1/2, 1)
        e = np.maximum(exponent - 7 + (mantissa > 127.0 / 128.0), -126)
        scale = np.where(safe > 0, np.ldexp(1.0, e), 0.0)
        q = np.rint(np.where(safe > 0, xs / np.where(safe > 0, scale, 1.0), 0.0))
    else:
        scale, q = safe / 127.0, _exact_quotient(xs, safe)
    return q.astype(np.int8), np.where(bad, np.nan, scale)[:, 0]


def rmsnorm(x, gamma, eps, residual=None):
    """(q, scale, h) with h = x + residual and p = h * gamma rounded to FP32, as the operator defines them."""
    f32 = np.float32
    with np.errstate(over="ignore", invalid="ignore"):
        h = np.asarray(x, dtype=f32) if residual is None else np.asarray(x, dtype=f32) + np.asarray(residual, dtype=f32)
        p = (h * np.asarray(gamma, dtype=f32)[None, :]).astype(np.float64)
    q, base = quantize(p)
    wide = h.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        rstd = 1.0 / np.sqrt(np.mean(wide * wide, axis=1) + eps)
        return q, np.where(base == 0, 0.0, base * rstd), wide


def restore(q, scale, kind):
    with np.errstate(invalid="ignore", over="ignore"):
        return round_to(q.astype(np.float32) * np.asarray(scale, dtype=np.float32)[:, None], kind)


def linear(qx, sx, qw, sw, bias=None):
    """Y before its rounding: [tokens, channels] in 64 bits."""
    acc = qx.astype(np.int64) @ qw.astype(np.int64).T if qx.shape[1] < 64 else (qx.astype(np.float64) @ qw.astype(np.float64).T)
    y = acc.astype(np.float64) * np.asarray(sx, dtype=np.float64)[:, None] * np.asarray(sw, dtype=np.float64)[None, :]
    return y if bias is None else y + np.asarray(bias, dtype=np.float64)[None, :]


def wgrad(q, scale, dy, kind, alpha=1.0, c=None, beta=0.0):
    """(dW before its rounding, the sum of magnitudes a bound is taken from): [channels, features] in 64 bits; `dy` holds values of
    the 16-bit type `kind`, the checkpoint's values are rounded to it."""
    values = restore(q, scale, kind)
    dw = alpha * (dy.astype(np.float64).T @ values)
    size = abs(alpha) * (np.abs(dy).astype(np.float64).T @ np.abs(values))
    if beta:
        dw, size = dw + beta * c.astype(np.float64), size + abs(beta) * np.abs(c).astype(np.float64)
    return dw, size
