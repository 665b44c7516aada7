"""Scaled rotary positions in 64 bits (numpy), with the error that f32 results may have."""
import numpy as np


def frequencies(n, base, scale, ext, orig, ff=None, beta_fast=32.0, beta_slow=1.0, attn=1.0):
    """f64 [n / 2] the angle of one position, and what values are multiplied by."""
    base, scale, ext, attn = (float(np.float32(v)) for v in (base, scale, ext, attn))
    i = np.arange(n // 2, dtype=np.float64)
    f = base ** (-2.0 * i / n)
    if ff is not None:
        f = f / np.asarray(ff, np.float64)
    if ext == 0.0:
        return f * scale, attn
    at = [n * np.log(orig / (2.0 * np.pi * np.float64(np.float32(b)))) / (2.0 * np.log(base)) for b in (beta_fast, beta_slow)]
    lo, hi = max(0.0, np.floor(at[0])), min(n - 1.0, np.ceil(at[1]))
    w = ext * (1.0 - np.clip((i - lo) / max(0.001, hi - lo), 0.0, 1.0))
    return f * (scale * (1.0 - w) + w), attn * (1.0 + 0.1 * np.log(1.0 / scale))


def rope(x, pos, n, halves, f, m):
    """x f32 [T, heads, hd], pos int [T] -> f64 result, and how far an f32 result may be from it: cosine and sine are off by
    their rounding (2^-24) and the angle's error (2^-50 of it, f64 products and the table's exponential, and 1.2e-10 of the
    sums), of the two products one is rounded, and the result is (2^-24 each)."""
    x64 = np.asarray(x, np.float64)
    a = np.asarray(pos, np.float64)[:, None] * f
    c, s = m * np.cos(a)[:, None], m * np.sin(a)[:, None]
    u = slice(0, n // 2) if halves else slice(0, n, 2)
    w = slice(n // 2, n) if halves else slice(1, n, 2)
    y, tol = x64.copy(), np.zeros_like(x64)
    p, q = x64[..., u], x64[..., w]
    y[..., u], y[..., w] = p * c - q * s, p * s + q * c
    off = abs(m) * (np.abs(a)[:, None] * 2.0 ** -50 + 1.5e-10) * (np.abs(p) + np.abs(q))
    one, two = np.abs(p * c) + np.abs(q * s), np.abs(p * s) + np.abs(q * c)
    tol[..., u], tol[..., w] = 3 * 2.0 ** -24 * one + off, 3 * 2.0 ** -24 * two + off
    return y, tol
