"""Plain 64-bit models of the 4-bit operators, in numpy, for the tests."""
import numpy as np


def quantise(x):
    """float64 [..., D] of fp16 values -> codes, s, m (float64) of every 32 channels: m the minimum, s the largest fp16 not
    above (max - min) / 15, code the nearest of 0..15; a group that holds a value that is not finite: s = m = NaN."""
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    ok = np.isfinite(g).all(-1, keepdims=True)
    g = np.where(ok, g, 0.0)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    s = ((hi - lo) / 15).astype(np.float16)
    s = np.where(s.astype(np.float64) > (hi - lo) / 15, np.nextafter(s, np.float16(0)), s).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s > 0, np.clip(np.rint((g - lo) / s), 0, 15), 0.0)
    return c, np.where(ok, s, np.nan), np.where(ok, lo, np.nan)


def entry(x):
    """What the cache holds for x, unrounded."""
    c, s, m = quantise(x)
    return (m + c * s).reshape(x.shape)


def rotate(x, pos, cos, sin, interleaved):
    """x float64 [tokens, heads, D] of fp16 values, turned and rounded once to fp16."""
    rot = 2 * cos.shape[1]
    y = x.copy()
    c, s = cos[pos].astype(np.float64)[:, None], sin[pos].astype(np.float64)[:, None]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y.astype(np.float16).astype(np.float64)


def scaled_codes(x):
    """s c of what the cache holds for x: the part above the group's minimum."""
    c, s, m = quantise(x)
    return (c * s).reshape(x.shape)


def attention(q, k, v, sc, scale):
    """q [T, Hq, D], k, v, sc [L, Hkv, D] float64 (sc = scaled_codes of the values, v = m + sc), row t sees keys 0 .. L - T + t.
    Returns the output and the error that a kernel with fp16 weights and fp32 sums may make.

    The kernel sums p~ m + (p~ s)~ c, where ~ rounds to fp16, off by a factor 1 + d with |d| <= 2^-11:
        p~ m + (p~ s)~ c = p (1 + d1) (m + (1 + d2) s c) = p v + d1 p v + (1 + d1) d2 p s c
    so the weights cost 2^-11 sum p |v| and their products with the scales 2^-11 sum p s c (a little more, for d1 d2); the sum of
    the weights is that of the unrounded ones, which costs another 2^-11 of sum p |v| at most; the output is rounded once, 2^-11
    |out|.  A score is an fp32 sum of at most D/8 + 16 terms of magnitude sum |q| |k| scale (its part for the minima is taken
    with group sums of q rounded to 22 bits, 2^-22 of sum |q| |k|, within four of the 2^-24 terms), so exp(score) is off by a
    factor of at most 2^-24 (D/8 + 20) of that, twice (numerator, denominator); weights and their products below the fp16
    range lose at most 2^-32 of the largest weight, or 2^-25 c in absolute terms after the factor 2^7 they carry, each.

    The kernel for many rows sums p~ v with keys and values rounded to fp16: handed those (k and v as kv_read returns them, sc zero)
    the same bound holds for it without its second term."""
    T, Hq, D = q.shape
    L, Hkv = k.shape[:2]
    out, tol = np.zeros_like(q), np.zeros_like(q)
    seen = np.arange(L)[None] <= np.arange(L - T, L)[:, None]          # [T, L]
    some = seen.any(1)
    for h in range(Hq):
        kk, vv, ss = (x[:, h // (Hq // Hkv)] for x in (k, v, sc))
        with np.errstate(invalid="ignore"):
            z = np.where(seen, (q[:, h] @ kk.T) * scale, -np.inf)
            mag = np.where(seen, (np.abs(q[:, h]) @ np.abs(kk).T) * abs(scale), 0).max(1, initial=0)[:, None]
            w = np.where(some[:, None], np.exp(z - z.max(1, initial=-np.inf, keepdims=True)), 0)
            total = np.where(some, w.sum(1), 1)[:, None]
        p = w / total
        o, a = p @ vv, p @ np.abs(vv)
        biggest = np.where(seen[:, :, None], np.abs(vv)[None], 0).max((1, 2), initial=0)[:, None] if L * T * D < 1 << 24 else np.abs(vv).max()
        out[:, h] = o
        tol[:, h] = 2 * 2.0 ** -11 * a + 1.001 * 2.0 ** -11 * (p @ ss) + 2.0 ** -11 * np.abs(o) \
            + 2 * 2.0 ** -24 * (D / 8 + 20) * mag * a + seen.sum(1)[:, None] / total * (2.0 ** -32 * biggest + 15 * 2.0 ** -32) + 2.0 ** -24
    return out, tol


def linear(codes, scales, zeros, x, bias, residual, relu, fp16_weights):
    """float64 y [N, M] and the error that fp32 sums (and, for fp16_weights, weights rounded to fp16) may make.

    Error: one rounding of the result to fp16, half a step; K / 16 + 64 fp32 additions (a matrix instruction adds 16 products
    at a time; then the groups, the warps and the thread blocks are added) of terms up to sum s (c + z) |x|; a weight
    rounded to fp16 is off by 2^-11 of itself."""
    M, K = codes.shape
    G = K // scales.shape[1]
    s, z = np.repeat(scales, G, 1), np.repeat(zeros, G, 1)
    w = s * (codes - z)
    y = x @ w.T
    terms = np.abs(x) @ (np.abs(s) * (codes + z)).T
    tol = (K / 16 + 64) * 2.0 ** -24 * terms + (2.0 ** -11 * (np.abs(x) @ np.abs(w).T) if fp16_weights else 0.0)
    if bias is not None:
        y = y + bias
    if relu:
        y = np.maximum(y, 0)
    if residual is not None:
        y = y + residual
    return y, tol + 2.0 ** -11 * np.abs(y) + 2.0 ** -24
