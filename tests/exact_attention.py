"""Attention over chosen keys in 64 bits, with a bound on what the kernels' roundings can make of it, row by row.

The bound counts roundings of at most half a step (fp16 2^-11 of the value, fp32 2^-24):
  a score      D products of halves summed in fp32: (D + 4) 2^-24 |q| |k|, and over quantised rows an operand level * scale + bias
               rounded to fp16: 2^-11 |k| per element; the score's own value takes 2^-22 of it into the exponent's argument;
  a weight     e^ds - 1 <= 2 ds for that (numerator and denominator: twice), and 2^-20 for exp2 and the sums;
  P            rounded to fp16 in front of the values: 2^-11 of a weight, below 2^-14 of the row's reference 2^-25 absolutely (the
               reference lies at most 2^8 below the row's largest score); over quantised rows the product with a group's scale
               is rounded once more, levels are at most 2^bits - 1, and the bias has its own sum;
  the output   2^-11 of it.
"""
import numpy as np

HALF16, HALF32 = 2.0 ** -11, 2.0 ** -24


def dequantise(rows, width, bits):
    """Stored rows (uint8 [n][stride]) -> (level * scale, bias), float64 [n][width]; fp16 rows have no bias."""
    n = rows.shape[0]
    if bits == 16:
        return rows.view(np.float16).astype(np.float64), np.zeros((n, width))
    cut, groups = width * bits // 8, width // 64
    levels = rows[:, :cut]
    if bits == 4:
        levels = np.stack([levels & 15, levels >> 4], -1).reshape(n, width)
    params = np.ascontiguousarray(rows[:, cut:cut + 4 * groups]).view(np.float16).astype(np.float64)
    scale, bias = np.repeat(params[:, :groups], 64, 1), np.repeat(params[:, groups:], 64, 1)
    return levels.astype(np.float64) * scale, bias


def stored_rows(values, bits):
    """fp16 values [n][width] as rows of the cache's stored format (any levels would do; these are near the values)."""
    values = np.ascontiguousarray(values, np.float16)
    n, width = values.shape
    if bits == 16:
        return values.view(np.uint8).reshape(n, width * 2).copy()
    x = values.astype(np.float32).reshape(n, width // 64, 64)
    bias = x.min(-1).astype(np.float16)
    scale = ((x.max(-1) - bias.astype(np.float32)) / (2 ** bits - 1)).astype(np.float16)
    safe = np.maximum(scale.astype(np.float32), 1e-7)[..., None]
    levels = np.clip(np.rint((x - bias.astype(np.float32)[..., None]) / safe), 0, 2 ** bits - 1).astype(np.uint8).reshape(n, width)
    if bits == 4:
        levels = levels[:, 0::2] | (levels[:, 1::2] << 4)
    return np.concatenate([levels, *(p.view(np.uint8).reshape(n, width // 32) for p in (scale, bias))], 1)


def attend(q, k, v, seen, scale, gate=None, bits=16):
    """q [heads][dim]; k, v pairs from ``dequantise`` over the same positions [n][kv_heads * dim]; seen: bool [n].
    Returns (out, bound), float64 [heads][dim]; zeros for a row that sees nothing."""
    heads, dim = q.shape
    kv_heads = k[0].shape[1] // dim
    group = heads // kv_heads
    at = np.flatnonzero(seen)
    out, bound = np.zeros((heads, dim)), np.zeros((heads, dim))
    if len(at) == 0:
        return out, bound
    q = q.astype(np.float64)
    for h in range(heads):
        if h % group == 0:
            cols = slice(h // group * dim, (h // group + 1) * dim)
            v_level, v_bias = v[0][at, cols], v[1][at, cols]
            kk, vv = k[0][at, cols] + k[1][at, cols], v_level + v_bias
            abs_k, abs_v, abs_level, abs_bias, top_v, top_bias = (np.abs(kk), np.abs(vv), np.abs(v_level), np.abs(v_bias), np.abs(vv).max(0),
                                                                 np.abs(v_bias).max(0))
        s = kk @ q[h] * scale
        mags = abs_k @ np.abs(q[h]) * abs(scale)
        ds = mags * ((dim + 4) * HALF32 + (0.0 if bits == 16 else HALF16)) + np.abs(s) * 2.0 ** -22
        w = np.exp(s - s.max())
        total = w.sum()
        w = w / total
        out[h] = w @ vv
        eps = 2.0 * 2.0 * ds.max() + 2.0 ** -20
        tiny = (w * total < 2.0 ** -13 * (1.0 if bits == 16 else 2.0 ** 8)).sum() / total
        if bits == 16:
            err = (w @ abs_v) * (eps + 2 * HALF16) + tiny * 2.0 ** -25 * top_v
        else:
            err = (w @ abs_v) * eps + (w @ abs_level) * 3 * HALF16 + (w @ abs_bias) * 2 * HALF16
            err += tiny * 2.0 ** -25 * ((2 ** bits - 1) / 4.0 + top_bias)
        bound[h] = err
    if gate is not None:
        g = 1.0 / (1.0 + np.exp(-gate.astype(np.float64)))
        out, bound = out * g, bound * g + np.abs(out * g) * 2.0 ** -20
    return out, bound + np.abs(out) * HALF16 + 2.0 ** -25


def check(got, pairs, what=""):
    """got [rows][heads][dim] against the (out, bound) of every row."""
    for r, (out, bound) in enumerate(pairs):
        g = got[r].astype(np.float64)
        assert np.isfinite(g).all(), f"{what} row {r}: not finite"
        over = np.abs(g - out) - bound
        assert over.max() <= 0, f"{what} row {r}: off by {np.abs(g - out).flat[over.argmax()]:.3e}, bound {bound.flat[over.argmax()]:.3e}"
