"""Differential attention in 64 bits, with a bound on what the kernels' roundings can make of it, element by element.

Keys of 8 and 4 bits are level * scale + bias rounded to fp16, which is what such a cache hands out (tt_hip_kv_read).  A map's roundings
are those that tests/exact_attention.py tells one by one: a weight is off by eta of itself at most, 4 ds + 2^-20 for scores of dim / 2
products and 2 * 2^-11 for P (numerator and denominator).  What eta makes of the sum over the values, e1 and e2:
  fp16 rows       the values' signs are independent of queries, keys and all weights' roundings, so that sum_j w_j eta_j v_j stays below
                  7.5 sqrt(sum_j (w_j eta_j v_j)^2) but for a chance of 2 exp(-7.5^2 / 2) = 1e-12 an element (Hoeffding); what is common
                  to all weights takes eta of the sum itself
  8 and 4 bits    levels have one sign: sum_j w_j eta_j |v_j|, and three roundings of level and bias parts
Then, with r = sqrt(mean(a^2) + eps):
  the difference   a1 - lambda a2:  d = e1 + |lambda| e2 + 2^-22 (|a1| + |lambda a2|)
  the norm         |a'/r' - a/r| <= (|a' - a| + |a| |r' - r| / r) / r', |r' - r| <= sqrt(mean(d^2)) (a norm's triangle inequality)
  the output       2^-20 of it for the fp32 arithmetic behind the norm, and one rounding to fp16: 2^-11 of it, 2^-25 where it is subnormal
"""
import numpy as np

from tests.exact_attention import HALF16, HALF32, dequantise


CHANCE = 7.5


def one_map(q, k, v_level, v_bias, seen, scale, bits):
    """q [rows, dim / 2], k [n, dim / 2], values [n, dim], seen [rows, n], all float64 tensors: (out, bound) [rows, dim]."""
    import torch
    dim = v_level.shape[1]
    v = v_level + v_bias
    s = (q @ k.T.contiguous()) * scale
    mags = (q.abs() @ k.abs().T.contiguous()) * abs(scale)
    ds = mags * ((dim + 4) * HALF32) + s.abs() * 2.0 ** -22
    ds = torch.where(seen, ds, torch.zeros_like(ds))
    some = seen.any(-1, keepdim=True)
    s = torch.where(seen, s, torch.full_like(s, -np.inf))
    top = torch.where(some, s.amax(-1, keepdim=True), torch.zeros_like(s[:, :1]))
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True).clamp_min(1e-300)
    w = e / total
    eps = 4.0 * ds.amax(-1, keepdim=True) + 2.0 ** -20
    tiny = (seen & (e < 2.0 ** -13 * (1.0 if bits == 16 else 2.0 ** 8))).sum(-1, keepdim=True) / total
    if bits == 16:
        bound = (CHANCE * ((w * w) @ (v * v)).sqrt() + (w @ v).abs()) * (eps + 2 * HALF16) + tiny * 2.0 ** -25 * v.abs().amax(0)
    else:
        bound = (w @ v.abs()) * eps + (w @ v_level.abs() + w @ v_bias.abs()) * 3 * HALF16
        bound = bound + tiny * 2.0 ** -25 * ((2 ** bits - 1) / 4.0 + v_bias.abs().amax(0) + v.abs().amax(0))
    return w @ v, torch.where(some, bound, torch.zeros_like(bound))


def attend_maps(q, k_rows, v_rows, kv_heads, positions, key_positions, window, scale, lambdas, bits=16, norm=None, eps=1e-5, out_scale=1.0,
                gate=None):
    """q, gate [rows, heads, dim] fp16 tensors, k_rows, v_rows stored rows (uint8 numpy [n][stride]) of key_positions [n], positions [rows],
    lambdas [heads] or [rows, heads].  Returns (out, bound), float64 [rows, heads, dim]."""
    import torch
    rows, heads, dim = q.shape
    dev, group, half = q.device, heads // kv_heads, dim // 2
    k = [torch.from_numpy(x).to(dev) for x in dequantise(k_rows, kv_heads * dim, bits)]
    v = [torch.from_numpy(x).to(dev) for x in dequantise(v_rows, kv_heads * dim, bits)]
    at, key = torch.as_tensor(positions, device=dev)[:, None], torch.as_tensor(key_positions, device=dev)[None]
    seen = key <= at
    if window:
        seen = seen & (key > at - window)
    lambdas = torch.as_tensor(lambdas, device=dev).double().expand(rows, heads)
    out, bound = (torch.zeros(rows, heads, dim, dtype=torch.float64, device=dev) for _ in range(2))
    for h in range(heads):
        cols = slice(h // group * dim, (h // group + 1) * dim)
        kk, level, bias = (k[0] + k[1])[:, cols].half().double(), v[0][:, cols], v[1][:, cols]
        row = q[:, h].double()
        a1, e1 = one_map(row[:, :half], kk[:, :half].contiguous(), level, bias, seen, scale, bits)
        a2, e2 = one_map(row[:, half:], kk[:, half:].contiguous(), level, bias, seen, scale, bits)
        lam = lambdas[:, h, None]
        out[:, h] = a1 - lam * a2
        bound[:, h] = e1 + lam.abs() * e2 + 2.0 ** -22 * (a1.abs() + (lam * a2).abs())
    if norm is not None:
        weight = norm.double() * out_scale
        r = (out.square().mean(-1, keepdim=True) + eps).sqrt()
        dr = bound.square().mean(-1, keepdim=True).sqrt()
        zero = out.abs().amax(-1, keepdim=True) == 0
        r = torch.where(zero, torch.ones_like(r), r)
        drowned = ~zero & (dr > 0.75 * r)  # (a difference that its bound nearly covers says nothing behind the norm)
        assert drowned.double().mean() <= 0.1, "most rows' differences have to stand out of their bounds"
        bound = torch.where(drowned, torch.full_like(bound, np.inf), weight.abs() * (bound + out.abs() * dr / r) / (r - dr).clamp_min(1e-300))
        out = out / r * weight
    else:
        out, bound = out * out_scale, bound * abs(out_scale)
    if gate is not None:
        g = torch.sigmoid(gate.double())
        out, bound = out * g, bound * g
    return out, bound + out.abs() * (2.0 ** -20 + HALF16) + 2.0 ** -25


def check(got, want, what=""):
    """got [rows, heads, dim] fp16 tensor against (out, bound)."""
    import torch
    out, bound = want
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got.double() - out).abs() - bound
    at = int(over.argmax())
    row = at // (got.shape[1] * got.shape[2])
    assert over.flatten()[at] <= 0, (f"{what}: row {row} head {at // got.shape[2] % got.shape[1]} dim {at % got.shape[2]} is {float(got.flatten()[at]):.6e}, "
                                     f"exactly {float(out.flatten()[at]):.6e}, bound {float(bound.flatten()[at]):.3e}")
