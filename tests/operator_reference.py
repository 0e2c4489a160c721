"""Plain 64-bit implementations of the serving operators, for their tests."""
import math

import numpy as np


def bf16_bits(x):
    """float32 array -> bf16 values (round to nearest even) as float32."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16) << 16
    return r.astype(np.uint32).view(np.float32)


def directed_bf16(x, up):
    """Doubles rounded up (or down) to bf16, as doubles; |x| in bf16's normal range or zero."""
    m, e = np.frexp(np.asarray(x, np.float64))     # x = m 2^e, 1/2 <= |m| < 1
    whole = np.ceil(m * 256.0) if up else np.floor(m * 256.0)
    return np.ldexp(whole, e - 8)


def quantise(x):
    """[..., dim] -> (codes [..., dim / 2] uint8, step and low [..., dim / 32], values float64)."""
    x = np.asarray(x, np.float64)
    dim = x.shape[-1]
    g = x.reshape(*x.shape[:-1], dim // 32, 32)
    low = directed_bf16(g.min(-1), False)
    step = directed_bf16((g.max(-1) - low) / 15.0, True)
    code = np.rint((g - low[..., None]) / np.where(step > 0, step, 1.0)[..., None])
    code = np.clip(np.where(step[..., None] > 0, code, 0), 0, 15)
    values = (low[..., None] + code * step[..., None]).reshape(x.shape)
    code = code.astype(np.uint8).reshape(x.shape)
    packed = np.zeros((*x.shape[:-1], dim // 2), np.uint8)
    for c in range(dim):
        group, half, nibble = c // 32, c % 32 // 4, c % 4
        byte = (half * (dim // 32) + group) * 2 + nibble // 2
        packed[..., byte] |= code[..., c] << (4 * (nibble % 2))
    return packed, step, low, values


def visible(position, keys, window, sinks):
    j = np.arange(keys)
    seen = j <= position
    if window:
        seen &= (position - j < window) | (j < sinks)
    return seen


def attend(q, k, v, first, window, sinks, scale):
    """One sequence: q [n, H, d] at positions first.., k and v [keys, KV, d]; out and, per query and
    head, the largest sum |q k| scale over its visible keys."""
    n, H, d = q.shape
    out = np.zeros((n, H, d))
    size = np.zeros((n, H))
    for i in range(n):
        seen = visible(first + i, k.shape[0], window, sinks) if first + i >= 0 else \
            np.zeros(k.shape[0], bool)
        if not seen.any():
            continue
        for h in range(H):
            kk, vv = k[seen, h * k.shape[1] // H], v[seen, h * k.shape[1] // H]
            s = kk @ q[i, h] * scale
            p = np.exp(s - s.max())
            out[i, h] = p @ vv / p.sum()
            size[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
    return out, size


def draw_token(logits, u, temperature, top_k, top_p, min_p):
    """The token, and how far (in the largest weight) the target is from the nearest border."""
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    V, top = len(x), x.max()
    if top == -np.inf:
        return -1, math.inf
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), math.inf
    with np.errstate(invalid="ignore"):
        z = np.where(x == top, 0.0, (x - top) / float(temperature))
    w = np.where(z >= -40 * math.log(2), np.exp(np.where(np.isnan(z), -np.inf, z)), 0.0)
    w[x == -np.inf] = 0.0
    s = w[order]
    keep = np.ones(V, bool)
    if top_k > 0:
        keep[top_k:] = False
    s = np.where(keep, s, 0.0)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(s)[:-1]])
        keep &= before < float(top_p) * s.sum()
        keep[0] = True
    if min_p > 0:
        keep &= s >= min(float(min_p), 1.0)
    w = np.zeros(V)
    w[order] = np.where(keep, s, 0.0)
    c = np.cumsum(w)
    target = min(max(float(u), 0.0), 1 - 2.0 ** -53) * c[-1]
    token = int((c <= target).sum())
    return token, float(np.abs(c - target).min())
