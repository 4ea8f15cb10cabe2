"""CPU restatement, in 64 bits, of the operators around a paged key/value cache: rotary embedding, quantised vectors, the append to
pages, and attention over the tokens of a sequence.  Test infrastructure only."""
import math

import numpy as np

LIMIT = {8: 127, 4: 7}


def rope(x, position, turns, interleaved=False, magnitude=1.0):
    """x [..., head_dim] float64 at one position."""
    out = np.array(x, np.float64)
    n = len(turns)
    if n == 0:
        return out
    angle = 2.0 * math.pi * np.remainder(position * np.asarray(turns, np.float64), 1.0)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = out[..., first].copy(), out[..., second].copy()
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    return out


def quantise(x, bits):
    """(codes int, scale float32) of vectors x [..., head_dim]."""
    m = LIMIT[bits]
    top = np.abs(x).max(-1, keepdims=True)
    codes = np.rint(np.divide(x * m, top, out=np.zeros_like(x), where=top > 0)).astype(np.int64)
    return codes, (top[..., 0] / m).astype(np.float32)


def pack(codes, bits):
    if bits == 8:
        return codes.astype(np.int8).view(np.uint8)
    c = (codes + 8).astype(np.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def unpack(stored, bits):
    if bits == 8:
        return stored.view(np.int8).astype(np.int64)
    return np.stack((stored & 15, stored >> 4), -1).reshape(stored.shape[:-1] + (-1,)).astype(np.int64) - 8


def attention(q, keys, values, first_position, scale, window=0):
    """q [n, heads, d], keys and values [tokens, kv_heads, d]; row i at position first_position + i.  Returns (out, sum_j p_j |v_j|, largest
    scale * sum |q k| of a visible key, visible keys, largest |v|) per row and head, for error bounds; a row that sees nothing is zero."""
    n, heads, d = q.shape
    group = heads // keys.shape[1] if keys.shape[1] else 1
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    most, seen, top_v = np.zeros((n, heads)), np.zeros((n, heads)), np.zeros((n, heads))
    for i in range(n):
        end = min(first_position + i + 1, len(keys))
        start = max(0, first_position + i + 1 - window) if window else 0
        if end <= start:
            continue
        for h in range(heads):
            k, v = keys[start:end, h // group], values[start:end, h // group]
            s = scale * (k @ q[i, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], mass[i, h] = p @ v, p @ np.abs(v)
            most[i, h] = abs(scale) * (np.abs(k) @ np.abs(q[i, h])).max()
            seen[i, h], top_v[i, h] = end - start, np.abs(v).max()
    return out, mass, most, seen, top_v
