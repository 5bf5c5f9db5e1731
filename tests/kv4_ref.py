"""64-bit restatement of the 4-bit paged key/value cache (q3t_kv4_*), spelled
out token by token: the block layout, the quantisation, rotary positions, and
attention over what the cache holds.  Shares no code with the library."""
import math

import numpy as np


def block_tables(D):
    """For a block of head_dim D: byte and shift of every (token, dim) digit of K and V, and the bf16 index of the
    {K scale, K zero, V scale, V zero} of every (token, dim)."""
    kb, ks, vb, vs, sc = (np.zeros((16, D), np.int64) for _ in range(5))
    G = D // 32
    for c in range(16):
        for d in range(D):
            j, t, b0, h, b1 = d // 32, d // 8 % 4, d // 4 % 2, d // 2 % 2, d % 2
            kb[c, d] = c * D // 2 + 4 * (G * t + j) + 2 * b1 + b0
            ks[c, d] = 4 * h
            M, m, h, g = d // 64, d // 16 % 4, d // 8 % 2, d % 8
            b0, t, b1 = c // 8, c // 2 % 4, c % 2
            vb[c, d] = 8 * D + 512 * M + 16 * (4 * g + t) + 4 * m + 2 * b1 + b0
            vs[c, d] = 4 * h
            sc[c, d] = (16 * D + 8 * (4 * (4 * j + t) + 2 * b0 + b1)) // 2
    return kb, ks, vb, vs, sc


def bf16_bits(x):
    """Round-to-nearest-even bf16 bit patterns of float32 values (finite)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(bits):
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def unpack(pool, D):
    """Keys, values and their scales [pages, heads, 16, D] in float64 of a uint8 pool [pages, heads, 20 D]."""
    kb, ks, vb, vs, sc = block_tables(D)
    with np.errstate(invalid="ignore"):  # stale blocks hold scales that are no numbers
        half = bf16_value(pool.reshape(*pool.shape[:2], -1).view(np.uint16)).astype(np.float64)
        k_s, k_z, v_s, v_z = (half[..., sc + i] for i in range(4))
        k = (pool[..., kb] >> ks & 15) * k_s + k_z
        v = (pool[..., vb] >> vs & 15) * v_s + v_z
    return k, v, k_s, v_s


def quantise(x):
    """(digits, scale, zero) of float32 x [..., D], the definition in float32 step by step."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.min(-1), g.max(-1)
    down = bf16_value(bf16_bits(lo))  # nearest, then one step down where that is above
    bits = bf16_bits(lo)
    above = down > lo
    neg = (bits >> 15).astype(bool)
    bits = np.where(above, np.where(neg | (bits == 0), bits + 1, bits - 1), bits).astype(np.uint16)
    zero = bf16_value(bits)
    scale = bf16_value(bf16_bits((hi * np.float32(0.5) - zero * np.float32(0.5)) * np.float32(2.0 / 15.0)))
    with np.errstate(all="ignore"):
        n = np.clip(np.rint((g - zero[..., None]) / scale[..., None]), 0, 15)
    n = np.where(scale[..., None] > 0, n, 0)
    return n.astype(np.uint8).reshape(x.shape), scale, zero


def frequencies(rot, theta, scaling="none", factor=1.0, low=1.0, high=4.0, original=4096):
    out = []
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        elif scaling == "bands":
            turns = original * f / (2 * math.pi)
            w = (turns - low) / (high - low)
            w = 0.0 if w < 0 else 1.0 if w > 1 else w
            f = w * f + (1 - w) * f / factor
        out.append(f)
    return np.array(out, np.float64)


def rotate(x, pos, freqs, layout, amplitude=1.0):
    """x [T, heads, D] float64 with its leading 2 len(freqs) dims turned."""
    x = x.copy()
    n = len(freqs)
    ang = np.asarray(pos, np.float64)[:, None] * freqs
    c, s = np.cos(ang)[:, None] * amplitude, np.sin(ang)[:, None] * amplitude
    a = x[..., :n].copy() if layout == "half" else x[..., 0:2 * n:2].copy()
    b = x[..., n:2 * n].copy() if layout == "half" else x[..., 1:2 * n:2].copy()
    if layout == "half":
        x[..., :n], x[..., n:2 * n] = a * c - b * s, b * c + a * s
    else:
        x[..., 0:2 * n:2], x[..., 1:2 * n:2] = a * c - b * s, b * c + a * s
    return x


def rms_norm(x, gamma, eps):
    return x if gamma is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma


def places(q_start, kv_len):
    """(row, sequence, position) of every row of the batch."""
    out = []
    for s in range(len(kv_len)):
        n = q_start[s + 1] - q_start[s]
        out += [(q_start[s] + i, s, kv_len[s] - n + i) for i in range(n)]
    return out


def attend(q, k_pool, v_pool, table, q_start, kv_len, scale, window=0, table_row=None, num_pages=None):
    """(out, bound) [T, heads, D]: attention in float64 over unpacked pools, and for every output the largest
    |value| of the dims' group among the keys its row sees (what its error scales with)."""
    T, H, D = q.shape
    kvh = k_pool.shape[1]
    P = k_pool.shape[0] if num_pages is None else num_pages
    out, bound = np.zeros((T, H, D)), np.zeros((T, H, D))
    for row, s, pos in places(q_start, kv_len):
        tr = s if table_row is None else table_row[s]
        lo = max(0, pos - window + 1) if window else 0
        keys = [p for p in range(lo, pos + 1) if p // 16 < table.shape[1] and 0 <= table[tr, p // 16] < P]
        if not keys:
            continue
        pg, sl = table[tr, np.array(keys) // 16], np.array(keys) % 16
        for h in range(H):
            kk, vv = k_pool[pg, h * kvh // H, sl], v_pool[pg, h * kvh // H, sl]
            y = kk @ q[row, h] * scale
            w = np.exp(y - y.max())
            out[row, h] = w @ vv / w.sum()
            bound[row, h] = np.repeat(np.abs(vv).max(0).reshape(-1, 32).max(1), 32)
    return out, bound
