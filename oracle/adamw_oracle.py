"""CPU oracle of the AdamW operators (adamw.py).  TEST INFRASTRUCTURE: only tests/ may import this.

``step64`` is the update in float64 from the formulas.  ``step8`` is the 8-bit form operation by operation in float32 (numpy's
+, *, / and sqrt round correctly, as the kernel's do), so that codes can be compared one by one; ``level_*`` give what a
code stands for in float64 from the definition of the format, apart from the bit patterns."""
import math

import numpy as np

f32 = np.float32
BLOCK = 64
M32 = 0xFFFFFFFF
ONE = 0x3F800000


def step64(p, g, m, v, t, lr, beta1, beta2, eps, weight_decay, coef=1.0):
    """-> (p, m, v, |update|, |beta1 m| + |(1 - beta1) g|, denominator), all float64; inputs untouched."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    g = g * coef
    size = np.abs(beta1 * m) + np.abs((1 - beta1) * g)
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    d = np.sqrt(v) / math.sqrt(1 - beta2 ** t) + eps
    with np.errstate(invalid="ignore", divide="ignore"):
        upd = lr / (1 - beta1 ** t) * m / d
    return p * (1 - lr * weight_decay) - upd, m, v, np.abs(upd), size, d


def mix(x):
    x = np.asarray(x, np.uint64) & np.uint64(M32)
    for shift, mul in ((16, 0x6A09E667), (15, 0xBB67AE85)):
        x = x ^ (x >> np.uint64(shift))
        x = (x * np.uint64(mul)) & np.uint64(M32)
    return x ^ (x >> np.uint64(16))


def random_bits(n, seed, index, t, first=0):
    """32 random bits for elements first..first+n-1 of tensor `index` at update t."""
    with np.errstate(over="ignore"):
        key = mix(int(mix((seed + 0x9E3779B9 * (index + 1)) & M32)) ^ (t & M32))
        e = np.arange(first, first + n, dtype=np.uint64)
        return mix((e & np.uint64(M32)) + key + (e >> np.uint64(32)) * np.uint64(0x3C6EF373))


def level_m(codes, scale):
    """float64 value of the first moment's codes: 8 levels per octave down from the scale."""
    c = np.asarray(codes).astype(np.int64)
    q = (c & 127) - 127
    f = np.exp2((q // 8).astype(np.float64)) * (1 + (q % 8) / 8)
    return np.where((c & 127) == 0, 0.0, f) * np.where(c & 128, -1.0, 1.0) * np.asarray(scale, np.float64)


def level_u(codes, scale):
    """float64 value of the second moment root's codes: 16 levels per octave."""
    q = np.asarray(codes).astype(np.int64) - 255
    f = np.exp2((q // 16).astype(np.float64)) * (1 + (q % 16) / 16)
    return np.where(q == -255, 0.0, f) * np.asarray(scale, np.float64)


def _blocks(x):
    x = np.asarray(x).reshape(-1)
    return np.concatenate([x, np.zeros(-x.size % BLOCK, x.dtype)]).reshape(-1, BLOCK)


def unpack(codes, scales):
    """(m, u) float32 of codes (n, 2) and scales (blocks, 2)."""
    n = codes.shape[0]
    s = np.repeat(scales, BLOCK, axis=0)[:n]
    c = codes.astype(np.int64)
    mag = c[:, 0] & 127
    fm = np.where(mag > 0, (ONE - ((127 - mag) << 20)).astype(np.uint32).view(f32), f32(0)) * s[:, 0]
    fu = np.where(c[:, 1] > 0, (ONE - ((255 - c[:, 1]) << 19)).astype(np.uint32).view(f32), f32(0)) * s[:, 1]
    return np.where(c[:, 0] & 128, -fm, fm).astype(f32), fu.astype(f32)


def pack(m, u, random=None):
    """codes (n, 2) uint8 and scales (blocks, 2) float32 of finite float32 m and u >= 0; random None: nearest level."""
    n = m.size
    r = np.full(n, 0x80008000, np.uint64) if random is None else random
    rb = _blocks(r)
    rm, ru = (rb & np.uint64(0xFFFF)).astype(np.int64), (rb >> np.uint64(16)).astype(np.int64)
    out, scales = [], []
    for x, is_m in ((np.abs(_blocks(m.astype(f32))), True), (_blocks(u.astype(f32)), False)):
        s = x.max(axis=1, keepdims=True) if x.size else np.zeros((0, 1), f32)
        s = np.where(s < f32(2.0 ** -126), f32(0), s)
        with np.errstate(divide="ignore", invalid="ignore"):
            inv = np.where(s > 0, f32(1) / s, f32(0)).astype(f32)
        rel = np.minimum(x * inv, f32(1)).astype(f32)
        bits = rel.view(np.uint32).astype(np.int64)
        if is_m:
            c = 127 + ((bits + rm * 16 - ONE) >> 20)
            low = (rel * f32(65536.0 / (1.25 * 2.0 ** -16)) > rm.astype(f32)).astype(np.int64)
            c = np.where(c < 1, low, c)
            c = c + np.where((_blocks(m) < 0) & (c > 0), 128, 0)
        else:
            c = np.maximum(255 + ((bits + ru * 8 - ONE) >> 19), 1)
            c = np.where((x == 0) | (s == 0), 0, c)
        out.append(c.reshape(-1)[:n].astype(np.uint8))
        scales.append(s)
    return np.stack(out, 1), np.concatenate(scales, 1).astype(f32)


def step8(p, g, codes, scales, t, lr, beta1, beta2, eps, weight_decay, random=None, coef=None):
    """One update with 8-bit states in float32 -> (p float32, codes, scales)."""
    g = np.asarray(g, f32).reshape(-1)
    if coef is not None:
        g = g * f32(coef)
    m, u = unpack(codes.reshape(-1, 2), scales)
    v = u * u
    m = m * f32(beta1) + g * f32(1 - beta1)
    v = v * f32(beta2) + (g * g) * f32(1 - beta2)
    u = np.sqrt(v)
    root = math.sqrt(1 - beta2 ** t)
    with np.errstate(invalid="ignore", divide="ignore"):
        upd = f32(-(lr / (1 - beta1 ** t))) * (m / (u * f32(1 / root) + f32(eps)))
    x = np.asarray(p, f32).reshape(-1) * f32(1 - lr * weight_decay) + upd
    c, s = pack(m, u, random)
    return x, c, s


def join(bf16_bits, low):
    """float32 behind bf16 bits (uint16) and a remainder (int16)."""
    return ((bf16_bits.astype(np.int64) << 16) + low.astype(np.int64)).astype(np.uint32).view(f32)


def split(x):
    """-> (bf16 bits uint16, remainder int16); halves away from zero."""
    b = np.asarray(x, f32).view(np.uint32).astype(np.int64)
    high = (b + 0x8000) >> 16
    return high.astype(np.uint16), (b - (high << 16)).astype(np.int16)
