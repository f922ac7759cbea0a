"""Plain 64-bit reference of the quantized-cache steps, and inputs for their tests."""
import numpy as np

import oracle
from aion_b200 import capi
from tests import refdata as rd  # noqa: F401  (re-exported for the tests)

F32, F16, Q4, Q8, I32 = capi.DTYPE_F32, capi.DTYPE_F16, capi.DTYPE_Q4_0, capi.DTYPE_Q8_0, capi.DTYPE_I32
BLOCK = {Q4: 18, Q8: 34}
NP = {F32: np.float32, F16: np.float16}


def pack(dtype, rows):
    """f32 [..., D] -> the stored rows: bytes [..., D / 32 * block] of a quantized cache, else the cast values."""
    if dtype not in BLOCK:
        return rows.astype(NP[dtype])
    D = rows.shape[-1]
    flat = np.ascontiguousarray(rows, dtype=np.float32).reshape(-1, D)
    return oracle.quantize(dtype, flat, 1).reshape(*rows.shape[:-1], D // 32 * BLOCK[dtype])


def unpack(dtype, stored):
    """The stored rows as f64 values (code x scale)."""
    if dtype not in BLOCK:
        return stored.astype(np.float64)
    b = stored.reshape(*stored.shape[:-1], -1, BLOCK[dtype])
    scale = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    if dtype == Q8:
        code = np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64)
    else:
        code = np.stack([b[..., 2:] & 15, b[..., 2:] >> 4], -1).reshape(*b.shape[:-1], 32).astype(np.float64) - 8
    with np.errstate(invalid="ignore"):
        return (code * scale).reshape(*stored.shape[:-1], -1)


def to_pool(cache, page, rng, spare=2):
    """A contiguous cache [B, T, ...] as (pool [pages, page, ...], table [B, ceil(T / page)]); spare room is 0xFF bytes (NaN)."""
    B, T = cache.shape[:2]
    per = -(-T // page)
    pool = np.empty((B * per + spare, page, *cache.shape[2:]), dtype=cache.dtype)
    pool.view(np.uint8)[:] = 0xFF
    table = rng.permutation(B * per + spare)[: B * per].reshape(B, per).astype(np.int32)
    for b in range(B):
        for i in range(per):
            part = cache[b, i * page:(i + 1) * page]
            pool[table[b, i], : part.shape[0]] = part
    return pool, table


def key_range(pos, length, T, rolling, left, right, chunk):
    unb = capi.WINDOW_UNBOUNDED
    anchor = pos // chunk * chunk if chunk else pos
    lo = max(0, anchor - left) if left != unb else 0
    hi = length if right == unb else min(length, anchor + (chunk or 1) + right)
    if rolling:
        lo = max(lo, length - T)
    return lo, max(lo, hi)


def attention(q, k, v, kdt, vdt, *, scale, positions, lengths, left=capi.WINDOW_UNBOUNDED, right=0, chunk=0, cap=0.0, rolling=False):
    """(out f64 [B, L, Hq, D], bound): stored k, v [B, T, Hkv, bytes]. `bound` is how far an f32 evaluation may be off, element by
    element, to first order, with eps = 2^-24 the rounding of one f32 operation:
      a logit is off by   (D + 8) eps scale sum|q k|          (a sum of D products in any order, and its scaling)
                        + 2^-22 scale max|q| sum|k|           (q in two f16 terms of 11 bits, normed by its largest value)
                        + 2^-20 cap                           (a division, tanh to 2^-22, a product)
                        + 2^-22 |logit|                       (its move to base 2, the subtraction of the maximum)
      a weight by that, relatively, and 2^-21 for exp2 and its two f16 terms;
      the quotient by twice the largest of these and by (N + 64) eps for its sums of N terms and the rescalings on the way,
    each times sum w |v| / sum w."""
    B, L, Hq, D = q.shape
    positions = np.asarray(positions)
    T, H = k.shape[1], k.shape[2]
    G = Hq // H
    out, bound = np.zeros((B, L, Hq, D)), np.zeros((B, L, Hq, D))
    eps = 2.0 ** -24
    for b in range(B):
        for l in range(L):
            lo, hi = key_range(int(positions[b, l]), int(lengths[b]), T, rolling, left, right, chunk)
            if hi <= lo:
                continue
            rows = np.arange(lo, hi) % T if rolling else np.arange(lo, hi)
            for h in range(H):
                kk, vv = unpack(kdt, k[b, rows, h]), unpack(vdt, v[b, rows, h])
                for g in range(G):
                    x = q[b, l, h * G + g].astype(np.float64)
                    y = kk @ x * scale
                    dy = (D + 8) * eps * scale * (np.abs(kk) @ np.abs(x)) + 2.0 ** -22 * scale * np.abs(x).max() * np.abs(kk).sum(1)
                    if cap:
                        y = cap * np.tanh(y / cap)
                        dy = dy + 2.0 ** -20 * cap
                    dy = dy + 2.0 ** -22 * np.abs(y)
                    w = np.exp(y - y.max())
                    mean_abs = w @ np.abs(vv) / w.sum()
                    out[b, l, h * G + g] = w @ vv / w.sum()
                    bound[b, l, h * G + g] = (2 * (dy.max() + 2.0 ** -21) + (hi - lo + 64) * eps) * mean_abs
    return out, bound


def norm_rope(x, gamma, positions, eps, base, proportion=1.0, scale_factor=1.0):
    """RMSNorm of every head of x [B, L, H, D] (gamma None: none) and RoPE1D, in f64; the angles are f32 by definition."""
    D = x.shape[-1]
    y = x.astype(np.float64)
    if gamma is not None:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps) * gamma.astype(np.float64)
    half = D // 2
    n = min(half, int(np.floor(np.float32(proportion) * np.float32(half))))
    step = np.float32(float(np.float32(base)) ** float(np.float32(-2.0) / np.float32(D)))
    f = np.empty(n, np.float32)
    cur = np.float32(scale_factor)
    for i in range(n):
        f[i] = cur
        cur = np.float32(cur * step)
    ang = (positions.astype(np.float32)[..., None] * f).astype(np.float64)[:, :, None]
    lo, hi = y[..., :n], y[..., half:half + n]
    out = y.copy()
    out[..., :n] = lo * np.cos(ang) - hi * np.sin(ang)
    out[..., half:half + n] = lo * np.sin(ang) + hi * np.cos(ang)
    return out
