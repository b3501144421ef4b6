"""Caches that hold a token in few bytes, in float64 numpy: the definitions of the 4-bit cache
(``ops.store_kvcache_mxfp4``, ``gather_kvcache_mxfp4``, ``mxfp4_paged_decode``) and of the latent
cache (``ops.latent_norm_rope_store``, ``gather_latent``, ``latent_decode``), one row at a time.

Each takes float arrays (bf16 and fp8 values widened by the caller).
"""
from __future__ import annotations

import numpy as np

from .partial import _attend, query_rows

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mxfp4_blocks(x):
    """x [..., D] -> (scale bytes [..., D / 32], codes [..., D])."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    m, e = np.frexp(np.where(bad, 1.0, top))  # top = m 2^e, 0.5 <= m < 1
    # (at most 252: 253's code for the greatest values would be 2^128, which bf16 has not)
    scale = np.where(top > 0, np.clip(e - 1 + (m >= 0.875) - 2 + 127, 0, 252), 0).astype(np.int64)
    v = np.abs(np.where(bad[..., None], 0.0, b)) / 2.0 ** (scale[..., None] - 127)
    code = np.zeros(b.shape, np.int64)
    for i in range(7):  # past the middle of codes i and i + 1; on it, to the even one
        mid = (GRID[i] + GRID[i + 1]) / 2
        code += (v > mid) | ((v == mid) & (i % 2 == 1))
    code |= (np.signbit(b) & ~bad[..., None]).astype(np.int64) << 3
    return np.where(bad, 255, scale).astype(np.uint8), code.astype(np.uint8).reshape(x.shape)


def mxfp4_values(scales, codes):
    """The inverse: codes [..., D] with scale bytes [..., D / 32] as float64 (255: NaN)."""
    codes = np.asarray(codes).reshape(*scales.shape, 32)
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    s = np.where(scales == 255, np.nan, 2.0 ** (np.minimum(scales, 254).astype(np.float64) - 127))
    return (v * s[..., None]).reshape(*codes.shape[:-2], -1)


def _nibbles(b):
    """Bytes [..., n] -> codes [..., 2 n], the low one first."""
    return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


def mxfp4_cache_values(k_cache, v_cache, k_scales, v_scales):
    """(k, v) [num_blocks, block_size, Hk, D] of the four uint8 arrays of a 4-bit cache."""
    nb, hk, page, half = k_cache.shape
    k = _nibbles(k_cache)
    v = _nibbles(v_cache)  # [nb, hk, page / 4, 16, 4, D / 16]
    v = v.transpose(0, 1, 2, 4, 3, 5).reshape(nb, hk, page, 2 * half)
    out = [mxfp4_values(s.transpose(0, 1, 3, 2), c) for s, c in ((k_scales, k), (v_scales, v))]
    return tuple(x.transpose(0, 2, 1, 3) for x in out)


def gather(cache, block_table, cu_seqlens_k, rows):
    """Rows [rows, ...] of a cache [num_blocks, block_size, ...]: zeros at masked pages, NaN in
    rows of no sequence."""
    nb, page = cache.shape[:2]
    out = np.full((rows, *cache.shape[2:]), np.nan)
    for b in range(len(cu_seqlens_k) - 1):
        for t in range(int(cu_seqlens_k[b]), min(int(cu_seqlens_k[b + 1]), rows)):
            j, i = divmod(t - int(cu_seqlens_k[b]), page)
            p = int(block_table[b, j]) if j < block_table.shape[1] else -1
            out[t] = cache[p, i] if 0 <= p < nb else 0.0
    return out


def _visible(caches, table, lo, hi):
    """Keys [lo, hi) of a sequence out of each cache, without those of masked pages."""
    nb, page = caches[0].shape[:2]
    out = [[np.zeros((0, *c.shape[2:]))] for c in caches]
    for j in range(lo // page, min(-(-hi // page), len(table))):
        p = int(table[j])
        if 0 <= p < nb:
            s = slice(max(lo - j * page, 0), min(hi - j * page, page))
            for o, c in zip(out, caches):
                o.append(c[p, s])
    return [np.concatenate(o) for o in out]


def paged_decode(q, k_cache, v_cache, block_table, cache_seqlens, scale, window_left=-1,
                 sinks=None, cu_seqlens_q=None):
    """(rows, averages of |v|, largest magnitudes), each [rows, Hq, D]; NaN in rows of none."""
    rows, hq, d = q.shape
    hk = k_cache.shape[2]
    g = hq // hk
    out, mean, mag = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros(q.shape)
    for t, b, vis in query_rows(cache_seqlens, cu_seqlens_q, rows):
        if t >= rows:
            continue
        lo = max(0, vis - 1 - window_left) if window_left >= 0 else 0
        k, v = _visible((k_cache, v_cache), block_table[b], lo, max(vis, 0))
        for h in range(hk):
            s = slice(h * g, (h + 1) * g)
            out[t, s], mean[t, s], mag[t, s] = _attend(q[t, s], k[:, h], v[:, h], scale,
                                                       None if sinks is None else sinks[s])
    return out, mean, np.abs(mag)


def latent_decode(q, cache, block_table, cache_seqlens, scale, latent=512, cu_seqlens_q=None):
    """(rows, averages of |c|, largest magnitudes) [rows, H, latent] and the log-sum-exp
    [H, rows]; NaN in rows of none."""
    rows, heads, _ = q.shape
    shape = (rows, heads, latent)
    out, mean, mag = np.full(shape, np.nan), np.zeros(shape), np.zeros(shape)
    lse = np.full((heads, rows), np.nan)
    for t, b, vis in query_rows(cache_seqlens, cu_seqlens_q, rows):
        if t >= rows:
            continue
        k, = _visible((cache,), block_table[b], 0, max(vis, 0))
        lse[:, t] = -np.inf
        if len(k) == 0:
            out[t] = 0.0
            continue
        x = scale * (q[t] @ k.T)
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        total = e.sum(1, keepdims=True)
        out[t], mean[t] = e / total @ k[:, :latent], e / total @ np.abs(k[:, :latent])
        mag[t] = abs(scale) * (np.abs(q[t]) @ np.abs(k).T).max()
        lse[:, t] = (m + np.log(total))[:, 0]
    return out, mean, mag, lse


def rotate(x, position, cos_sin, is_neox):
    """x [..., P] rotated by the angles of a position, as it is outside the table."""
    if not 0 <= position < len(cos_sin):
        return np.array(x, np.float64)
    half = x.shape[-1] // 2
    c, s = cos_sin[position, :half], cos_sin[position, half:]
    a, b = (x[..., :half], x[..., half:]) if is_neox else (x[..., ::2], x[..., 1::2])
    y = (a * c - b * s, b * c + a * s)
    return np.concatenate(y, -1) if is_neox else np.stack(y, -1).reshape(x.shape)


def latent_rows(latent, key_rope, positions, cos_sin, is_neox, weight=None, eps=1e-6):
    """(c [N, R], k [N, P]): the normed latents and the rotated keys."""
    c = np.asarray(latent, np.float64)
    if weight is not None:
        c = c / np.sqrt((c * c).mean(-1, keepdims=True) + eps) * weight
    return c, np.stack([rotate(k, int(p), cos_sin, is_neox) for k, p in zip(key_rope, positions)])
