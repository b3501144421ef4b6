"""Attention that reads part of a paged cache, in float64 numpy: the definitions of
``ops.update_key_bounds``, ``block_scores``, ``select_blocks``, ``sparse_paged_decode`` and
``shared_prefix_decode``, one row at a time.

Each takes float arrays (fp8 and bf16 values widened by the caller); the attention functions
also return what a tolerance is made of: the same average of |v|, and the largest
scale * sum_d |q_d k_d| of a row.
"""
from __future__ import annotations

import numpy as np


def query_rows(cache_seqlens, cu_seqlens_q=None, rows=None):
    """(row, sequence, visible keys) of every query row of the batch."""
    if cu_seqlens_q is None:
        n = len(cache_seqlens) if rows is None else rows
        return [(b, b, int(cache_seqlens[b])) for b in range(n)]
    out = []
    for b in range(len(cu_seqlens_q) - 1):
        lo, hi = int(cu_seqlens_q[b]), int(cu_seqlens_q[b + 1])
        out += [(t, b, int(cache_seqlens[b]) - (hi - 1 - t)) for t in range(lo, hi)]
    return out


def update_key_bounds(bounds, k_cache, block_table, cache_seqlens, cu_seqlens_q=None):
    """bounds [blocks, Hk, 2, D] with the touched pages replaced (a copy)."""
    out = np.array(bounds, np.float64)
    page = k_cache.shape[1]
    for b, n in enumerate(cache_seqlens if cu_seqlens_q is None
                          else cache_seqlens[:len(cu_seqlens_q) - 1]):
        n = int(n)
        new = 1 if cu_seqlens_q is None else int(cu_seqlens_q[b + 1] - cu_seqlens_q[b])
        if n <= 0 or new <= 0:
            continue
        for j in range(max(n - new, 0) // page, -(-n // page)):
            p = int(block_table[b, j]) if j < block_table.shape[1] else -1
            if 0 <= p < k_cache.shape[0]:
                x = np.asarray(k_cache[p, :n - j * page], np.float64)
                out[p, :, 0], out[p, :, 1] = x.min(0), x.max(0)
    return out


def block_scores(q, bounds, block_table, cache_seqlens, page, width, k_scale=None,
                 cu_seqlens_q=None):
    """(scores, magnitudes) [rows, Hk, width]; rows behind the last sequence are NaN.  The
    magnitudes are sum_d |q_d| max(|lo_d|, |hi_d|), for a tolerance."""
    rows, hq, d = q.shape
    hk = bounds.shape[1]
    out = np.full((rows, hk, width), np.nan)
    mag = np.zeros((rows, hk, width))
    ks = np.ones(hk) if k_scale is None else np.asarray(k_scale, np.float64)
    q = np.asarray(q, np.float64).reshape(rows, hk, hq // hk, d)
    for t, b, vis in query_rows(cache_seqlens, cu_seqlens_q, rows):
        out[t] = -np.inf
        for j in range(min(-(-max(vis, 0) // page), width, block_table.shape[1])):
            p = int(block_table[b, j])
            if 0 <= p < bounds.shape[0]:
                x = np.asarray(bounds[p], np.float64) * ks[:, None, None]
                e = np.maximum(q[t] * x[:, None, 0], q[t] * x[:, None, 1]).sum(-1)
                out[t, :, j] = e.max(1)
                mag[t, :, j] = (np.abs(q[t]) * np.abs(x).max(1)[:, None]).sum(-1).max(1)
    return out, mag


def select_blocks(scores, cache_seqlens, page, keep, keep_first, keep_last, cu_seqlens_q=None,
                  fill=-7):
    """int64 [rows, Hk, keep]; rows behind the last sequence hold ``fill``."""
    rows, hk, width = scores.shape
    out = np.full((rows, hk, keep), fill, np.int64)
    for t, _, vis in query_rows(cache_seqlens, cu_seqlens_q, rows):
        n = min(-(-max(vis, 0) // page), width)
        for h in range(hk):
            s = scores[t, h, :n]
            rank = sorted(range(n), key=lambda j: (
                not (j < keep_first or j >= n - keep_last),
                (0, 0.0) if np.isnan(s[j]) else (1, -float(s[j])), j))
            best = sorted(rank[:keep])
            out[t, h] = best + [-1] * (keep - len(best))
    return out


def _attend(q, k, v, scale, sinks):
    """q [G, D], k / v [keys, D], sinks [G] or None: (row, average |v|, largest magnitude)."""
    if len(k) == 0:
        return np.zeros_like(q), np.zeros_like(q), 0.0
    x = scale * (q @ k.T)
    m = x.max(1) if sinks is None else np.maximum(x.max(1), sinks)
    e = np.exp(x - m[:, None])
    total = e.sum(1)
    if sinks is not None:
        total = total + np.exp(sinks - m)
    w = e / total[:, None]
    return w @ v, w @ np.abs(v), float(scale * (np.abs(q) @ np.abs(k).T).max())


def _attend_rows(q, hk, keys_of, scale, sinks):
    """keys_of(row, kv head) -> (k, v) or None for a row that is not written (NaN)."""
    rows, hq, d = q.shape
    g = hq // hk
    out = np.full((rows, hk, g, d), np.nan)
    mean = np.zeros_like(out)
    mag = np.zeros((rows, hk, 1, 1))
    q = np.asarray(q, np.float64).reshape(rows, hk, g, d)
    s = None if sinks is None else np.asarray(sinks, np.float64).reshape(hk, g)
    for t in range(rows):
        for h in range(hk):
            kv = keys_of(t, h)
            if kv is not None:
                out[t, h], mean[t, h], mag[t, h] = _attend(q[t, h], *kv, scale,
                                                           None if s is None else s[h])
    shape = (rows, hq, d)
    mag = np.broadcast_to(mag, out.shape)
    return out.reshape(shape), mean.reshape(shape), mag.reshape(shape)


def _scales(scale, hk):
    return np.ones(hk) if scale is None else np.asarray(scale, np.float64)


def sparse_paged_decode(q, k_cache, v_cache, block_table, cache_seqlens, indices, scale,
                        k_scale=None, v_scale=None, sinks=None, cu_seqlens_q=None):
    nb, page, hk, _ = k_cache.shape
    ks, vs = _scales(k_scale, hk), _scales(v_scale, hk)
    info = {t: (b, vis) for t, b, vis in query_rows(cache_seqlens, cu_seqlens_q, q.shape[0])}

    def keys_of(t, h):
        if t not in info:
            return None
        b, vis = info[t]
        k, v = [np.zeros((0, q.shape[2]))], [np.zeros((0, q.shape[2]))]
        for j in indices[t, h]:
            j = int(j)
            p = int(block_table[b, j]) if 0 <= j < block_table.shape[1] else -1
            n = min(page, vis - j * page)
            if 0 <= p < nb and n > 0:
                k.append(np.asarray(k_cache[p, :n, h], np.float64) * ks[h])
                v.append(np.asarray(v_cache[p, :n, h], np.float64) * vs[h])
        return np.concatenate(k), np.concatenate(v)

    return _attend_rows(q, hk, keys_of, scale, sinks)


def shared_prefix_decode(q, k_cache, v_cache, block_table, cache_seqlens, cu_groups,
                         prefix_lens, scale, k_scale=None, v_scale=None, window_left=-1,
                         sinks=None):
    nb, page, hk, d = k_cache.shape
    ks, vs = _scales(k_scale, hk), _scales(v_scale, hk)
    table = {b: (b, 0) for b in range(q.shape[0])}  # row -> (row of the prefix's table, length)
    for g in range(len(cu_groups) - 1):
        for b in range(int(cu_groups[g]), int(cu_groups[g + 1])):
            table[b] = (int(cu_groups[g]), int(prefix_lens[g]))
    rows_k = {}

    def keys_of(b, h):
        if b not in rows_k:
            first, prefix = table[b]
            n = int(cache_seqlens[b])
            lo = max(0, n - 1 - window_left) if window_left >= 0 else 0
            at = []
            for t in range(lo, n):
                j = t // page
                p = int(block_table[first if t < prefix else b, j]) \
                    if j < block_table.shape[1] else -1
                if 0 <= p < nb:
                    at.append((p, t % page))
            at = np.array(at, np.int64).reshape(-1, 2)
            rows_k[b] = (np.asarray(k_cache[at[:, 0], at[:, 1]], np.float64),
                         np.asarray(v_cache[at[:, 0], at[:, 1]], np.float64))
        k, v = rows_k[b]
        return k[:, h] * ks[h], v[:, h] * vs[h]

    return _attend_rows(q, hk, keys_of, scale, sinks)
