"""Performance cases of caches that hold a token in few bytes, and of the attention over them.

Kinds (``case["kind"]``):

    kv4_chunk      a 4-bit cache as a chunk of prompts meets it: ops.store_kvcache_mxfp4 of the
                   chunk's tokens, then ops.gather_kvcache_mxfp4 of the whole contexts, whose
                   keys and values the chunk's attention reads
    kv4_decode     ops.mxfp4_paged_decode: decode attention over the 4-bit cache
    latent_chunk   ops.latent_norm_rope_store of new tokens (latent norm, rotary of the shared
                   key and of the queries), and with ``gather`` ops.gather_latent of the whole
                   contexts, which the expanded form projects up
    latent_decode  ops.latent_decode: attention over the latent cache in the absorbed form

Where ``own`` is false, ``run`` computes the same in elementary torch operations in float32.
Sequence lengths are part of a case (drawn from ``len_seed`` between ``lo`` and ``hi``); the
values come from the seed given to ``prepare``.  ``rows`` is the most query rows a sequence
has: 1 is a plain decode step, more is a step that checks several drafted tokens, ragged.

The 4-bit format: a block is 32 dims of one token and kv head; its scale is 2^(E - 127), one
byte E, its values codes of {0, 0.5, 1, 1.5, 2, 3, 4, 6} with a sign.  K codes lie as
[page, head, token, D/2] (two dims a byte, the even one low), V codes as
[page, head, 4 tokens, 16, token, D/32], scales as [page, head, D/32, token].
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
_FP8 = torch.float8_e4m3fn
_R, _P = 512, 64  # dims of a latent row: the latent, and the key's rotary part
_EPS = 1e-6
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _kv4_chunk(batch, lo, hi, new, hk=8, d=128, page=16, len_seed=1):
    """lo .. hi: tokens of a sequence with its chunk; new: tokens of a chunk at most."""
    return dict(kind="kv4_chunk", batch=batch, lo=lo, hi=hi, new=new, hk=hk, d=d, page=page,
                len_seed=len_seed)


def _kv4_decode(batch, lo, hi, rows=1, hq=32, hk=8, d=128, page=16, sinks=False, window=-1,
                len_seed=1):
    return dict(kind="kv4_decode", batch=batch, lo=lo, hi=hi, rows=rows, hq=hq, hk=hk, d=d,
                page=page, sinks=sinks, window=window, len_seed=len_seed)


def _latent_chunk(batch, lo, hi, new, hq=16, page=64, kv="bf16", neox=False, gather=True,
                  len_seed=1):
    return dict(kind="latent_chunk", batch=batch, lo=lo, hi=hi, new=new, hq=hq, page=page, kv=kv,
                neox=neox, gather=gather, len_seed=len_seed)


def _latent_decode(batch, lo, hi, rows=1, hq=128, page=64, kv="bf16", len_seed=1):
    return dict(kind="latent_decode", batch=batch, lo=lo, hi=hi, rows=rows, hq=hq, page=page,
                kv=kv, len_seed=len_seed)


def listed():
    return [
        # The last few tokens of a short prompt.
        dict(_kv4_chunk(1, 117, 117, 17), name="kv4_chunk_b1"),
        # Chunks of four long prompts.
        dict(_kv4_chunk(4, 9000, 16384, 2048), name="kv4_chunk_b4"),
        # One user far into a long document.
        dict(_kv4_decode(1, 40000, 40000), name="kv4_b1"),
        # A full decode batch at the headline's shape.
        dict(_kv4_decode(64, 512, 8192), name="kv4_b64"),
        # Drafted tokens of 32 users, Llama-3-70B heads, pages of 64 tokens, sinks.
        dict(_kv4_decode(32, 2000, 16000, rows=4, hq=64, page=64, sinks=True),
             name="kv4_b32_drafts"),
        # Eight very long documents.
        dict(_kv4_decode(8, 16000, 65536, hq=64, page=256), name="kv4_b8_long"),
        # A decode step of 64 users, all heads on one device.
        dict(_latent_chunk(64, 64, 512, 1, hq=128, gather=False), name="latent_step_b64"),
        # Chunks of four prompts into an fp8 cache, read back for the expanded form.
        dict(_latent_chunk(4, 5000, 16384, 4096, kv="fp8"), name="latent_chunk_b4_fp8"),
        # One user far into a long document, 16 heads of one of eight devices.
        dict(_latent_decode(1, 40000, 40000, hq=16, page=16), name="latent_b1"),
        # A full decode batch, all 128 heads on one device.
        dict(_latent_decode(64, 512, 8192), name="latent_b64"),
        # Many users, 16 heads of one of eight devices, fp8 cache.
        dict(_latent_decode(128, 1000, 16384, hq=16, kv="fp8"), name="latent_b128_fp8"),
        # A step that checks up to four drafted tokens of 16 long sequences, all heads.
        dict(_latent_decode(16, 2000, 16384, rows=4), name="latent_b16_drafts"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, kv heads, head size) of the models whose decode the path serves.
_HEADS = [(32, 8, 128), (32, 8, 128), (64, 8, 128), (16, 2, 256), (20, 20, 64), (64, 8, 64),
          (8, 1, 128)]


def draw(rng):
    """One more case of the ranges above; sizes spread over their logarithm."""
    kind = rng.choice(["kv4_chunk", "kv4_decode", "kv4_decode", "latent_chunk", "latent_decode",
                       "latent_decode"])
    ls = rng.randrange(1 << 20)
    hq, hk, d = rng.choice(_HEADS)
    page = rng.choice([16, 16, 32, 64, 256])
    rows = rng.choice([1, 1, 2, 4, 5])
    low = rng.uniform(0.05, 1.0)
    if kind == "kv4_chunk":
        batch = _log_int(rng, 1, 64)
        # at most the tokens of kv4_chunk_b4
        hi = _log_int(rng, 16, max(17, 4 * 12000 * 1024 // (batch * hk * d)))
        return _kv4_chunk(batch, max(1, int(hi * low)), hi, min(hi, _log_int(rng, 1, 4096)),
                          hk=hk, d=d, page=page, len_seed=ls)
    if kind == "kv4_decode":
        batch = _log_int(rng, 1, 128)
        rows = max(1, min(rows, 128 // batch))
        # at most the keys of kv4_b64 per pass over them, and the pairs of kv4_b32_drafts
        cap = min(64 * 4096 * 1024 // (batch * hk * d), 32 * 4 * 9000 * 64 * 128 //
                  (batch * rows * hq * d))
        hi = _log_int(rng, 50, max(51, min(65536, cap)))
        return _kv4_decode(batch, max(1, int(hi * low)), hi, rows=rows, hq=hq, hk=hk, d=d,
                           page=page, sinks=rng.random() < 0.3,
                           window=_log_int(rng, 64, 4096) if rng.random() < 0.2 else -1,
                           len_seed=ls)
    kv = rng.choice(["bf16", "bf16", "fp8"])
    if kind == "latent_chunk":
        batch = _log_int(rng, 1, 128)
        hi = _log_int(rng, 16, max(17, 4 * 11000 // batch))
        hq = rng.choice([8, 16, 16, 32, 128])
        new = min(hi, _log_int(rng, 1, max(2, 4 * 4096 * 16 // (hq * batch))))
        return _latent_chunk(batch, max(1, int(hi * low)), hi, new, hq=hq, page=page, kv=kv,
                             neox=rng.random() < 0.3, len_seed=ls)
    batch = _log_int(rng, 1, 128)
    hq = rng.choice([8, 16, 16, 32, 64, 128, 20])
    rows = max(1, min(rows, 128 // batch))
    # at most the pairs of latent_b16_drafts, and the keys of latent_b64
    cap = min(16 * 9000 * 3 * 128 // (batch * rows * hq), 64 * 4096 // batch)
    hi = _log_int(rng, 50, max(51, min(65536, cap)))
    return _latent_decode(batch, max(1, int(hi * low)), hi, rows=rows, hq=hq, page=page, kv=kv,
                          len_seed=ls)


# ---------------------------------------------------------------------------
# Lengths and sizes
# ---------------------------------------------------------------------------
def _lens(case, n, lo, hi, salt=0):
    """n lengths in [lo, hi], the longest among them (a case costs what its bounds say)."""
    g = random.Random(case["len_seed"] * 7919 + salt)
    out = [g.randint(lo, hi) for _ in range(n)]
    out[g.randrange(n)] = hi
    return out


def _ctx(case):
    return _lens(case, case["batch"], case["lo"], case["hi"])


def _new(case):
    """Tokens that each sequence has just got: all but at most `new` were there before."""
    return [min(case["new"], c) for c in _ctx(case)]


def _q_lens(case):
    """Query rows per sequence: at most ``rows``, and at most its tokens."""
    n = _lens(case, case["batch"], 1, case["rows"], 1)
    return [min(a, c) for a, c in zip(n, _ctx(case))]


def _visible(case):
    """(sequence, first visible key, visible end) of every query row."""
    out, w = [], case.get("window", -1)
    for b, (c, n) in enumerate(zip(_ctx(case), _q_lens(case))):
        for i in range(n):
            end = c - n + i + 1
            out.append((b, max(0, end - 1 - w) if w >= 0 else 0, end))
    return out


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return _int32(cu)


def _tables(pages, seed):
    """Non-overlapping pages in random order, -1 padded; returns (tables, pool pages)."""
    pool = sum(pages) + 8
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    bt = torch.full((len(pages), max(pages)), -1, dtype=torch.int32)
    at = 0
    for i, p in enumerate(pages):
        bt[i, :p] = perm[at:at + p]
        at += p
    return bt, pool


def _paged(case, seed):
    lens, page = _ctx(case), case["page"]
    bt, pool = _tables([-(-n // page) for n in lens], seed)
    return dict(bt=bt.to(DEV), ctx=_int32(lens), page=page), pool


def _slots(case, bt):
    """Cache slots of the tokens that are new, in the sequences' order."""
    page, out = case["page"], []
    for b, (c, n) in enumerate(zip(_ctx(case), _new(case))):
        pos = torch.arange(c - n, c)
        out.append(bt[b].cpu()[pos // page].long() * page + pos % page)
    return torch.cat(out).to(DEV)


# ---------------------------------------------------------------------------
# The 4-bit format, in elementary operations
# ---------------------------------------------------------------------------
def _quantize(x):
    """x [.., D] float32 -> codes [.., D] (0 .. 15) and scale bytes [.., D/32]."""
    x = x.unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    # the exponent of the greatest value rounded to two significant bits, less that of 4
    e = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(0, 254)
    y = x * (254 - e << 23).view(torch.float32).unsqueeze(-1)
    a = y.abs()
    # to the nearest of the grid, ties to the even code
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + \
        (a >= 3.5) + (a > 5)
    code = code + 8 * torch.signbit(y)
    bad = ~torch.isfinite(top)
    code = torch.where(bad.unsqueeze(-1), 0, code)
    return code.flatten(-2).to(torch.uint8), torch.where(bad, 255, e).to(torch.uint8)


def _pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _dequantize(packed, scales):
    """packed [.., D/2] and scale bytes [.., D/32] -> float32 [.., D]."""
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), device=DEV)
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    e = scales.to(torch.int32)
    f = torch.where(e == 0, 0x400000, torch.where(e == 255, 0x7fc00000, e << 23))
    x = grid[codes.int()].unflatten(-1, (-1, 32)) * f.view(torch.float32).unsqueeze(-1)
    return x.flatten(-2)


def _v_rows(v):
    """V codes [pages, Hk, page/4, 16, 4, D/32] as rows [pages, Hk, page, D/2] (a copy)."""
    return v.permute(0, 1, 2, 4, 3, 5).flatten(4).flatten(2, 3)


def _kv4_cache(g, pool, page, hk, d):
    """Pages of N(0, 1) values with a bias per channel, as keys have: (codes, scales), in
    slices, so that a large pool needs no float32 copy.  Codes as rows of tokens."""
    out = torch.empty(pool, hk, page, d // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(pool, hk, d // 32, page, dtype=torch.uint8, device=DEV)
    bias = 0.5 * torch.randn(hk, 1, d, generator=g, device=DEV)
    step = max(1, (1 << 26) // (page * hk * d))
    for a in range(0, pool, step):
        x = torch.randn(min(step, pool - a), hk, page, d, generator=g, device=DEV) + bias
        codes, e = _quantize(x.to(torch.bfloat16).float())
        out[a:a + step], scales[a:a + step] = _pack(codes), e.transpose(2, 3)
    return out, scales


def _v_layout(rows):
    """The inverse of _v_rows."""
    pool, hk, page, half = rows.shape
    return rows.view(pool, hk, page // 4, 4, 16, half // 16).permute(0, 1, 2, 4, 3, 5).contiguous()


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def _prepare_kv4_chunk(case, seed):
    g = _gen(seed)
    s, pool = _paged(case, seed)
    hk, d = case["hk"], case["d"]
    s["k"], s["ks"] = _kv4_cache(g, pool, case["page"], hk, d)
    rows, s["vs"] = _kv4_cache(g, pool, case["page"], hk, d)
    s["v"] = _v_layout(rows)
    s["slots"] = _slots(case, s["bt"])
    n = s["slots"].numel()
    bias = 0.5 * torch.randn(hk, d, generator=g, device=DEV)
    s["key"] = (torch.randn(n, hk, d, generator=g, device=DEV) + bias).to(torch.bfloat16)
    s["value"] = _randn(g, n, hk, d)
    s["cu"], s["total"] = _cu(_ctx(case)), sum(_ctx(case))
    return s


def _prepare_kv4_decode(case, seed):
    g = _gen(seed)
    s, pool = _paged(case, seed)
    hk, d, n = case["hk"], case["d"], _q_lens(case)
    s["k"], s["ks"] = _kv4_cache(g, pool, case["page"], hk, d)
    rows, s["vs"] = _kv4_cache(g, pool, case["page"], hk, d)
    s["v"] = _v_layout(rows)
    s["q"] = _randn(g, sum(n), case["hq"], d)
    s["sinks"] = torch.randn(case["hq"], generator=g, device=DEV) if case["sinks"] else None
    s.update(cu=_cu(n) if max(n) > 1 else None, max_q=max(n), scale=d ** -0.5,
             window=case["window"])
    return s


def _latent_cache(g, pool, page, kv, scale):
    out = torch.empty(pool, page, _R + _P, dtype=_FP8 if kv == "fp8" else torch.bfloat16,
                      device=DEV)
    weight = 1.0 + 0.2 * torch.randn(_R + _P, generator=g, device=DEV)
    step = max(1, (1 << 26) // (page * (_R + _P)))
    for a in range(0, pool, step):
        x = torch.randn(min(step, pool - a), page, _R + _P, generator=g, device=DEV) * weight
        if kv == "fp8":
            x = (x / scale).clamp_(-448.0, 448.0)
        out[a:a + step] = x.to(out.dtype)
    return out


def _latent_scale(g, kv):
    return 0.01 + 0.03 * torch.rand(1, generator=g, device=DEV) if kv == "fp8" else None


def _prepare_latent_chunk(case, seed):
    g = _gen(seed)
    s, pool = _paged(case, seed)
    s["kscale"] = _latent_scale(g, case["kv"])
    s["cache"] = _latent_cache(g, pool, case["page"], case["kv"], s["kscale"])
    s["slots"] = _slots(case, s["bt"])
    n, hq = s["slots"].numel(), case["hq"]
    # the latent and the rotary key are one projection's output, the queries' rotary part the
    # tail of each head of another's
    down = 2.0 * _randn(g, n, _R + _P)
    s["latent"], s["key_rope"] = down[:, :_R], down[:, _R:]
    s["query_rope"] = _randn(g, n, hq, 128 + _P)[:, :, 128:]
    s["weight"] = (1.0 + 0.2 * torch.randn(_R, generator=g, device=DEV)).to(torch.bfloat16)
    s["pos"] = torch.cat([torch.arange(c - k, c) for c, k in zip(_ctx(case), _new(case))]).to(DEV)
    angles = torch.outer(torch.arange(max(_ctx(case)), dtype=torch.float64),
                         10000.0 ** -(torch.arange(0, _P, 2, dtype=torch.float64) / _P))
    s["cos_sin"] = torch.cat([angles.cos(), angles.sin()], -1).float().to(DEV)
    s["query"] = torch.zeros(n, hq, _R + _P, dtype=torch.bfloat16, device=DEV)
    s["cu"], s["total"] = _cu(_ctx(case)), sum(_ctx(case))
    s.update(neox=case["neox"], gather=case["gather"])
    return s


def _prepare_latent_decode(case, seed):
    g = _gen(seed)
    s, pool = _paged(case, seed)
    n = _q_lens(case)
    s["kscale"] = _latent_scale(g, case["kv"])
    s["cache"] = _latent_cache(g, pool, case["page"], case["kv"], s["kscale"])
    s["q"] = _randn(g, sum(n), case["hq"], _R + _P)
    s.update(cu=_cu(n) if max(n) > 1 else None, max_q=max(n), scale=(128 + _P) ** -0.5)
    return s


_PREPARE = {"kv4_chunk": _prepare_kv4_chunk, "kv4_decode": _prepare_kv4_decode,
            "latent_chunk": _prepare_latent_chunk, "latent_decode": _prepare_latent_decode}


def prepare(case, seed):
    return dict(_PREPARE[case["kind"]](case, seed), kind=case["kind"])


# ---------------------------------------------------------------------------
# run: the framework's operators
# ---------------------------------------------------------------------------
def _own(s):
    from fastkernels_amd import ops

    kind = s["kind"]
    if kind == "kv4_chunk":
        ops.store_kvcache_mxfp4(s["key"], s["value"], s["k"], s["v"], s["ks"], s["vs"],
                                s["slots"])
        key = s["key"].new_empty((s["total"], *s["key"].shape[1:]))
        value = torch.empty_like(key)
        ops.gather_kvcache_mxfp4(key, value, s["k"], s["v"], s["ks"], s["vs"], s["bt"], s["cu"])
        return key, value
    if kind == "kv4_decode":
        out = torch.empty_like(s["q"])
        ops.mxfp4_paged_decode(out, s["q"], s["k"], s["v"], s["ks"], s["vs"], s["bt"], s["ctx"],
                               s["scale"], window_left=s["window"], sinks=s["sinks"],
                               cu_seqlens_q=s["cu"], max_seqlen_q=s["max_q"])
        return out
    if kind == "latent_chunk":
        ops.latent_norm_rope_store(s["cache"], s["slots"], s["pos"], s["latent"], s["key_rope"],
                                   s["cos_sin"], s["neox"], weight=s["weight"], eps=_EPS,
                                   scale=s["kscale"], query_rope=s["query_rope"],
                                   query_out=s["query"][:, :, _R:])
        if not s["gather"]:
            return s["query"], s["cache"]
        rows = torch.empty(s["total"], _R + _P, dtype=torch.bfloat16, device=DEV)
        ops.gather_latent(rows, s["cache"], s["bt"], s["cu"], scale=s["kscale"])
        return s["query"], rows
    out = s["q"].new_empty((*s["q"].shape[:2], _R))
    ops.latent_decode(out, s["q"], s["cache"], s["bt"], s["ctx"], s["scale"], scale=s["kscale"],
                      cu_seqlens_q=s["cu"], max_seqlen_q=s["max_q"])
    return out


# ---------------------------------------------------------------------------
# run: the plain forms
# ---------------------------------------------------------------------------
def _row_info(s, n):
    """(sequence, visible end) of each query row, on the device."""
    ctx = s["ctx"].long()
    t = torch.arange(n, device=DEV)
    if s["cu"] is None:
        return t, ctx
    cu = s["cu"].long()
    seq = torch.bucketize(t, cu[1:], right=True)
    return seq, ctx[seq] - cu[seq + 1] + t + 1


def _places(s):
    """(page, token in it) of every token of the contexts, one sequence after another."""
    cu = s["cu"].long()
    t = torch.arange(s["total"], device=DEV)
    seq = torch.bucketize(t, cu[1:], right=True)
    pos = t - cu[seq]
    return s["bt"].long()[seq, pos // s["page"]], pos % s["page"]


def _softmax_rows(x, seen, v, sinks):
    """sum_j softmax(x)_j v_j over the keys that are seen; the sink joins the denominator."""
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    none = total == 0
    if sinks is not None:
        total = total + torch.exp(sinks - m)
    return torch.where(none, 0.0, (e @ v) / torch.where(none, 1.0, total))


def _plain_kv4_chunk(s):
    page, tok = s["slots"] // s["page"], s["slots"] % s["page"]
    for x, scales, v in ((s["key"], s["ks"], False), (s["value"], s["vs"], True)):
        codes, e = _quantize(x.float())
        packed = _pack(codes)
        scales.transpose(2, 3)[page, :, tok] = e
        if v:
            s["v"].permute(0, 2, 4, 1, 3, 5)[page, tok // 4, tok % 4] = \
                packed.unflatten(-1, (16, -1))
        else:
            s["k"][page, :, tok] = packed
    page, tok = _places(s)
    v = s["v"].permute(0, 2, 4, 1, 3, 5)[page, tok // 4, tok % 4].flatten(2)
    ks, vs = (x.transpose(2, 3)[page, :, tok] for x in (s["ks"], s["vs"]))
    return (_dequantize(s["k"][page, :, tok], ks).to(torch.bfloat16),
            _dequantize(v, vs).to(torch.bfloat16))


def _plain_kv4_decode(s):
    q, bt = s["q"].float(), s["bt"].long().clamp(min=0)
    n, hq, d = q.shape
    hk = s["k"].shape[1]
    b, width = bt.shape
    k, v = (_dequantize(c[bt], e[bt].transpose(3, 4)).transpose(1, 2).reshape(b, hk, -1, d)
            for c, e in ((s["k"], s["ks"]), (_v_rows(s["v"]), s["vs"])))
    seq, vis = _row_info(s, n)
    if s["cu"] is not None:
        k, v = k[seq], v[seq]
    x = (q.view(n, hk, hq // hk, d) @ k.transpose(-1, -2)) * s["scale"]
    at = torch.arange(width * s["page"], device=DEV)
    vis = vis.view(-1, 1, 1, 1)
    seen = at < vis
    if s["window"] >= 0:
        seen = seen & (at >= vis - 1 - s["window"])
    sinks = None if s["sinks"] is None else s["sinks"].view(1, hk, hq // hk, 1)
    return _softmax_rows(x, seen, v, sinks).view(n, hq, d).to(s["q"].dtype)


def _rotate(x, s):
    """x [n, heads, _P] rotated by the positions' angles."""
    cs = s["cos_sin"][s["pos"]].unsqueeze(1)
    c, n = cs[..., :_P // 2], cs[..., _P // 2:]
    if s["neox"]:
        a, b = x[..., :_P // 2], x[..., _P // 2:]
        return torch.cat([a * c - b * n, b * c + a * n], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)


def _plain_latent_chunk(s):
    x = s["latent"].float()
    c = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * s["weight"].float()
    row = torch.cat([c, _rotate(s["key_rope"].float().unsqueeze(1), s).squeeze(1)], -1)
    cache = s["cache"].view(-1, _R + _P)
    if s["kscale"] is None:
        cache[s["slots"]] = row.to(torch.bfloat16)
    else:
        row = (row / s["kscale"]).clamp(-448.0, 448.0).to(_FP8)
        cache.view(torch.uint8)[s["slots"]] = row.view(torch.uint8)
    s["query"][:, :, _R:] = _rotate(s["query_rope"].float(), s).to(torch.bfloat16)
    if not s["gather"]:
        return s["query"], s["cache"]
    page, tok = _places(s)
    return s["query"], _latent_rows(s, page * s["page"] + tok).to(torch.bfloat16)


def _latent_rows(s, slots):
    cache = s["cache"].view(-1, _R + _P)
    if s["kscale"] is None:
        return cache[slots].float()
    return cache.view(torch.uint8)[slots].view(_FP8).float() * s["kscale"]


def _plain_latent_decode(s):
    q, bt = s["q"].float(), s["bt"].long().clamp(min=0)
    page = s["page"]
    slots = (bt.unsqueeze(-1) * page + torch.arange(page, device=DEV)).flatten(1)
    k = _latent_rows(s, slots)
    seq, vis = _row_info(s, q.shape[0])
    if s["cu"] is not None:
        k = k[seq]
    x = (q @ k.transpose(-1, -2)) * s["scale"]
    seen = torch.arange(k.shape[1], device=DEV) < vis.view(-1, 1, 1)
    return _softmax_rows(x, seen, k[..., :_R], None).to(s["q"].dtype)


_PLAIN = {"kv4_chunk": _plain_kv4_chunk, "kv4_decode": _plain_kv4_decode,
          "latent_chunk": _plain_latent_chunk, "latent_decode": _plain_latent_decode}


def run(state):
    return _own(state) if own else _PLAIN[state["kind"]](state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def _keys_once(case):
    """Keys that at least one row of their sequence sees."""
    lo, hi = {}, {}
    for b, a, e in _visible(case):
        lo[b], hi[b] = min(lo.get(b, a), a), max(hi.get(b, e), e)
    return sum(hi[b] - lo[b] for b in hi)


def work(case):
    kind = case["kind"]
    if kind == "kv4_chunk":
        hd = case["hk"] * case["d"]
        new, total = sum(_new(case)), sum(_ctx(case))
        # new tokens in and their codes out; the contexts' codes in and their values out
        return {"bytes": int(2 * hd * (new + total) * (2 + 0.5 + 1 / 32)), "flops": 0.0}
    if kind == "latent_chunk":
        elt = 1 if case["kv"] == "fp8" else 2
        new, total = sum(_new(case)), sum(_ctx(case)) if case["gather"] else 0
        return {"bytes": (new + total) * (_R + _P) * (2 + elt) + 4 * new * case["hq"] * _P,
                "flops": 0.0}
    pairs = sum(e - a for _, a, e in _visible(case))
    rows = sum(_q_lens(case))
    if kind == "kv4_decode":
        hq, hk, d = case["hq"], case["hk"], case["d"]
        return {"bytes": 2 * _keys_once(case) * hk * (d // 2 + d // 32) + 4 * rows * hq * d,
                "flops": 4.0 * pairs * hq * d}
    elt = 1 if case["kv"] == "fp8" else 2
    return {"bytes": _keys_once(case) * (_R + _P) * elt + 2 * rows * case["hq"] * (2 * _R + _P),
            "flops": 2.0 * pairs * case["hq"] * (2 * _R + _P)}


# ---------------------------------------------------------------------------
# exact: the definitions, in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------
def _decode64(nibbles, e):
    """Values of codes [.., D] (two planes already apart) with exponents [.., D]."""
    m = (nibbles & 7).to(torch.float64)
    # 0 and 0.5 below the first normal, then (2 + m odd) / 2 2^(m / 2 - 1)
    a = torch.where(m < 2, m / 2, (2 + m % 2) / 2 * torch.exp2(torch.floor(m / 2) - 1))
    a = torch.where(nibbles >= 8, -a, a) * torch.exp2(e.to(torch.float64) - 127)
    return torch.where(e == 255, math.nan, a)


def _kv64(s, which, pages, n):
    """[n, Hk, D] values of a sequence's first n tokens from its pages."""
    e = s["ks" if which == "k" else "vs"][pages]
    if which == "k":
        rows = s["k"][pages]
    else:
        v = s["v"][pages]  # [pages, Hk, page/4, 16, 4, D/32]
        rows = torch.stack([v[:, :, i // 4, :, i % 4].flatten(2) for i in range(s["page"])], 2)
    out = torch.empty(*rows.shape[:3], 2 * rows.shape[3], dtype=torch.float64, device=DEV)
    e = e.transpose(2, 3).repeat_interleave(32, -1)
    out[..., 0::2] = _decode64(rows % 16, e[..., 0::2])
    out[..., 1::2] = _decode64(rows // 16, e[..., 1::2])
    return out.transpose(1, 2).flatten(0, 1)[:n]


def _round64(x):
    """What the 4-bit format holds of x [n, Hk, D], by the definition: of each block of 32 the
    nearest multiples of its power of two, ties to the even code."""
    grid = torch.tensor(_GRID, dtype=torch.float64, device=DEV)
    b = x.to(torch.float64).unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    low = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    low = low + (top / torch.exp2(low) >= 1.75)
    scale = torch.exp2((low - 2).clamp(min=-127))
    y = b / scale
    lo = (torch.bucketize(y.abs(), grid, right=True) - 1).clamp(max=6)
    a, c = y.abs() - grid[lo], grid[lo + 1] - y.abs()
    code = lo + ((a > c) | ((a == c) & (lo % 2 == 1)))
    return (torch.copysign(grid[code], y) * scale).flatten(-2)


def _turn64(x, pos, neox):
    """x [n, heads, _P] rotated by pos times the frequencies."""
    f = 10000.0 ** -(torch.arange(0, _P, 2, dtype=torch.float64, device=DEV) / _P)
    z = torch.polar(torch.ones_like(f), pos.to(torch.float64).view(-1, 1, 1) * f)
    x = x.to(torch.float64)
    if neox:
        y = torch.complex(x[..., :_P // 2], x[..., _P // 2:]) * z
        return torch.cat([y.real, y.imag], -1)
    y = torch.complex(x[..., 0::2], x[..., 1::2]) * z
    return torch.view_as_real(y).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    kind, page, ctx = case["kind"], case["page"], _ctx(case)
    bt = s["bt"].long()
    pages = [bt[b, :-(-c // page)] for b, c in enumerate(ctx)]
    if kind == "kv4_chunk":
        keys, values, at = [], [], 0
        new = _round64(s["key"]), _round64(s["value"])
        for b, (c, n) in enumerate(zip(ctx, _new(case))):
            for out, which, x in ((keys, "k", new[0]), (values, "v", new[1])):
                out.append(torch.cat([_kv64(s, which, pages[b], c)[:c - n], x[at:at + n]]))
            at += n
        return torch.cat(keys), torch.cat(values)
    scale64 = None if s.get("kscale") is None else s["kscale"].to(torch.float64)
    if kind == "latent_chunk":
        x = s["latent"].to(torch.float64)
        c = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + _EPS) * s["weight"].to(torch.float64)
        k = _turn64(s["key_rope"].unsqueeze(1), s["pos"], case["neox"]).squeeze(1)
        row = torch.cat([c, k], -1)
        query = s["query"].to(torch.float64)
        query[:, :, _R:] = _turn64(s["query_rope"], s["pos"], case["neox"])
        if not case["gather"]:
            cache = s["cache"].to(torch.float64)
            cache.view(-1, _R + _P)[s["slots"]] = row
            return query, cache
        if scale64 is not None:
            # the codes are the nearest e4m3 values of what is stored
            row = (row / scale64).clamp(-448, 448).float().to(_FP8).to(torch.float64) * scale64
        rows, at = [], 0
        for b, (c, n) in enumerate(zip(ctx, _new(case))):
            old = s["cache"].view(torch.uint8)[pages[b]].view(s["cache"].dtype).to(torch.float64)
            old = old.flatten(0, 1)[:c - n]
            rows.append(torch.cat([old if scale64 is None else old * scale64, row[at:at + n]]))
            at += n
        return query, torch.cat(rows)
    q, seen = s["q"].to(torch.float64), _visible(case)
    hq, out, t = case["hq"], [], 0
    for b, c in enumerate(ctx):
        if kind == "kv4_decode":
            k, v = _kv64(s, "k", pages[b], c), _kv64(s, "v", pages[b], c)
            k, v = k.permute(1, 2, 0), v.transpose(0, 1)
        else:
            k = s["cache"].view(torch.uint8)[pages[b]].view(s["cache"].dtype)
            k = k.to(torch.float64).flatten(0, 1)[:c]
            k = k if scale64 is None else k * scale64
            k, v = k.T.unsqueeze(0), k[:, :_R].unsqueeze(0)
        while t < len(seen) and seen[t][0] == b:
            _, lo, hi = seen[t]
            x = (q[t].view(k.shape[0], -1, k.shape[1]) @ k[:, :, lo:hi]) * s["scale"]
            logs = x
            if s.get("sinks") is not None:
                extra = s["sinks"].to(torch.float64).view(*x.shape[:2], 1)
                logs = torch.cat([x, extra], -1)
            w = torch.exp(x - torch.logsumexp(logs, -1, keepdim=True))
            out.append((w @ v[:, lo:hi]).reshape(hq, -1))
            t += 1
    return torch.stack(out)
