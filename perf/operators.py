"""Performance cases of the attention operators that read less than the whole paged cache.

Kinds (``case["kind"]``), one operator each:

    bounds   ops.update_key_bounds: the per-page minimum and maximum of the keys, kept beside
             the cache as tokens arrive (a decode step, or the chunks of prompts)
    scores   ops.block_scores: every page's upper bound of q . k per query row and kv head
    select   ops.select_blocks: the pages a row attends to, from their scores
    sparse   ops.sparse_paged_decode: attention over the selected pages
    prefix   ops.shared_prefix_decode: decode attention of a batch in groups that share a long
             prefix, each prefix read once for its group

Where ``own`` is false, ``run`` computes the same in elementary torch operations in float32.
Sequence lengths are part of a case (drawn from ``len_seed`` between ``lo`` and ``hi``); the
values come from the seed given to ``prepare``.  ``rows`` is the most query rows a sequence
has: 1 is a plain decode step, more is a step that checks several drafted tokens, ragged.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
_FP8 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _bounds(batch, lo, hi, new, hk=8, d=128, page=16, kv="bf16", len_seed=1):
    """new: tokens each sequence has just stored (0: all of them, whole prompts)."""
    return dict(kind="bounds", batch=batch, lo=lo, hi=hi, new=new, hk=hk, d=d, page=page, kv=kv,
                len_seed=len_seed)


def _scores(batch, lo, hi, rows=1, hq=32, hk=8, d=128, page=16, kv="bf16", len_seed=1):
    return dict(kind="scores", batch=batch, lo=lo, hi=hi, rows=rows, hq=hq, hk=hk, d=d, page=page,
                kv=kv, len_seed=len_seed)


def _select(batch, lo, hi, keep, rows=1, hk=8, page=16, first=1, last=4, len_seed=1):
    return dict(kind="select", batch=batch, lo=lo, hi=hi, keep=keep, rows=rows, hk=hk, page=page,
                first=first, last=last, len_seed=len_seed)


def _sparse(batch, lo, hi, keep, rows=1, hq=32, hk=8, d=128, page=16, kv="bf16", sinks=False,
            len_seed=1):
    return dict(kind="sparse", batch=batch, lo=lo, hi=hi, keep=keep, rows=rows, hq=hq, hk=hk, d=d,
                page=page, kv=kv, sinks=sinks, len_seed=len_seed)


def _prefix(batch, groups, plo, phi, lo, hi, hq=32, hk=8, d=128, page=16, kv="bf16", sinks=False,
            len_seed=1):
    """lo .. hi: the tokens a sequence has of its own, behind its group's prefix."""
    return dict(kind="prefix", batch=batch, groups=groups, plo=plo, phi=phi, lo=lo, hi=hi, hq=hq,
                hk=hk, d=d, page=page, kv=kv, sinks=sinks, len_seed=len_seed)


def listed():
    return [
        # A decode step of 64 users: one new token each, the smallest calls.
        dict(_bounds(64, 512, 8192, 1), name="bounds_step_b64"),
        # Four prompts that have just been stored, on fp8 pages of 64 tokens.
        dict(_bounds(4, 1000, 8192, 0, page=64, kv="fp8"), name="bounds_prompts_fp8"),
        # One user far into a long document.
        dict(_scores(1, 40000, 40000), name="scores_b1"),
        # Long documents of many users: the most pages to score.
        dict(_scores(32, 16000, 131072), name="scores_b32_long"),
        # The same single user: a few rows, latency.
        dict(_select(1, 40000, 40000, 128), name="select_b1"),
        # A step that checks up to four drafted tokens of each of 32 long documents.
        dict(_select(32, 16000, 131072, 128, rows=4), name="select_b32_drafts"),
        # One user's attention over 2048 selected tokens.
        dict(_sparse(1, 40000, 40000, 128), name="sparse_b1"),
        # A full decode batch, 2048 selected tokens each.
        dict(_sparse(64, 1500, 65536, 128), name="sparse_b64"),
        # Drafted tokens on fp8 pages of 64 tokens, Llama-3-70B heads.
        dict(_sparse(32, 8000, 65536, 32, rows=4, hq=64, page=64, kv="fp8"),
             name="sparse_b32_drafts_fp8"),
        # A small batch behind one system prompt.
        dict(_prefix(8, 1, 1500, 1500, 30, 400), name="prefix_b8"),
        # A full batch over one long shared document, the Qwen3-8B heads of the headline.
        dict(_prefix(64, 1, 8192, 8192, 100, 2000), name="prefix_b64"),
        # Three documents shared among 128 users, fp8 pages, Llama-3-70B heads.
        dict(_prefix(128, 3, 4096, 16384, 200, 1000, hq=64, kv="fp8"), name="prefix_b128_fp8"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, kv heads, head size) of the models whose decode the path serves.
_HEADS = [(32, 8, 128), (32, 8, 128), (64, 8, 128), (16, 2, 256), (20, 20, 64), (64, 8, 64),
          (8, 1, 128)]


def draw(rng):
    """One more case of the ranges above; sizes spread over their logarithm."""
    kind = rng.choice(["bounds", "scores", "select", "sparse", "sparse", "prefix", "prefix"])
    ls = rng.randrange(1 << 20)
    hq, hk, d = rng.choice(_HEADS)
    page = rng.choice([16, 16, 32, 64, 256])
    kv = rng.choice(["bf16", "bf16", "fp8"])
    elt = 1 if kv == "fp8" else 2
    if kind == "bounds":
        step = rng.random() < 0.5
        batch = _log_int(rng, 1, 160 if step else 8)
        hi = _log_int(rng, 16, 8192)
        new = rng.choice([1, 1, 5, 64]) if step else 0
        return _bounds(batch, max(1, int(hi * rng.uniform(0.1, 1.0))), hi, min(new, hi), hk=hk,
                       d=d, page=page, kv="bf16" if step else kv, len_seed=ls)
    rows = rng.choice([1, 1, 2, 4, 5])
    if kind == "scores":
        batch = _log_int(rng, 1, 64)
        # at most the bytes of scores_b32_long, at most its rows and its length
        rows = max(1, min(rows, 32 // batch))
        cap = int(32 * 65536 * 2048 / 16 / (hk * d * elt * batch) * page)
        hi = _log_int(rng, 100, max(101, min(131072, cap)))
        return _scores(batch, max(1, int(hi * rng.uniform(0.1, 1.0))), hi, rows=rows, hq=hq, hk=hk,
                       d=d, page=page, kv=kv, len_seed=ls)
    if kind == "select":
        batch = _log_int(rng, 1, 64)
        rows = max(1, min(rows, 128 // batch))
        hi = _log_int(rng, 100, max(101, min(131072, (1 << 26) // (hk * rows * batch) * page)))
        keep = rng.choice([16, 37, 64, 128, 250])
        first, last = rng.choice([(0, 1), (1, 4), (2, 8)])
        return _select(batch, max(1, int(hi * rng.uniform(0.05, 1.0))), hi, keep, rows=rows, hk=hk,
                       page=page, first=first, last=last, len_seed=ls)
    if kind == "sparse":
        batch = _log_int(rng, 1, 128)
        rows = max(1, min(rows, 128 // batch))
        # at most the keys of sparse_b64, or the pairs of rows and keys of sparse_b32_drafts_fp8
        cap = (128 * 2048 * 1024) // (rows * batch * hk * d * elt)
        keep = max(1, min(_log_int(rng, 128, 8192), cap) // page)
        hi = _log_int(rng, 100, min(65536, max(101, (1 << 33) // (batch * hk * d * 4))))
        return _sparse(batch, max(1, int(hi * rng.uniform(0.05, 1.0))), hi, keep, rows=rows, hq=hq,
                       hk=hk, d=d, page=page, kv=kv, sinks=rng.random() < 0.3, len_seed=ls)
    batch = _log_int(rng, 2, 128)
    groups = rng.choice([1, 1, 2, 5])
    # at most half of the pairs of prefix_b128_fp8, and own keys of at most prefix_b64's bytes
    cap = (128 * 16384 * 512) // (batch * max(hk * d, hq * d // 8))
    phi = _log_int(rng, 200, max(201, min(32768, cap)))
    hi = _log_int(rng, 10, max(11, min(4096, cap, (1 << 27) // (batch * hk * d * elt))))
    return _prefix(batch, min(groups, batch), max(1, int(phi * rng.uniform(0.2, 1.0))), phi,
                   max(1, int(hi * rng.uniform(0.05, 1.0))), hi, hq=hq, hk=hk, d=d, page=page,
                   kv=kv, sinks=rng.random() < 0.3, len_seed=ls)


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


def _q_lens(case):
    """Query rows per sequence: at most ``rows``, and at most its tokens."""
    n = _lens(case, case["batch"], 1, case["rows"], 1)
    return [min(a, c) for a, c in zip(n, _ctx(case))]


def _visible(case):
    """(sequence, visible keys) of every query row."""
    out = []
    for b, (c, n) in enumerate(zip(_ctx(case), _q_lens(case))):
        out += [(b, c - n + i + 1) for i in range(n)]
    return out


def _groups(case):
    """(first rows of the groups, prefix tokens per group, own tokens per sequence); the
    prefixes are whole pages, as a prefix cache shares them."""
    b, n = case["batch"], case["groups"]
    cuts = sorted(random.Random(case["len_seed"]).sample(range(1, b), n - 1))
    page = case["page"]
    pre = [p // page * page for p in _lens(case, n, case["plo"], case["phi"], 3)]
    return [0, *cuts, b], pre, _lens(case, b, case["lo"], case["hi"], 4)


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


def _cache(g, pool, page, hk, d, kv, scale=None):
    """Pages of N(0, 1) values with a bias per channel, as keys have; fp8: codes of
    x / scale[kv head], saturated.  In slices, so that a large pool needs no float32 copy."""
    out = torch.empty(pool, page, hk, d, dtype=_FP8 if kv == "fp8" else torch.bfloat16, device=DEV)
    bias = 0.5 * torch.randn(hk, d, generator=g, device=DEV)
    step = max(1, (1 << 26) // (page * hk * d))
    for a in range(0, pool, step):
        x = torch.randn(min(step, pool - a), page, hk, d, generator=g, device=DEV) + bias
        if scale is not None:
            x = x / scale.view(1, 1, -1, 1)
        out[a:a + step] = x.clamp_(-448.0, 448.0).to(out.dtype) if kv == "fp8" else x.to(out.dtype)
    return out


def _scale(g, hk, kv):
    return 0.01 + 0.09 * torch.rand(hk, generator=g, device=DEV) if kv == "fp8" else None


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def _prepare_bounds(case, seed):
    g = _gen(seed)
    lens, page = _ctx(case), case["page"]
    bt, pool = _tables([-(-n // page) for n in lens], seed)
    k = _cache(g, pool, page, case["hk"], case["d"], case["kv"],
               0.05 * torch.ones(case["hk"], device=DEV) if case["kv"] == "fp8" else None)
    new = [min(case["new"] or n, n) for n in lens]
    s = dict(k=k, bt=bt.to(DEV), ctx=_int32(lens), max_new=max(new),
             cu=_cu(new) if max(new) > 1 else None)
    s["bounds"] = torch.zeros(pool, case["hk"], 2, case["d"], dtype=k.dtype, device=DEV)
    return s


def _rows_state(case, seed, ctx):
    n = _q_lens(case)
    return dict(ctx=_int32(ctx), cu=_cu(n) if max(n) > 1 else None, max_q=max(n), n=sum(n))


def _prepare_scores(case, seed):
    g = _gen(seed)
    lens, page = _ctx(case), case["page"]
    s = _rows_state(case, seed, lens)
    bt, pool = _tables([-(-n // page) for n in lens], seed)
    hk, d = case["hk"], case["d"]
    s["ks"] = _scale(g, hk, case["kv"])
    # two keys per page stand for its least and its greatest values
    pair = _cache(g, pool, 2, hk, d, case["kv"], s["ks"]).transpose(1, 2)
    s["bounds"] = torch.empty(pool, hk, 2, d, dtype=pair.dtype, device=DEV)
    step = max(1, (1 << 26) // (2 * hk * d))
    for a in range(0, pool, step):
        s["bounds"][a:a + step] = pair[a:a + step].float().sort(dim=2).values.to(pair.dtype)
    s["bt"], s["page"] = bt.to(DEV), page
    s["q"] = _randn(g, s["n"], case["hq"], d)
    return s


def _prepare_select(case, seed):
    g = _gen(seed)
    lens, page = _ctx(case), case["page"]
    s = _rows_state(case, seed, lens)
    width = -(-max(lens) // page)
    x = 10.0 * torch.randn(s["n"], case["hk"], width, generator=g, device=DEV)
    # pages of equal content score alike: one row in three is on a coarse grid, with many ties
    coarse = torch.arange(s["n"], device=DEV).view(-1, 1, 1) % 3 == 0
    s["scores"] = torch.where(coarse, (4 * x).round() / 4, x)
    s.update(keep=case["keep"], first=case["first"], last=case["last"], page=page)
    return s


def _prepare_sparse(case, seed):
    g = _gen(seed)
    lens, page, hk, d = _ctx(case), case["page"], case["hk"], case["d"]
    s = _rows_state(case, seed, lens)
    bt, pool = _tables([-(-n // page) for n in lens], seed)
    s["ks"], s["vs"] = _scale(g, hk, case["kv"]), _scale(g, hk, case["kv"])
    s["k"] = _cache(g, pool, page, hk, d, case["kv"], s["ks"])
    s["v"] = _cache(g, pool, page, hk, d, case["kv"], s["vs"])
    s["bt"] = bt.to(DEV)
    s["q"] = _randn(g, s["n"], case["hq"], d)
    s["sinks"] = torch.randn(case["hq"], generator=g, device=DEV) if case["sinks"] else None
    s["scale"] = d ** -0.5
    # Pages as scores select them: the first, the last, and the best of random scores, which
    # the rows of one sequence mostly share.
    vis = _visible(case)
    seq = torch.tensor([b for b, _ in vis], device=DEV)
    nblk = torch.tensor([-(-v // page) for _, v in vis], device=DEV).view(-1, 1, 1)
    at = torch.arange(bt.shape[1], device=DEV)
    x = torch.rand(case["batch"], hk, bt.shape[1], generator=g, device=DEV)[seq]
    x = x + 0.02 * torch.rand(x.shape, generator=g, device=DEV)
    x = torch.where((at < 1) | (at == nblk - 1), 2.0, torch.where(at < nblk, x, -1.0))
    keep = min(case["keep"], bt.shape[1])
    top = x.topk(keep, dim=2)
    idx = torch.where(top.values >= 0, top.indices, 1 << 30).sort(dim=2).values
    s["idx"] = torch.where(idx < 1 << 30, idx, -1).to(torch.int32).contiguous()
    return s


def _prepare_prefix(case, seed):
    g = _gen(seed)
    cu, pre, tail = _groups(case)
    page, hk, d = case["page"], case["hk"], case["d"]
    of = [next(i for i in range(len(pre)) if b < cu[i + 1]) for b in range(case["batch"])]
    ctx = [pre[of[b]] + t for b, t in enumerate(tail)]
    own_pages = [-(-c // page) - pre[of[b]] // page for b, c in enumerate(ctx)]
    pages, pool = _tables([p // page for p in pre] + own_pages, seed)
    bt = torch.full((len(ctx), -(-max(ctx) // page)), -1, dtype=torch.int32)
    for b, n in enumerate(own_pages):
        p = pre[of[b]] // page
        bt[b, :p] = pages[of[b], :p]
        bt[b, p:p + n] = pages[len(pre) + b, :n]
    s = dict(ks=_scale(g, hk, case["kv"]), vs=_scale(g, hk, case["kv"]))
    s["k"] = _cache(g, pool, page, hk, d, case["kv"], s["ks"])
    s["v"] = _cache(g, pool, page, hk, d, case["kv"], s["vs"])
    s["q"] = _randn(g, len(ctx), case["hq"], d)
    s["sinks"] = torch.randn(case["hq"], generator=g, device=DEV) if case["sinks"] else None
    s.update(bt=bt.to(DEV), ctx=_int32(ctx), cu=_int32(cu), pre=_int32(pre), scale=d ** -0.5,
             max_prefix=max(pre))
    return s


_PREPARE = {"bounds": _prepare_bounds, "scores": _prepare_scores, "select": _prepare_select,
            "sparse": _prepare_sparse, "prefix": _prepare_prefix}


def prepare(case, seed):
    return dict(_PREPARE[case["kind"]](case, seed), kind=case["kind"])


# ---------------------------------------------------------------------------
# run: the framework's operators
# ---------------------------------------------------------------------------
def _own(s):
    from fastkernels_amd import ops

    kind = s["kind"]
    if kind == "bounds":
        ops.update_key_bounds(s["bounds"], s["k"], s["bt"], s["ctx"], cu_seqlens_q=s["cu"],
                              max_seqlen_q=s["max_new"])
        return _values(s["bounds"])
    if kind == "scores":
        out = torch.empty(s["n"], s["bounds"].shape[1], s["bt"].shape[1], device=DEV)
        ops.block_scores(out, s["q"], s["bounds"], s["bt"], s["ctx"], s["page"], k_scale=s["ks"],
                         cu_seqlens_q=s["cu"], max_seqlen_q=s["max_q"])
        return out
    if kind == "select":
        n, hk, _ = s["scores"].shape
        out = torch.empty(n, hk, s["keep"], dtype=torch.int32, device=DEV)
        ops.select_blocks(out, s["scores"], s["ctx"], s["page"], keep_first=s["first"],
                          keep_last=s["last"], cu_seqlens_q=s["cu"])
        return out
    out = torch.empty_like(s["q"])
    if kind == "sparse":
        ops.sparse_paged_decode(out, s["q"], s["k"], s["v"], s["bt"], s["ctx"], s["idx"],
                                s["scale"], k_scale=s["ks"], v_scale=s["vs"], sinks=s["sinks"],
                                cu_seqlens_q=s["cu"])
    else:
        ops.shared_prefix_decode(out, s["q"], s["k"], s["v"], s["bt"], s["ctx"], s["cu"],
                                 s["pre"], s["scale"], k_scale=s["ks"], v_scale=s["vs"],
                                 sinks=s["sinks"], max_prefix_len=s["max_prefix"])
    return out


# ---------------------------------------------------------------------------
# run: the plain forms
# ---------------------------------------------------------------------------
def _values(t):
    """fp8 codes as the values they stand for."""
    return t.float() if t.dtype == _FP8 else t


def _take(t, at):
    """t[at] along the first dimensions, also of fp8 pages, as float32."""
    if t.dtype == _FP8:
        return t.view(torch.uint8)[at].view(_FP8).float()
    return t[at].float()


def _row_info(s, n):
    """(sequence, visible keys) of each query row, on the device."""
    ctx = s["ctx"].long()
    t = torch.arange(n, device=DEV)
    if s["cu"] is None:
        return t, ctx
    cu = s["cu"].long()
    seq = torch.bucketize(t, cu[1:], right=True)
    return seq, ctx[seq] - cu[seq + 1] + t + 1


def _plain_bounds(s):
    k, bt, ctx, page = s["k"], s["bt"].long(), s["ctx"].long(), s["k"].shape[1]
    new = torch.ones_like(ctx) if s["cu"] is None else (s["cu"][1:] - s["cu"][:-1]).long()
    first = (ctx - new).clamp(min=0) // page
    most = (s["max_new"] + page - 2) // page + 1
    at = first[:, None] + torch.arange(most, device=DEV)
    ok = at * page < ctx[:, None]
    p = torch.where(ok, bt.gather(1, at.clamp(max=bt.shape[1] - 1)), -1)
    x = _take(k, p.clamp(min=0))  # [B, pages, page, Hk, D]
    pos = at[:, :, None] * page + torch.arange(page, device=DEV)
    seen = (pos < ctx[:, None, None])[..., None, None]
    lo = torch.where(seen, x, math.inf).amin(2)
    hi = torch.where(seen, x, -math.inf).amax(2)
    both = torch.stack([lo, hi], dim=3).to(k.dtype)
    s["bounds"].view(torch.uint8)[p[ok]] = both[ok].view(torch.uint8)
    return _values(s["bounds"])


def _plain_scores(s):
    q, bounds, bt = s["q"].float(), s["bounds"], s["bt"].long()
    n, hq, d = q.shape
    hk = bounds.shape[1]
    seq, vis = _row_info(s, n)
    p = bt[seq]
    b = _take(bounds, p.clamp(min=0)).permute(0, 2, 3, 4, 1)  # [N, Hk, 2, D, S]
    q = q.view(n, hk, hq // hk, d)
    x = (q.clamp(min=0) @ b[:, :, 1] + q.clamp(max=0) @ b[:, :, 0]).amax(2)
    if s["ks"] is not None:
        x = x * s["ks"].view(1, -1, 1)
    at = torch.arange(bt.shape[1], device=DEV)
    seen = (p >= 0) & (at * s["page"] < vis[:, None])
    return torch.where(seen[:, None], x, -math.inf)


def _plain_select(s):
    x, keep, page = s["scores"], s["keep"], s["page"]
    n, hk, width = x.shape
    _, vis = _row_info(s, n)
    nblk = ((vis + page - 1) // page).clamp(0, width).view(-1, 1, 1)
    at = torch.arange(width, device=DEV).expand(n, hk, width)
    # by three keys, the least first, stably: the score, what is always kept, what is visible
    order = x.sort(dim=2, descending=True, stable=True).indices
    for mark in ((at < s["first"]) | (at >= nblk - s["last"]), at < nblk):
        k = mark.gather(2, order).to(torch.uint8).sort(dim=2, descending=True, stable=True)
        order = order.gather(2, k.indices)
    top = order[:, :, :keep]
    top = torch.where(top < nblk, top, width).sort(dim=2).values
    out = torch.full((n, hk, keep), -1, dtype=torch.int32, device=DEV)
    out[:, :, :top.shape[2]] = torch.where(top < width, top, -1).to(torch.int32)
    return out


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


def _scaled(x, scale):
    """x [.., Hk, keys, D] times the scale of its kv head."""
    return x if scale is None else x * scale.view(-1, 1, 1)


def _plain_sparse(s):
    q, idx, bt = s["q"].float(), s["idx"].long(), s["bt"].long()
    n, hq, d = q.shape
    _, page, hk, _ = s["k"].shape
    seq, vis = _row_info(s, n)
    p = torch.where(idx >= 0, bt[seq[:, None, None], idx.clamp(min=0)], -1)
    head = torch.arange(hk, device=DEV).view(1, -1, 1)
    keys = [_take(c.transpose(1, 2), (p.clamp(min=0), head)).reshape(n, hk, -1, d)
            for c in (s["k"], s["v"])]
    k, v = _scaled(keys[0], s["ks"]), _scaled(keys[1], s["vs"])
    pos = idx[..., None] * page + torch.arange(page, device=DEV)
    seen = ((p >= 0)[..., None] & (pos < vis.view(-1, 1, 1, 1))).reshape(n, hk, 1, -1)
    x = (q.view(n, hk, hq // hk, d) @ k.transpose(-1, -2)) * s["scale"]
    sinks = None if s["sinks"] is None else s["sinks"].view(1, hk, hq // hk, 1)
    return _softmax_rows(x, seen, v, sinks).view(n, hq, d).to(s["q"].dtype)


def _plain_prefix(s):
    q, bt = s["q"].float(), s["bt"].long()
    n, hq, d = q.shape
    _, page, hk, _ = s["k"].shape
    k, v = (_take(c, bt.clamp(min=0)).reshape(n, -1, hk, d).transpose(1, 2)
            for c in (s["k"], s["v"]))
    k, v = _scaled(k, s["ks"]), _scaled(v, s["vs"])
    seen = torch.arange(bt.shape[1] * page, device=DEV) < s["ctx"].view(-1, 1, 1, 1)
    x = (q.view(n, hk, hq // hk, d) @ k.transpose(-1, -2)) * s["scale"]
    sinks = None if s["sinks"] is None else s["sinks"].view(1, hk, hq // hk, 1)
    return _softmax_rows(x, seen, v, sinks).view(n, hq, d).to(s["q"].dtype)


_PLAIN = {"bounds": _plain_bounds, "scores": _plain_scores, "select": _plain_select,
          "sparse": _plain_sparse, "prefix": _plain_prefix}


def run(state):
    return _own(state) if own else _PLAIN[state["kind"]](state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    kind, page = case["kind"], case["page"]
    elt = 1 if case.get("kv") == "fp8" else 2
    hk = case["hk"]
    if kind == "bounds":
        rows = pages = 0
        for n in _ctx(case):
            first = (n - min(case["new"] or n, n)) // page
            rows += n - first * page
            pages += -(-n // page) - first
        return {"bytes": (rows + 2 * pages) * hk * case["d"] * elt, "flops": 0.0}
    if kind == "scores":
        pages = sum(-(-n // page) for n in _ctx(case))
        vis = [-(-v // page) for _, v in _visible(case)]
        d = case["d"]
        return {"bytes": 2 * pages * hk * d * elt + 4 * hk * len(vis) * max(vis) +
                2 * len(vis) * case["hq"] * d, "flops": 4.0 * case["hq"] * d * sum(vis)}
    if kind == "select":
        vis = [-(-v // page) for _, v in _visible(case)]
        return {"bytes": 4 * hk * (sum(vis) + len(vis) * case["keep"]), "flops": 0.0}
    hq, d = case["hq"], case["d"]
    if kind == "sparse":
        vis = _visible(case)
        keys = [min(v, case["keep"] * page) for _, v in vis]
        # the rows of a sequence mostly share their pages: once per sequence at the least
        once = {}
        for (b, _), n in zip(vis, keys):
            once[b] = max(once.get(b, 0), n)
        return {"bytes": 2 * sum(once.values()) * hk * d * elt + 4 * len(vis) * hq * d +
                4 * hk * len(vis) * case["keep"], "flops": 4.0 * hq * d * sum(keys)}
    cu, pre, tail = _groups(case)
    per = [p for i, p in enumerate(pre) for _ in range(cu[i], cu[i + 1])]
    return {"bytes": 2 * (sum(pre) + sum(tail)) * hk * d * elt + 4 * len(tail) * hq * d,
            "flops": 4.0 * hq * d * (sum(per) + sum(tail))}


# ---------------------------------------------------------------------------
# exact: the definitions, in 64 bits, one sequence or row at a time
# ---------------------------------------------------------------------------
def _f64(t, at):
    """t[at] for a list of page numbers (or one index) as float64."""
    return (t.view(torch.uint8)[at].view(_FP8) if t.dtype == _FP8 else t[at]).to(torch.float64)


def _attend64(q, k, v, scale, sinks):
    """q [Hk, G, D], k and v [keys, Hk, D], sinks [Hk, G] or None."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    x = scale * torch.einsum("hgd,thd->hgt", q, k)
    logs = x if sinks is None else torch.cat([x, sinks[..., None].expand(*x.shape[:2], 1)], -1)
    w = torch.exp(x - torch.logsumexp(logs, -1, keepdim=True))
    return torch.einsum("hgt,thd->hgd", w, v)


def exact(case, seed):
    s = prepare(case, seed)
    kind, page = case["kind"], case["page"]
    bt = s["bt"].tolist() if "bt" in s else None
    hk = case["hk"]
    if kind == "bounds":
        out = torch.zeros(s["bounds"].shape, dtype=torch.float64, device=DEV)
        for b, n in enumerate(_ctx(case)):
            for j in range((n - min(case["new"] or n, n)) // page, -(-n // page)):
                x = _f64(s["k"], bt[b][j])[:n - j * page]
                out[bt[b][j], :, 0], out[bt[b][j], :, 1] = x.min(0).values, x.max(0).values
        return out
    vis = None if kind == "prefix" else _visible(case)
    if kind == "select":
        out = torch.full((s["n"], hk, s["keep"]), -1, dtype=torch.int64)
        x = s["scores"].cpu().tolist() if s["scores"].numel() < 1 << 22 else None
        if x is None:
            return None
        for t, (_, v) in enumerate(vis):
            n = -(-v // page)
            for h in range(hk):
                best = sorted(range(n), key=lambda j: (not (j < s["first"] or j >= n - s["last"]),
                                                       -x[t][h][j], j))
                best = sorted(best[:s["keep"]])
                out[t, h, :len(best)] = torch.tensor(best)
        return out
    hq, d = case["hq"], case["d"]
    q = s["q"].to(torch.float64).view(-1, hk, hq // hk, d)
    ks = torch.ones(hk, device=DEV) if s["ks"] is None else s["ks"]
    if kind == "scores":
        out = torch.full((s["n"], hk, len(bt[0])), -math.inf, dtype=torch.float64, device=DEV)
        for t, (b, v) in enumerate(vis):
            n = -(-v // page)
            x = _f64(s["bounds"], bt[b][:n]) * ks.to(torch.float64).view(1, -1, 1, 1)
            for g in range(hq // hk):
                e = torch.maximum(q[t, :, g] * x[:, :, 0], q[t, :, g] * x[:, :, 1]).sum(-1)
                out[t, :, :n] = torch.maximum(out[t, :, :n], e.T)
        return out
    vs = torch.ones(hk, device=DEV) if s["vs"] is None else s["vs"]
    ks, vs = ks.to(torch.float64).view(1, -1, 1), vs.to(torch.float64).view(1, -1, 1)
    sinks = None if s["sinks"] is None else s["sinks"].to(torch.float64).view(hk, -1)
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    if kind == "prefix":
        for b, n in enumerate(s["ctx"].tolist()):
            at = bt[b][:-(-n // page)]
            k, v = (_f64(s[c], at).reshape(-1, hk, d)[:n] for c in "kv")
            out[b] = _attend64(q[b], k * ks, v * vs, s["scale"], sinks)
        return out.view(-1, hq, d)
    idx = s["idx"].tolist()
    for t, (b, n) in enumerate(vis):
        for h in range(hk):
            at = [j for j in idx[t][h] if j >= 0]
            pos = torch.tensor([j * page + i for j in at for i in range(page)], device=DEV)
            k, v = (_f64(s[c][:, :, h], [bt[b][j] for j in at]).reshape(-1, 1, d)[pos < n]
                    for c in "kv")
            one = None if sinks is None else sinks[h:h + 1]
            out[t, h:h + 1] = _attend64(q[t, h:h + 1], k * ks[:, h:h + 1], v * vs[:, h:h + 1],
                                        s["scale"], one)
    return out.view(-1, hq, d)
