"""Block-sparse attention over a paged cache (GPU): page bounds, page scores, selection and
sparse decode against float64 definitions (``oracle.partial``), and a run of them together.

Tolerances.  Bounds and selections are exact.  A score is a float32 sum of 2 D exact products:
2 D 2^-24 times the sum of their magnitudes.  An attention output rounds each weight to bf16
(2^-8 relative of the average of |v|) and the result once more (2^-8 of it); the logits'
float32 sums (D 2^-24 of their magnitudes, with as much again for the scaling and the
exponential) move each weight by twice that relative amount.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import partial as ref

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
U = 2.0 ** -8  # half a bf16 step, relative


def f64(t):
    return t.float().double().cpu().numpy() if t is not None else None


def make_cache(g, nb, page, hk, d, kv, dev, bias=True):
    x = torch.randn(nb, page, hk, d, generator=g, device=dev)
    if bias:
        x = x + 0.5 * torch.randn(hk, d, generator=g, device=dev)
    return (x * 4).clamp(-448, 448).to(FP8) if kv == "fp8" else x.to(torch.bfloat16)


def poison(cache, mask):
    """NaN at cache[mask] (fp8: the NaN code)."""
    if cache.dtype == FP8:
        cache.view(torch.uint8)[mask] = 0x7F
    else:
        cache[mask] = float("nan")


def tables(g, pages, dev, extra=3):
    """Random distinct pages, -1 behind; pool size."""
    pool = sum(pages) + extra
    perm = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    bt = torch.full((len(pages), max([1, *pages]) + 1), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, p in enumerate(pages):
        bt[i, :p] = perm[at:at + p]
        at += p
    return bt, pool


def int32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def cu_of(n, dev):
    return int32(np.concatenate([[0], np.cumsum(n)]).tolist(), dev)


def attn_tolerance(want, mean, mag, d):
    return U * (mean + np.abs(want)) * 1.01 + 4 * d * 2.0 ** -24 * mag * mean + 1e-30


def check_attn(out, want, mean, mag):
    got = f64(out)
    seen = ~np.isnan(want)
    assert np.isfinite(got[seen]).all()
    err = np.abs(got - want)[seen] - attn_tolerance(want, mean, mag, want.shape[2])[seen]
    assert err.size == 0 or err.max() <= 0, f"beyond the tolerance by {err.max()}"
    return seen


# ---------------------------------------------------------------------------
# update_key_bounds
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kv,d,hk,page,lens,new", [
    ("bf16", 128, 8, 16, [1, 16, 17, 0, 500], None),
    ("bf16", 64, 5, 32, [33, 64, 7], [3, 33, 7]),
    ("bf16", 256, 2, 256, [300, 256, 1], [300, 1, 1]),
    ("fp8", 128, 8, 64, [200, 65, 0, 64], [200, 2, 0, 64]),
    ("fp8", 64, 20, 16, [90, 3], None),
    ("fp8", 256, 1, 128, [129, 1000], [129, 500]),
])
def test_key_bounds(cuda, kv, d, hk, page, lens, new):
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(len(lens) + d)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    k = make_cache(g, pool, page, hk, d, kv, cuda)
    # what lies behind a sequence's tokens is not to be seen; one key that counts is NaN
    for b, n in enumerate(lens):
        if n % page:
            poison(k, (int(bt[b, n // page]), slice(n % page, None)))
    b0 = max(range(len(lens)), key=lambda b: lens[b])
    poison(k, (int(bt[b0, (lens[b0] - 1) // page]), (lens[b0] - 1) % page, 0, 5))
    bounds = torch.full((pool, hk, 2, d), 3.0, device=cuda).to(k.dtype)
    cu = None if new is None else cu_of(new, cuda)
    want = ref.update_key_bounds(f64(bounds), f64(k), bt.cpu().numpy(), lens,
                                 None if cu is None else cu.cpu().numpy())
    for _ in range(2):  # a second call changes nothing
        ops.update_key_bounds(bounds, k, bt, int32(lens, cuda), cu, 1 if new is None else max(new))
        assert np.array_equal(f64(bounds), want, equal_nan=True)
    assert np.isnan(want).any()


def test_key_bounds_masked_pages_and_draft_rollback(cuda):
    """Pages without a table entry are left alone, and a page's bounds follow the length."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(3)
    k = make_cache(g, 6, 16, 2, 128, "bf16", cuda)
    bt = int32([[2, -1, 4], [9, 1, 0]], cuda)
    bounds = ops.new_key_bounds(k)
    for lens, new in (([40, 30], [40, 30]), ([36, 20], [4, 4])):
        want = ref.update_key_bounds(f64(bounds), f64(k), bt.cpu().numpy(), lens,
                                     np.concatenate([[0], np.cumsum(new)]))
        ops.update_key_bounds(bounds, k, bt, int32(lens, cuda), cu_of(new, cuda), 40)
        assert np.array_equal(f64(bounds), want)


# ---------------------------------------------------------------------------
# block_scores
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kv,hq,hk,d,page,lens,rows", [
    ("bf16", 32, 8, 128, 16, [700, 1, 0, 16, 333], None),
    ("bf16", 20, 20, 64, 32, [400, 90], [5, 17]),
    ("bf16", 16, 2, 256, 64, [1000, 64, 63], [3, 0, 1]),
    ("bf16", 15, 5, 128, 16, [130, 40], [4, 6]),
    ("bf16", 66, 2, 128, 16, [290], None),
    ("fp8", 64, 8, 128, 16, [500, 257], [2, 4]),
    ("fp8", 10, 2, 64, 256, [4000, 10], None),
    ("fp8", 8, 1, 256, 16, [300], [9]),
])
def test_block_scores(cuda, kv, hq, hk, d, page, lens, rows):
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(hq + d + page)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    pair = make_cache(g, pool, 2, hk, d, kv, cuda).transpose(1, 2).float()
    bounds = pair.sort(dim=2).values.to(FP8 if kv == "fp8" else torch.bfloat16).contiguous()
    if lens[0] > 100:
        bt[0, 3] = -1
    cu = None if rows is None else cu_of(rows, cuda)
    n = len(lens) if rows is None else sum(rows) + 2  # two rows behind the last sequence
    ks = torch.linspace(-0.5, 0.7, hk, device=cuda) if kv == "fp8" else None
    # q rows as a view of a wider projection; scores of every other row of a wider buffer
    q = torch.randn(n, (hq + 4) * d, generator=g, device=cuda).to(torch.bfloat16)[:, :hq * d]
    q = q.view(n, hq, d)
    for width in (bt.shape[1], max(1, bt.shape[1] - 3), bt.shape[1] + 5):
        buf = torch.full((n, 2 * hk, width + 3), 7.0, device=cuda)
        scores = buf[:, ::2, 1:1 + width]
        ops.block_scores(scores, q, bounds, bt, int32(lens, cuda), page, ks, cu,
                         1 if rows is None else max(rows))
        want, mag = ref.block_scores(f64(q), f64(bounds), bt.cpu().numpy(), lens, page, width,
                                     f64(ks), None if cu is None else cu.cpu().numpy())
        got = scores.double().cpu().numpy()
        behind = np.isnan(want)
        assert (got[behind] == 7.0).all()
        seen = np.isfinite(want)
        assert np.array_equal(np.isneginf(got), np.isneginf(want))
        assert (np.abs(got[seen] - want[seen]) <= 2 * d * 2.0 ** -24 * mag[seen]).all()
        left = buf.clone()
        left[:, ::2, 1:1 + width] = 7.0
        assert (left == 7.0).all()  # nothing else is written


def test_block_scores_bound_the_logits_and_show_nan(cuda):
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(1)
    hq, hk, d, page, n = 8, 2, 128, 16, 100
    bt, pool = tables(g, [7], cuda)
    k = make_cache(g, pool, page, hk, d, "bf16", cuda)
    bounds = ops.new_key_bounds(k)
    ctx = int32([n], cuda)
    q = torch.randn(1, hq, d, generator=g, device=cuda).to(torch.bfloat16)
    scores = torch.empty(1, hk, 7, device=cuda)
    ops.update_key_bounds(bounds, k, bt, ctx, cu_of([n], cuda), n)
    ops.block_scores(scores, q, bounds, bt, ctx, page)
    x = torch.einsum("hgd,pthd->hpgt", q[0].double().view(hk, -1, d), k[bt[0, :7].long()].double())
    x[:, 6, :, n - 96:] = -float("inf")
    assert (scores[0].double() >= x.amax((2, 3)) - 1e-4).all()
    k[int(bt[0, 2]), 4, 1, 9] = float("nan")
    ops.update_key_bounds(bounds, k, bt, ctx, cu_of([n], cuda), n)
    ops.block_scores(scores, q, bounds, bt, ctx, page)
    assert torch.isnan(scores[0, 1, 2]) and int(torch.isnan(scores).sum()) == 1


# ---------------------------------------------------------------------------
# select_blocks
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("width,keep,first,last,lens,rows", [
    (50, 8, 1, 2, [800, 1, 0, 130, 128], None),
    (50, 8, 0, 0, [790], [5]),
    (300, 37, 2, 8, [4800, 4000], [3, 2]),
    (2100, 128, 1, 4, [33600, 20001, 600], [2, 1, 1]),
    (20000, 250, 0, 1, [320000], [2]),
    (64, 5, 3, 2, [1024], None),
    (64, 64, 0, 1, [1024, 1009], None),
    (70000, 16, 1, 1, [1120000], None),
    (10, 300, 0, 1, [160], None),
    (1, 1, 0, 1, [16], None),
])
def test_select_blocks(cuda, width, keep, first, last, lens, rows):
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(width + keep)
    cu = None if rows is None else cu_of(rows, cuda)
    n = len(lens) if rows is None else sum(rows) + 1
    x = torch.randn(n, 3, width, generator=g, device=cuda)
    kinds = (x * 4, (x * 2).round() / 2, torch.zeros_like(x))  # distinct, ties, all equal
    for i, s in enumerate(kinds):
        s = s.contiguous()
        if width > 4:
            s[:, 0, 2::7] = -float("inf")
            s[:, 1, 1::9] = float("nan")
            s[:, 2, ::3] = -0.0
            s[:, 1, 3::11] = float("inf")
        # the rows' strides are the caller's
        buf = torch.full((n, 4, width + 1), 1e9, device=cuda)
        buf[:, :3, 1:] = s
        out = torch.full((n, 3, keep + 2), -7, dtype=torch.int32, device=cuda)
        ops.select_blocks(out[:, :, 1:1 + keep], buf[:, :3, 1:], int32(lens, cuda), 16, first,
                          last, cu)
        want = ref.select_blocks(s.cpu().numpy(), lens, 16, keep, first, last,
                                 None if cu is None else cu.cpu().numpy())
        got = out.cpu().numpy()
        assert np.array_equal(got[:, :, 1:1 + keep], want), f"kind {i}"
        assert (got[:, :, 0] == -7).all() and (got[:, :, -1] == -7).all()


@pytest.mark.parametrize("kind", ["outlier", "low_outlier", "close", "negative", "denormal", "huge",
                                  "two", "few_equal", "sorted", "tiny_steps"])
@pytest.mark.parametrize("width,keep,first,last", [(70, 9, 1, 1), (600, 128, 1, 1), (5000, 64, 0, 2),
                                                   (9000, 700, 3, 0), (32768, 1000, 1, 1)])
def test_select_blocks_of_finite_scores(cuda, kind, width, keep, first, last):
    """Distributions that put the lowest selected score where it is hard to find."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(width)
    x = torch.randn(2, 1, width, generator=g, device=cuda)
    if kind == "outlier":
        x[:, :, width // 2] = 1e30
    elif kind == "low_outlier":
        x[:, :, width // 3] = -3e38
    elif kind == "close":
        x = 1 + (x * 50).round() * 2.0 ** -23
    elif kind == "negative":
        x = -x.abs() - 1
    elif kind == "denormal":
        x = x * 1e-40
    elif kind == "huge":
        x = x.clamp(-3, 3) * 1.1e38
    elif kind == "two":
        x = (x > 0.5).float()
    elif kind == "few_equal":
        x[:, :, ::width // 30] = x.flatten().sort().values[-keep]
    elif kind == "sorted":
        x = x.sort(dim=2, descending=True).values
    else:
        x = torch.arange(width, device=cuda).expand(2, 1, width) * 1e-31
    lens = [16 * width, 16 * width - 37]
    out = torch.full((2, 1, keep), -7, dtype=torch.int32, device=cuda)
    ops.select_blocks(out, x.contiguous(), int32(lens, cuda), 16, first, last)
    want = ref.select_blocks(x.cpu().numpy(), lens, 16, keep, first, last)
    assert np.array_equal(out.cpu().numpy(), want)


# ---------------------------------------------------------------------------
# sparse_paged_decode
# ---------------------------------------------------------------------------
def pick(g, n, hk, keep, nblk, dev):
    """Distinct visible blocks per (row, kv head), -1 behind."""
    idx = torch.full((n, hk, keep), -1, dtype=torch.int32)
    for t in range(n):
        for h in range(hk):
            k = min(keep, nblk[t])
            idx[t, h, :k] = torch.randperm(nblk[t], generator=g)[:k].sort().values.to(torch.int32)
    return idx.to(dev)


SPARSE = [
    ("bf16", 32, 8, 128, 16, [900, 1, 0, 47], None, 20),
    ("bf16", 32, 8, 128, 16, [5000], None, 200),
    ("bf16", 20, 20, 64, 32, [300, 64], [3, 5], 4),
    ("bf16", 16, 2, 256, 64, [700, 65], [2, 1], 3),
    ("bf16", 15, 5, 128, 16, [333], [6], 9),
    ("bf16", 40, 2, 128, 128, [1500, 129], None, 5),
    ("bf16", 32, 2, 256, 256, [3000], None, 12),
    ("bf16", 4, 4, 128, 16, [40] * 70, None, 3),
    ("fp8", 64, 8, 128, 64, [2000, 70, 64], [4, 1, 2], 11),
    ("fp8", 8, 1, 64, 16, [100], None, 1),
    ("fp8", 24, 2, 256, 32, [500], [3], 7),
    ("fp8", 6, 3, 128, 1024, [5000, 1024], None, 2),
]


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("kv,hq,hk,d,page,lens,rows,keep", SPARSE)
def test_sparse_decode(cuda, kv, hq, hk, d, page, lens, rows, keep, sinks):
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(hq * d + page)
    cpu = torch.Generator().manual_seed(page + hq)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    k = make_cache(g, pool, page, hk, d, kv, cuda)
    v = make_cache(g, pool, page, hk, d, kv, cuda)
    cu = None if rows is None else cu_of(rows, cuda)
    n = len(lens) if rows is None else sum(rows) + 1
    info = ref.query_rows(lens, None if cu is None else cu.cpu().numpy(), n)
    nblk = [0] * n
    for t, _, vis in info:
        nblk[t] = max(-(-vis // page), 0)
    idx = pick(cpu, n, hk, keep, nblk, cuda)
    # keys that no row attends to are NaN: unused pages, and what lies behind the sequences
    used = torch.zeros(pool, page, dtype=torch.bool, device=cuda)
    for t, b, vis in info:
        for j in set(idx[t].flatten().tolist()) - {-1}:
            used[int(bt[b, j]), :max(0, min(page, lens[b] - j * page))] = True
    for c in (k, v):
        poison(c, ~used)
    ks = vs = None
    if kv == "fp8":
        ks, vs = torch.linspace(0.1, 0.3, hk, device=cuda), torch.linspace(0.2, 0.4, hk,
                                                                          device=cuda)
    s = torch.randn(hq, generator=g, device=cuda) if sinks else None
    q = torch.randn(n, hq + 2, d, generator=g, device=cuda).to(torch.bfloat16)[:, :hq]
    out = torch.full((n, hq + 1, d), 9.0, dtype=torch.bfloat16, device=cuda)
    ops.sparse_paged_decode(out[:, :hq], q, k, v, bt, int32(lens, cuda), idx, d ** -0.5, ks, vs, s,
                            cu)
    want, mean, mag = ref.sparse_paged_decode(
        f64(q), f64(k), f64(v), bt.cpu().numpy(), lens, idx.cpu().numpy(), d ** -0.5, f64(ks),
        f64(vs), f64(s), None if cu is None else cu.cpu().numpy())
    seen = check_attn(out[:, :hq], want, mean, mag)
    assert (f64(out)[:, hq] == 9.0).all() and (f64(out)[:, :hq][~seen] == 9.0).all()


def test_sparse_decode_lists(cuda):
    """Entries in any order, out of range, at masked pages, and twice; an empty list."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(11)
    hq, hk, d, page, lens = 8, 2, 128, 16, [150, 150, 20]
    bt, pool = tables(g, [10, 10, 2], cuda)
    bt[1, 4] = -1
    bt[1, 5] = 10 ** 6
    k, v = (make_cache(g, pool, page, hk, d, "bf16", cuda) for _ in range(2))
    q = torch.randn(3, hq, d, generator=g, device=cuda).to(torch.bfloat16)
    idx = int32([[[9, 0, 3, 3, -1, 7], [-5, 2, 10, 2 ** 31 - 1, 1, 1]],
                 [[4, 5, -1, -1, -1, -1], [4, 5, 6, 8, 0, 2]],
                 [[2, 3, 9, -1, -1, -1], [-1, -1, -1, -1, -1, 1]]], cuda)
    for keep in (6, 1, 0):
        i = idx[:, :, :keep]
        out = torch.full_like(q, 5.0)
        ops.sparse_paged_decode(out, q, k, v, bt, int32(lens, cuda), i, d ** -0.5)
        want = ref.sparse_paged_decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), lens,
                                       i.cpu().numpy(), d ** -0.5)
        check_attn(out, *want)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def load(stem, name):
    import importlib

    return getattr(importlib.import_module(f"fastkernels_amd.candidate.L1.{stem}"), name)


@pytest.mark.parametrize("kv,hq,hk,d,page", [("bf16", 32, 8, 128, 16), ("fp8", 16, 2, 256, 32),
                                             ("bf16", 6, 2, 64, 16)])
def test_sparse_steps(cuda, kv, hq, hk, d, page):
    """A prompt stored in two chunks and decode steps after it: store, bounds, forward_sparse.
    With every page selected the result is decode attention's; with few, attention over the
    pages that the scores select."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(d)
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)
    lens = [37, 300]
    bt, pool = tables(g, [20, 40], cuda)
    dtype = FP8 if kv == "fp8" else torch.bfloat16
    kc = torch.zeros(pool, page, hk, d, device=cuda).to(dtype)
    vc = kc.clone()
    bounds = ops.new_key_bounds(kc)
    scale = dict(k_scale=0.05, v_scale=0.08) if kv == "fp8" else {}

    def store(old, new):
        total = sum(new)
        k, v = (20 * torch.randn(total, hk, d, generator=g, device=cuda).to(torch.bfloat16)
                if kv == "fp8" else torch.randn(total, hk, d, generator=g,
                                                device=cuda).to(torch.bfloat16)
                for _ in range(2))
        slots = [int(bt[b, t // page]) * page + t % page
                 for b in range(2) for t in range(old[b], old[b] + new[b])]
        ops.store_kvcache(k, v, kc, vc, torch.tensor(slots, device=cuda))
        now = int32([a + b for a, b in zip(old, new)], cuda)
        ops.update_key_bounds(bounds, kc, bt, now, cu_of(new, cuda), max(new))
        return now

    store([0, 0], [20, 123])
    store([20, 123], [17, 177])
    for step in range(3):
        ctx = store([n + step for n in lens], [1, 1])
        q = torch.randn(2, hq, d, generator=g, device=cuda).to(torch.bfloat16)
        every = attn.forward_sparse(q, kc, vc, bounds, ctx, 40, block_table=bt, **scale)
        dense = attn(q, kc, vc, ctx, block_table=bt, **scale)
        now = ctx.tolist()
        all_idx = np.tile(np.arange(bt.shape[1]), (2, hk, 1))
        one = {k: np.full(hk, v) for k, v in scale.items()}
        want = ref.sparse_paged_decode(f64(q), f64(kc), f64(vc), bt.cpu().numpy(), now, all_idx,
                                       d ** -0.5, **one)
        check_attn(every, *want)
        check_attn(dense, *want)
        few = attn.forward_sparse(q, kc, vc, bounds, ctx, 4, keep_first=1, keep_last=1,
                                  block_table=bt, max_seq_len=max(now), **scale)
        width = -(-max(now) // page)
        scores = torch.empty(2, hk, width, device=cuda)
        ops.block_scores(scores, q, bounds, bt, ctx, page,
                         torch.full((hk,), 0.05, device=cuda) if kv == "fp8" else None)
        idx = ref.select_blocks(scores.cpu().numpy(), now, page, 4, 1, 1)
        want = ref.sparse_paged_decode(f64(q), f64(kc), f64(vc), bt.cpu().numpy(), now, idx,
                                       d ** -0.5, **one)
        check_attn(few, *want)


def test_sparse_in_a_graph(cuda):
    """forward_sparse captured once and replayed as the lengths grow, with eager calls of
    another size between; every replay against the eager result."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(2)
    hq, hk, d, page = 32, 8, 128, 16
    bt, pool = tables(g, [60, 60, 60], cuda)
    k, v = (make_cache(g, pool, page, hk, d, "bf16", cuda) for _ in range(2))
    bounds = ops.new_key_bounds(k)
    ctx = int32([400, 950, 17], cuda)
    q = torch.randn(3, hq, d, generator=g, device=cuda).to(torch.bfloat16)
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)

    def step():
        ops.update_key_bounds(bounds, k, bt, ctx)
        return attn.forward_sparse(q, k, v, bounds, ctx, 24, keep_last=2, block_table=bt)

    ops.update_key_bounds(bounds, k, bt, ctx, cu_of(ctx.tolist(), cuda), 950)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for new in ([400, 950, 17], [401, 951, 18], [500, 960, 0], [33, 1, 31]):
        ctx.copy_(int32(new, cuda))
        ops.update_key_bounds(bounds, k, bt, ctx, cu_of(new, cuda), 960)
        q.copy_(torch.randn(3, hq, d, generator=g, device=cuda))
        graph.replay()
        got = out.clone()
        other = attn.forward_sparse(q[:2], k, v, bounds, ctx, 9, block_table=bt)
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and bool(torch.isfinite(other).all())


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("sign", [-1, 1])
def test_scores_of_great_magnitude(cuda, rows, sign):
    """Logits of +-2^123, all equal: the mean of V, in fp32 exactly (64 small integers)."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(rows)
    hq, hk, d, page = 4, 2, 64, 16
    k = torch.full((4, page, hk, d), sign * 2.0 ** 60, dtype=torch.bfloat16, device=cuda)
    v = torch.randint(-3, 4, (4, page, hk, d), generator=g, device=cuda).to(torch.bfloat16)
    q = torch.full((rows, hq, d), 2.0 ** 60, dtype=torch.bfloat16, device=cuda)
    bt = int32([[2, 0, 3, 1]] * rows, cuda)
    ctx = int32([64] * rows, cuda)
    want = v.float().sum((0, 1)).div(64).repeat_interleave(hq // hk, 0).to(torch.bfloat16)
    sparse, prefix = torch.zeros_like(q), torch.zeros_like(q)
    ops.sparse_paged_decode(sparse, q, k, v, bt, ctx,
                            int32([[[0, 1, 2, 3]] * hk] * rows, cuda), d ** -0.5)
    ops.shared_prefix_decode(prefix, q, k, v, bt, ctx, int32([0, rows], cuda), int32([40], cuda),
                             d ** -0.5)
    assert torch.equal(sparse, want.expand_as(q)) and torch.equal(prefix, want.expand_as(q))


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_score_above_great_ones(cuda, kv, d):
    """Logits near +-2^100 whose rounding alone is beyond any exponent: the greatest key's V."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(d)
    hq, hk, page, n = 4, 2, 16, 150
    q = (torch.randn(2, hq, d, generator=g, device=cuda).abs() + 0.1) * 2.0 ** 96
    q[1] *= -1
    row = torch.randn(1, 1, hk, d, generator=g, device=cuda).abs() + 0.1
    k = row.expand(10, page, hk, d).clone()
    k[4, 3] *= 4     # the greatest logit of row 0
    k[8, 9] *= 0.25  # and of row 1
    dtype = FP8 if kv == "fp8" else torch.bfloat16
    k, q = k.to(dtype), q.to(torch.bfloat16)
    v = torch.randint(-8, 9, (10, page, hk, d), generator=g, device=cuda).to(dtype)
    bt, ctx = int32([list(range(10))] * 2, cuda), int32([n, n], cuda)
    one = torch.ones(hk, device=cuda) if kv == "fp8" else None
    want = torch.stack([v[4, 3], v[8, 9]]).to(torch.bfloat16).repeat_interleave(hq // hk, 1)
    sparse, prefix = torch.zeros_like(q), torch.zeros_like(q)
    ops.sparse_paged_decode(sparse, q, k, v, bt, ctx,
                            int32([[list(range(10))] * hk] * 2, cuda), 0.1, one, one)
    ops.shared_prefix_decode(prefix, q, k, v, bt, ctx, int32([0, 2], cuda), int32([100], cuda), 0.1,
                             one, one)
    assert torch.equal(sparse, want) and torch.equal(prefix, want)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_caches_past_4_gib(cuda, kv):
    """Pages whose byte offsets pass 32 bits, against the same pages in a small cache."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(3)
    hq, hk, d, page = 16, 8, 128, 256
    dtype = FP8 if kv == "fp8" else torch.bfloat16
    nb = (5 << 30) // (page * hk * d * dtype.itemsize)
    at = [0, nb - 1, nb // 2 + 1, nb - 2]
    small = [make_cache(g, 4, page, hk, d, kv, cuda) for _ in range(2)]
    big = [torch.empty(nb, page, hk, d, dtype=dtype, device=cuda) for _ in range(2)]
    for x, y in zip(big, small):
        for i, p in enumerate(at):
            x[p] = y[i]
    q = torch.randn(3, hq, d, generator=g, device=cuda).to(torch.bfloat16)
    one = torch.ones(hk, device=cuda) if kv == "fp8" else None
    ctx = int32([1000, 1024, 700], cuda)
    got = []
    for (k, v), pages in ((small, [0, 1, 2, 3]), (big, at)):
        bt = int32([pages] * 3, cuda)
        bounds = ops.new_key_bounds(k)
        # (of the sequence that fills them: bounds of a shared page are those of one caller)
        ops.update_key_bounds(bounds, k, bt[1:2], ctx[1:2], int32([0, 1024], cuda), 1024)
        scores = torch.empty(3, hk, 4, device=cuda)
        ops.block_scores(scores, q, bounds, bt, ctx, page, one)
        idx = torch.empty(3, hk, 3, dtype=torch.int32, device=cuda)
        ops.select_blocks(idx, scores, ctx, page)
        sparse, prefix = torch.empty_like(q), torch.empty_like(q)
        ops.sparse_paged_decode(sparse, q, k, v, bt, ctx, idx, d ** -0.5, one, one)
        ops.shared_prefix_decode(prefix, q, k, v, bt, ctx, int32([0, 3], cuda),
                                 int32([600], cuda), d ** -0.5, one, one)
        got.append((bounds[pages].float(), scores, idx, sparse, prefix))
    for name, a, b in zip(("bounds", "scores", "pages", "sparse", "prefix"), *got):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_logits_next_to_the_least_float(cuda, kv):
    """Scaled logits between -3.4e38 and -3e38, all equal: the mean of V."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(5)
    hq, hk, d, page = 4, 2, 64, 16
    dtype = FP8 if kv == "fp8" else torch.bfloat16
    k = torch.full((4, page, hk, d), -1.0, device=cuda).to(dtype)
    v = torch.randint(-3, 4, (4, page, hk, d), generator=g, device=cuda).to(dtype)
    q = torch.full((2, hq, d), 2.0 ** 120, dtype=torch.bfloat16, device=cuda)
    bt, ctx = int32([[2, 0, 3, 1]] * 2, cuda), int32([64, 64], cuda)
    one = torch.ones(hk, device=cuda) if kv == "fp8" else None
    want = v.float().sum((0, 1)).div(64).repeat_interleave(hq // hk, 0).to(torch.bfloat16)
    # 2^126 * 2.6 * log2(e) = 3.19e38
    sparse, prefix = torch.zeros_like(q), torch.zeros_like(q)
    ops.sparse_paged_decode(sparse, q, k, v, bt, ctx, int32([[[0, 1, 2, 3]] * hk] * 2, cuda), 2.6,
                            one, one)
    ops.shared_prefix_decode(prefix, q, k, v, bt, ctx, int32([0, 2], cuda), int32([40], cuda), 2.6,
                             one, one)
    assert torch.equal(sparse, want.expand_as(q)) and torch.equal(prefix, want.expand_as(q))


def test_drafted_rows_of_several_chunks(cuda):
    """forward_sparse of more rows per sequence than one group of score columns holds."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(8)
    hq, hk, d, page, lens, rows = 32, 8, 128, 16, [700, 90, 333], [9, 5, 1]
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    k, v = (make_cache(g, pool, page, hk, d, "bf16", cuda) for _ in range(2))
    bounds, ctx, cu = ops.new_key_bounds(k), int32(lens, cuda), cu_of(rows, cuda)
    ops.update_key_bounds(bounds, k, bt, ctx, cu_of(lens, cuda), max(lens))
    q = torch.randn(sum(rows), hq, d, generator=g, device=cuda).to(torch.bfloat16)
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)
    out = attn.forward_sparse(q, k, v, bounds, ctx, 6, cu_seqlens_q=cu, max_seqlen_q=9,
                              block_table=bt)
    scores = torch.empty(sum(rows), hk, bt.shape[1], device=cuda)
    ops.block_scores(scores, q, bounds, bt, ctx, page, None, cu, 9)
    host_cu, host_bt = cu.cpu().numpy(), bt.cpu().numpy()
    s, mag = ref.block_scores(f64(q), f64(bounds), host_bt, lens, page, bt.shape[1], None, host_cu)
    got, seen = scores.double().cpu().numpy(), np.isfinite(s)
    assert np.array_equal(np.isneginf(got), np.isneginf(s))
    assert (np.abs(got[seen] - s[seen]) <= 2 * d * 2.0 ** -24 * mag[seen]).all()
    idx = ref.select_blocks(scores.cpu().numpy(), lens, page, 6, 1, 1, host_cu)
    want = ref.sparse_paged_decode(f64(q), f64(k), f64(v), host_bt, lens, idx, d ** -0.5, None,
                                   None, None, host_cu)
    check_attn(out, *want)


@pytest.mark.parametrize("batch", [65, 150, 5000])
def test_many_sequences(cuda, batch):
    """More sequences than a wave has lanes, of 0 to 3 rows each: every operator of a step."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(batch)
    hq, hk, d, page, keep = 4, 1, 64, 16, 2
    lens = [(23 * b) % 90 for b in range(batch)]
    rows = [min(lens[b], (2, 0, 1, 0, 0, 3)[b * 5 // 7 % 6]) for b in range(batch)]
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    k, v = (make_cache(g, pool, page, hk, d, "bf16", cuda) for _ in range(2))
    cu, ctx, n = cu_of(rows, cuda), int32(lens, cuda), sum(rows) + 2
    host_cu, host_bt = cu.cpu().numpy(), bt.cpu().numpy()
    bounds = ops.new_key_bounds(k)
    ops.update_key_bounds(bounds, k, bt, ctx, cu_of(lens, cuda), max(lens))
    want = ref.update_key_bounds(np.zeros(bounds.shape), f64(k), host_bt, lens,
                                 np.concatenate([[0], np.cumsum(lens)]))
    assert np.array_equal(f64(bounds), want)
    q = torch.randn(n, hq, d, generator=g, device=cuda).to(torch.bfloat16)
    scores = torch.full((n, hk, bt.shape[1]), 7.0, device=cuda)
    ops.block_scores(scores, q, bounds, bt, ctx, page, None, cu, 3)
    want, mag = ref.block_scores(f64(q), f64(bounds), host_bt, lens, page, bt.shape[1], None,
                                 host_cu)
    got = scores.double().cpu().numpy()
    assert (got[np.isnan(want)] == 7.0).all()
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    seen = np.isfinite(want)
    assert (np.abs(got[seen] - want[seen]) <= 2 * d * 2.0 ** -24 * mag[seen]).all()
    idx = torch.full((n, hk, keep), -7, dtype=torch.int32, device=cuda)
    ops.select_blocks(idx, scores, ctx, page, 0, 1, cu)
    want = ref.select_blocks(scores.cpu().numpy(), lens, page, keep, 0, 1, host_cu)
    assert np.array_equal(idx.cpu().numpy(), want)
    out = torch.full_like(q, 9.0)
    ops.sparse_paged_decode(out, q, k, v, bt, ctx, idx, d ** -0.5, cu_seqlens_q=cu)
    want = ref.sparse_paged_decode(f64(q), f64(k), f64(v), host_bt, lens, idx.cpu().numpy(),
                                   d ** -0.5, None, None, None, host_cu)
    seen = check_attn(out, *want)
    assert (f64(out)[~seen] == 9.0).all()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("scale", [-0.11, 0.0])
def test_sparse_of_odd_arguments(cuda, kv, scale):
    """Lengths past the table, a scale that is not positive, key scales of either sign, the
    output in place of the query."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(13)
    hq, hk, d, page, width = 24, 2, 128, 16, 12
    lens = [48, 10 ** 6, 2 ** 31 - 1, 0]
    bt = torch.stack([torch.randperm(40, generator=g, device=cuda)[:width] for _ in lens])
    bt = bt.to(torch.int32)
    k, v = (make_cache(g, 40, page, hk, d, kv, cuda) for _ in range(2))
    q = torch.randn(len(lens), hq, d, generator=g, device=cuda).to(torch.bfloat16)
    ks = vs = None
    if kv == "fp8":
        ks, vs = torch.tensor([0.2, -0.3], device=cuda), torch.tensor([-0.1, 0.4], device=cuda)
    bounds, ctx = ops.new_key_bounds(k), int32(lens, cuda)
    ops.update_key_bounds(bounds, k, bt, int32([min(n, width * page) for n in lens], cuda),
                          int32([0, 48, 240, 432, 432], cuda), 192)
    scores = torch.empty(4, hk, width, device=cuda)
    ops.block_scores(scores, q, bounds, bt, ctx, page, ks)
    want, mag = ref.block_scores(f64(q), f64(bounds), bt.cpu().numpy(), lens, page, width, f64(ks))
    got, seen = scores.double().cpu().numpy(), np.isfinite(want)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    assert (np.abs(got[seen] - want[seen]) <= 2 * d * 2.0 ** -24 * mag[seen]).all()
    idx = torch.empty(4, hk, 7, dtype=torch.int32, device=cuda)
    ops.select_blocks(idx, scores, ctx, page, 1, 2)
    assert np.array_equal(idx.cpu().numpy(),
                          ref.select_blocks(scores.cpu().numpy(), lens, page, 7, 1, 2))
    want, mean, mag = ref.sparse_paged_decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), lens,
                                              idx.cpu().numpy(), scale, f64(ks), f64(vs))
    ops.sparse_paged_decode(q, q, k, v, bt, ctx, idx, scale, ks, vs)
    check_attn(q, want, np.abs(mean), np.abs(mag))
