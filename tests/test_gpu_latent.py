"""The latent cache (GPU): store with norm and rotation, read-back and decode attention against
float64 definitions (``oracle.small_cache``), and a run of them together.

Tolerances.  A stored value is computed in float32 and rounded once: 2^-8 (bf16) or 2^-4 (fp8; at
least half its smallest step, 2^-10) of it, after float32 errors: 2^-24 for each of the 512
squares of the norm's sum and 8 roundings around it, 4 for the two products of a rotation, of the
sum of their magnitudes.  The attention's operands are exact (an fp8 code is a bf16 value, its
scale goes to the logits and the result): its output differs as that of any bf16 cache, with 576
products a logit, and by the float32 sums over the keys, 2^-24 of the average of |c| for each.
The log-sum-exp differs by the logits' errors, the sum's (2^-24 a key), and 8 roundings of it.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import small_cache as ref
from test_gpu_sparse import U, attn_tolerance, cu_of, f64, int32, load, tables

pytestmark = pytest.mark.gpu

BF, FP8 = torch.bfloat16, torch.float8_e4m3fn
E24 = 2.0 ** -24


def check(out, lse, want, mean, mag, want_lse, keys, dims=576):
    """NaN in `want`: not compared.  dims: products of a logit that are not zero."""
    got, seen = f64(out), ~np.isnan(want)
    assert np.isfinite(got[seen]).all()
    tol = attn_tolerance(want, mean, mag, dims) + keys * E24 * mean
    err = (np.abs(got - want) - tol)[seen]
    assert err.size == 0 or err.max() <= 0, f"beyond the tolerance by {err.max()}"
    if lse is not None:
        got = lse.double().cpu().numpy()
        rows = ~np.isnan(want_lse)
        none = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(got) & rows, none)
        tol = 4 * dims * E24 * mag[:, :, 0].T + keys * E24 + 8 * E24 * (1 + np.abs(want_lse))
        some = rows & ~none
        err = np.abs(got[some] - want_lse[some]) - tol[some]
        assert err.size == 0 or err.max() <= 0, f"lse beyond the tolerance by {err.max()}"
    return seen


def make_cache(g, nb, page, kv, dev):
    x = torch.randn(nb, page, 576, generator=g, device=dev)
    x = x + 0.5 * torch.randn(576, generator=g, device=dev)
    return (x * 4).to(FP8) if kv == "fp8" else x.to(BF)


def poison(cache, bt, lens, keep=None):
    """NaN, and infinities where the type has them, wherever no sequence has a token."""
    nb, page, _ = cache.shape
    used = torch.zeros(nb, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(min(-(-n // page), bt.shape[1])):
            if 0 <= int(bt[b, j]) < nb:
                used[int(bt[b, j]), :min(page, n - j * page)] = True
    free = (~used).to(cache.device)
    if cache.dtype == FP8:
        cache.view(torch.uint8)[free] = 0x7F
    else:
        cache[free] = float("nan")
        cache[free.logical_and(torch.arange(page, device=cache.device) % 2 == 1)] = float("inf")


def scale_of(kv, dev):
    return torch.tensor([0.21], device=dev) if kv == "fp8" else None


def dense(cache, scale):
    return f64(cache) * (1.0 if scale is None else float(scale.item()))


# ---------------------------------------------------------------------------
# store and read-back
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("n,heads,page,i64,cs", [(1, 16, 16, True, "f32"), (65, 128, 64, False, "f32"),
                                                 (300, 5, 16, True, "bf16"), (7, 0, 32, False, "f32"),
                                                 (33, 20, 256, False, "bf16")])
def test_store(cuda, kv, neox, n, heads, page, i64, cs):
    """Rows of wider tensors, skipped and out-of-range slots, positions past the table, with and
    without the norm and the extra outputs; everything else left as it was."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(n + heads)
    nb = -(-n // page) + 1
    cache = make_cache(g, nb, page, kv, cuda)
    before = f64(cache)
    scale = scale_of(kv, cuda)
    proj = torch.randn(n, 512 + 64 + 8, generator=g, device=cuda).to(BF) * 3
    latent, key = proj[:, :512], proj[:, 512:576]
    qp = torch.randn(n, max(heads, 1), 192, generator=g, device=cuda).to(BF)
    absorbed = torch.full((n, max(heads, 1), 576), 9.0, dtype=BF, device=cuda)
    cos_sin = torch.randn(40, 64, generator=g, device=cuda).to(BF if cs == "bf16" else torch.float32)
    pos = torch.randint(0, 40, (n,), generator=g, device=cuda)
    if n > 6:
        pos[3], pos[5] = 40, -1
    slots = torch.randperm(nb * page, generator=g, device=cuda)[:n]
    if n > 6:
        slots[2], slots[6] = -1, nb * page
    if n > 100:
        slots[7] = 1 << 40
    w = None if n == 33 else (torch.rand(512, generator=g, device=cuda) + 0.5).to(BF)
    c_out = torch.full((n, 520), 9.0, dtype=BF, device=cuda)
    k_out = torch.full((n, 72), 9.0, dtype=BF, device=cuda)
    q = {} if heads == 0 else dict(query_rope=qp[:, :, 128:], query_out=absorbed[:, :, 512:])
    extra = dict(latent_out=c_out[:, :512], key_rope_out=k_out[:, 8:]) if n != 65 else {}
    ops.latent_norm_rope_store(cache, slots if i64 else slots.to(torch.int32), pos, latent, key,
                               cos_sin, neox, w, 1e-5, scale, **q, **extra)
    cs64, p = f64(cos_sin), pos.tolist()
    c, k = ref.latent_rows(f64(latent), f64(key), p, cs64, neox, None if w is None else f64(w), 1e-5)
    k_mag = np.abs(f64(key)) + np.abs(f64(key)).max(-1, keepdims=True)  # of both products, at least
    k_mag = k_mag * max(1.0, np.abs(cs64).max())
    f32 = np.concatenate([(520 * E24 if w is not None else 0) * np.abs(c), 4 * E24 * k_mag], 1)
    rows = np.concatenate([c, k], 1)

    def close(got, want, err, half=U, least=0.0):
        bad = np.abs(got - want) - (np.maximum(half * np.abs(want), least) + err * (1 + half))
        assert bad.max() <= 0, bad.max()

    want, s = before.copy(), 1.0 if scale is None else float(scale.item())
    slack = np.zeros_like(want)
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < nb * page:
            want[slot // page, slot % page] = np.clip(rows[t] / s, -448, 448) if kv == "fp8" else rows[t]
            slack[slot // page, slot % page] = f32[t] / s + E24 * np.abs(rows[t] / s)
    got, mine = f64(cache), slack.max(-1) > 0
    assert np.array_equal(got[~mine], before[~mine])
    if mine.any():
        close(got[mine], want[mine], slack[mine], *((2.0 ** -4, 2.0 ** -10) if kv == "fp8" else (U,)))
    if extra:
        close(f64(c_out[:, :512]), c, f32[:, :512])
        close(f64(k_out[:, 8:]), k, f32[:, 512:])
        assert bool((c_out[:, 512:] == 9.0).all()) and bool((k_out[:, :8] == 9.0).all())
    if heads:
        qx = f64(qp[:, :, 128:])
        wq = np.stack([ref.rotate(x, i, cs64, neox) for x, i in zip(qx, p)])
        mag = 2 * np.abs(qx).max(-1, keepdims=True) * max(1.0, np.abs(cs64).max())
        close(f64(absorbed[:, :, 512:]), wq, 4 * E24 * np.broadcast_to(mag, wq.shape))
        assert bool((absorbed[:, :, :512] == 9.0).all())


def test_store_in_place_and_special_values(cuda):
    """Outputs that are their own inputs; NaN, infinities and rows of zeros."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(1)
    latent = torch.randn(5, 512, generator=g, device=cuda).to(BF)
    key = torch.randn(5, 64, generator=g, device=cuda).to(BF)
    query = torch.randn(5, 16, 64, generator=g, device=cuda).to(BF)
    latent[1], latent[2, 7], latent[3, 9], key[4, 5] = 0.0, float("nan"), float("inf"), float("nan")
    cos_sin = torch.randn(8, 64, generator=g, device=cuda)
    pos = torch.arange(5, device=cuda)
    w = torch.ones(512, dtype=BF, device=cuda)
    for kv in ("bf16", "fp8"):
        got = []
        for inplace in (False, True):
            x = [t.clone() for t in (latent, key, query)]
            y = x if inplace else [torch.empty_like(t) for t in x]
            cache = torch.zeros(1, 16, 576, device=cuda).to(FP8 if kv == "fp8" else BF)
            ops.latent_norm_rope_store(cache, pos, pos, x[0], x[1], cos_sin, True, w, 1e-6,
                                       query_rope=x[2], query_out=y[2], latent_out=y[0],
                                       key_rope_out=y[1])
            got.append([cache.float()] + [t.float() for t in y])
        for a, b in zip(*got):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
        rows = got[0][0][0]
        assert bool((rows[1, :512] == 0).all()) and bool(rows[2, :512].isnan().all())
        assert bool(rows[3, 9].isnan()) and bool((rows[3, :9] == 0).all())  # inf / inf, x / inf
        assert rows[4, 512:].isnan().sum() == 2 and not rows[4, :512].isnan().any()
        assert not rows[0].isnan().any()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("page,lens", [(16, [17, 0, 1, 300]), (64, [64, 65, 200]), (256, [1]),
                                       (32, [0, 33, 0, 0, 90]), (16, [1500, 0, 1601]),
                                       (64, [9000, 1, 8001])])
def test_gather(cuda, kv, page, lens):
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(page)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = make_cache(g, pool, page, kv, cuda)
    poison(cache, bt, lens)
    scale = scale_of(kv, cuda)
    if lens[-1] > page:
        bt[-1, 0], bt[-1, 1] = -1, pool
    cu, total = cu_of(lens, cuda) + 2, sum(lens) + 7
    out = torch.full((total, 584), 9.0, dtype=BF, device=cuda)
    ops.gather_latent(out[:, :576], cache, bt, cu, scale)
    want = ref.gather(f64(cache), bt.cpu().numpy(), cu.tolist(), total)
    s = 1.0 if scale is None else np.float32(scale.item())
    want = torch.tensor(want).float() * torch.tensor(s)  # the product in float32, rounded once
    want[:2], want[2 + sum(lens):] = 9.0, 9.0
    assert torch.equal(out[:, :576].cpu(), want.to(BF)) and bool((out[:, 576:] == 9.0).all())


# ---------------------------------------------------------------------------
# decode attention
# ---------------------------------------------------------------------------
BATCHES = {
    "one": ([1], None), "zeros": ([0, 0], None), "short": ([31, 33, 0, 1, 16], None),
    "mixed": ([700, 5, 0, 1300, 64, 63, 65], None),
    "drafts": ([300, 3, 40, 1, 900], [4, 3, 1, 1, 5]),
    "holes": ([300, 2, 0, 70], [0, 3, 2, 2]),  # more rows than tokens: the first see none
    "many": ([17 * i % 90 for i in range(70)], None),
    "negative": ([40, -3, 20], None),  # a length below zero is none
}


def run(cuda, cache, heads, bt, lens, rows, scale, s, g, spare=0, most=None, q=None):
    """(out, lse, what is to be compared with) of a call with strided tensors."""
    from fastkernels_amd import ops

    n = len(lens) if rows is None else sum(rows)
    if q is None:
        q = torch.randn(n + spare, heads + 1, 584, generator=g, device=cuda).to(BF)[:, :heads, :576]
    out = torch.full((n + spare, heads + 2, 520), 9.0, dtype=BF, device=cuda)
    lse = torch.full((heads, n + spare + 1), 9.0, device=cuda)[:, :n + spare]
    cu = None if rows is None else cu_of(rows, cuda)
    ops.latent_decode(out[:, :heads, :512], q, cache, bt, int32(lens, cuda), s, scale, cu,
                      most or (None if rows is None else max(rows)), lse)
    want = ref.latent_decode(f64(q), dense(cache, scale), bt.cpu().numpy(), lens, s,
                             cu_seqlens_q=None if cu is None else cu.tolist())
    assert bool((out[:, heads:] == 9.0).all()) and bool((out[:, :, 512:] == 9.0).all())
    assert bool((out[n:] == 9.0).all()) and bool((lse[:, n:] == 9.0).all())
    return out[:, :heads, :512], lse, want


@pytest.mark.parametrize("name", list(BATCHES))
@pytest.mark.parametrize("kv,heads,page", [("bf16", 16, 16), ("bf16", 128, 64), ("bf16", 20, 256),
                                           ("fp8", 16, 64), ("fp8", 128, 16), ("bf16", 33, 32),
                                           ("fp8", 1, 128), ("fp8", 70, 32), ("bf16", 64, 16),
                                           ("bf16", 150, 16), ("fp8", 256, 64)])
def test_decode(cuda, kv, heads, page, name):
    lens, rows = BATCHES[name]
    g = torch.Generator(device=cuda).manual_seed(heads + page + len(lens))
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = make_cache(g, pool, page, kv, cuda)
    poison(cache, bt, lens)
    out, lse, want = run(cuda, cache, heads, bt, lens, rows, scale_of(kv, cuda), 0.05, g,
                         0 if rows is None else 3)
    check(out, lse, *want, max(lens))


@pytest.mark.parametrize("s", [-0.06, 0.0, 0.3])
@pytest.mark.parametrize("kv,heads", [("bf16", 24), ("bf16", 100), ("fp8", 8), ("fp8", 64)])
def test_decode_of_odd_arguments(cuda, kv, heads, s):
    """Masked pages (the first, some in between, all), lengths past the table, a bound that is too
    large, scales that are not positive."""
    page, lens, rows = 16, [500, 90, 64, 1000], [2, 1, 3, 1]
    g = torch.Generator(device=cuda).manual_seed(heads)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = make_cache(g, pool, page, kv, cuda)
    bt[0, :5], bt[0, 9], bt[0, 11:13], bt[1, 4] = -1, pool, -5, -1
    bt[2, :] = -1
    bt = bt[:, :40]  # the last sequence is longer than its table
    poison(cache, bt, lens)
    out, lse, want = run(cuda, cache, heads, bt, lens, rows, scale_of(kv, cuda), s, g, most=60)
    assert check(out, lse, *want, 1000).all()
    assert bool((out[3:6] == 0).all()) and bool(lse[:, 3:6].isneginf().all())


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("heads", [5, 64])
def test_decode_nan_stays_with_the_rows_that_see_it(cuda, kv, heads):
    page, lens, rows = 16, [70, 100, 45], [4, 4, 2]
    g = torch.Generator(device=cuda).manual_seed(heads)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = make_cache(g, pool, page, kv, cuda)
    t = lens[0] - 2  # seen by rows 2 and 3 of the first sequence
    p = int(bt[0, t // page])
    if kv == "fp8":
        cache.view(torch.uint8)[p, t % page, 5] = 0x7F
    else:
        cache[p, t % page, 5] = float("nan")
    out, lse, want = run(cuda, cache, heads, bt, lens, rows, scale_of(kv, cuda), 0.05, g)
    seen = check(out, lse, *want, 100)
    assert bool(out[2:4].isnan().all()) and not seen[2:4].any() and seen[4:].all() and seen[:2].all()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("heads", [16, 48])
@pytest.mark.parametrize("step", [1, 30, 37, 200])
def test_decode_of_growing_logits(cuda, kv, heads, step):
    """Greatest logits that grow by 2^30 and more (base 2: by 30) again and again, at other keys
    for other heads, over masked pages at the front."""
    page, lens = 16, [1000, 4001]
    g = torch.Generator(device=cuda).manual_seed(step)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = make_cache(g, pool, page, kv, cuda).float()
    # dim 512 + i of a key: how high its logit is for the heads that look there
    cache[:, :, 512:] = 0
    for b, n in enumerate(lens):
        for i in range(4):
            for j, t in enumerate(range(3 + 50 * i, n, step + 97 * (i + 1))):
                cache[int(bt[b, t // page]), t % page, 512 + i] = min(j + 1, 12)
    cache = cache.to(FP8 if kv == "fp8" else BF)
    scale = torch.ones(1, device=cuda) if kv == "fp8" else None
    bt[1, :3] = -1
    q = torch.zeros(2, heads, 576, dtype=BF, device=cuda)
    for h in range(heads):
        q[:, h, 512 + h % 4] = [32.0, 64.0, 24.0, 1.0][h // 4 % 4]
    out, lse, want = run(cuda, cache, heads, bt, lens, None, scale, 1.0, g, q=q)
    assert check(out, lse, *want, 4001, dims=1).all()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("sign", [1, -1])
def test_decode_of_great_magnitudes(cuda, kv, sign):
    """Logits of 2^90 and more, where the greatest alone counts, and nearly all of them equal."""
    page, n, heads = 16, 150, 40
    g = torch.Generator(device=cuda).manual_seed(7)
    cache = torch.randint(-8, 9, (10, page, 576), generator=g, device=cuda).float()
    cache[:, :, 512:] = 1.0
    cache[4, 3, 512:], cache[8, 9, 512:] = 4.0, 0.25
    cache = cache.to(FP8 if kv == "fp8" else BF)
    q = torch.zeros(1, heads, 576, dtype=BF, device=cuda)
    q[:, :, 512:] = sign * 2.0 ** 96
    bt = int32([list(range(10))], cuda)
    out, lse, _ = run(cuda, cache, heads, bt, [n], None, None, 0.1, g, q=q)
    row = cache[4, 3] if sign > 0 else cache[8, 9]
    assert torch.equal(out[0].float(), row[:512].float().expand(heads, 512))
    logit = 0.1 * sign * 2.0 ** 96 * 64 * (4.0 if sign > 0 else 0.25)
    assert torch.allclose(lse[:, 0].double(), torch.tensor(logit, device=cuda, dtype=torch.double),
                          rtol=1e-6)


@pytest.mark.parametrize("kv,power", [("bf16", 109), ("bf16", -100), ("bf16", -115), ("fp8", 110),
                                      ("fp8", -110)])
@pytest.mark.parametrize("heads", [16, 40])
@pytest.mark.parametrize("raised", [True, False])
def test_decode_of_great_and_small_values(cuda, kv, power, heads, raised):
    """Values of one sign next to 2^119 / 700 keys, and small ones, under logits that rise by nearly
    2^32 (base 2: by 32) behind the first 32 keys, or do not: what the sums come to is finite, and
    as exact as elsewhere.  Many rows, so that parts hold whole sequences.

    Small values: a weight is 2^-24 of the sum at least, a sum of n products is off by 2^-150 for
    each where they are no normal numbers, so the result by n 2^-126; and by half of bf16's least
    step, 2^-134."""
    from fastkernels_amd import ops

    n, page, batch = 700, 64, 600
    g = torch.Generator(device=cuda).manual_seed(heads)
    cache = torch.rand(11, page, 576, generator=g, device=cuda)
    scale = torch.tensor([2.0 ** power], device=cuda) if kv == "fp8" else None
    cache *= 440.0 if kv == "fp8" else 2.0 ** power
    cache[:, :, 512:] = 0
    if raised:
        cache[:, :, 512] = 22.0 if kv == "fp8" else 21.75
        cache[0, :32, 512] = 0
    cache = cache.to(FP8 if kv == "fp8" else BF)
    q = torch.zeros(batch, heads, 576, dtype=BF, device=cuda)
    q[:, :, 512] = 1
    s = 1.0 if kv == "bf16" else 2.0 ** -power
    out = torch.empty(batch, heads, 512, dtype=BF, device=cuda)
    lse = torch.empty(heads, batch, device=cuda)
    ops.latent_decode(out, q, cache, int32([list(range(11))] * batch, cuda),
                      int32([n] * batch, cuda), s, scale, lse=lse)
    want, mean, _, want_lse = ref.latent_decode(f64(q[:1]), dense(cache, scale),
                                                np.arange(11)[None], [n], s)
    assert np.isfinite(f64(out)).all()
    tol = attn_tolerance(want, mean, 22.0, 1) - 1e-30 + n * E24 * mean + \
        (n * 2.0 ** -126 if kv == "bf16" else 0) + 2.0 ** -134
    assert (np.abs(f64(out) - want) <= tol).all()
    tol = 4 * E24 * 22 + n * E24 + 8 * E24 * (1 + np.abs(want_lse))
    assert (np.abs(lse.double().cpu().numpy() - want_lse) <= tol).all()


@pytest.mark.parametrize("kv,heads,page,n,rows", [("bf16", 16, 16, 33001, 1), ("fp8", 128, 64, 20000, 2),
                                                  ("bf16", 40, 256, 9000, 5)])
def test_decode_of_one_long_sequence(cuda, kv, heads, page, n, rows):
    g = torch.Generator(device=cuda).manual_seed(n)
    bt, pool = tables(g, [-(-n // page)], cuda)
    cache = make_cache(g, pool, page, kv, cuda)
    out, lse, want = run(cuda, cache, heads, bt, [n], [rows], scale_of(kv, cuda), 0.05, g)
    assert check(out, lse, *want, n).all()


@pytest.mark.parametrize("batch", [257, 1500])
def test_decode_of_many_sequences(cuda, batch):
    g = torch.Generator(device=cuda).manual_seed(batch)
    lens = torch.randint(0, 40, (batch,), generator=g, device=cuda).tolist()
    rows = torch.randint(0, 3, (batch,), generator=g, device=cuda).tolist()
    bt, pool = tables(g, [-(-n // 16) for n in lens], cuda)
    cache = make_cache(g, pool, 16, "bf16", cuda)
    poison(cache, bt, lens)
    out, lse, want = run(cuda, cache, 4, bt, lens, rows, None, 0.05, g)
    assert check(out, lse, *want, 40).all()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_caches_past_4_gib(cuda, kv):
    """Pages whose byte offsets pass 32 bits, against the same pages in a small cache."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(3)
    page, dtype = 64, FP8 if kv == "fp8" else BF
    nb = (5 << 30) // (page * 576 * dtype.itemsize)
    at = [0, nb - 1, nb // 2 + 1, nb - 2]
    small, scale = make_cache(g, 4, page, kv, cuda), scale_of(kv, cuda)
    big = torch.empty(nb, page, 576, dtype=dtype, device=cuda)
    for i, p in enumerate(at):
        big[p] = small[i]
    latent = torch.randn(40, 512, generator=g, device=cuda).to(BF)
    key = torch.randn(40, 64, generator=g, device=cuda).to(BF)
    cos_sin = torch.randn(8, 64, generator=g, device=cuda)
    q = torch.randn(3, 16, 576, generator=g, device=cuda).to(BF)
    ctx, got = int32([250, 256, 100], cuda), []
    for cache, pages in ((small, [0, 1, 2, 3]), (big, at)):
        bt = int32([pages] * 3, cuda)
        slots = torch.tensor([p * page + 3 * i for p in pages for i in range(10)], device=cuda)
        ops.latent_norm_rope_store(cache, slots, slots * 0 + 3, latent, key, cos_sin, False,
                                   scale=scale)
        rows = torch.empty(256, 576, dtype=BF, device=cuda)
        ops.gather_latent(rows, cache, bt[1:2], int32([0, 256], cuda), scale)
        out = torch.empty(3, 16, 512, dtype=BF, device=cuda)
        ops.latent_decode(out, q, cache, bt, ctx, 0.05, scale)
        got.append((rows, out))
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("neox", [False, True])
def test_prompt_then_steps(cuda, kv, neox):
    """A latent attention layer: prompts stored in chunks and attended to in the expanded form, from
    the read-back; then steps in the absorbed form.  Both against float64 attention over the
    cache's rows; and a long context whose halves are attended to apart and merged."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(11)
    heads, page, s = 16, 16, 192 ** -0.5
    final, bounds = [130, 47, 300], ([64, 40, 200], [126, 41, 290])
    bt, pool = tables(g, [-(-n // page) for n in final], cuda)
    cache = torch.zeros(pool, page, 576, device=cuda).to(FP8 if kv == "fp8" else BF)
    scale = torch.tensor([0.02], device=cuda) if kv == "fp8" else None
    rope = load("rotary_emb", "RotaryEmbedding")(64, 512, 10000.0, is_neox_style=neox).to(cuda)
    norm = load("rms_norm", "RMSNorm")(512).to(cuda, BF)
    attn = load("latent_attn", "LatentAttnDecode")(heads, s)
    up = torch.randn(heads, 128, 512, generator=g, device=cuda) * 512 ** -0.5
    up_v = torch.randn(heads, 128, 512, generator=g, device=cuda) * 512 ** -0.5

    def store(old, new, query_rope, query_out=None):
        at = [(b, t) for b, (a, z) in enumerate(zip(old, new)) for t in range(a, z)]
        slots = torch.tensor([int(bt[b, t // page]) * page + t % page for b, t in at], device=cuda)
        proj = torch.randn(len(at), 576, generator=g, device=cuda).to(BF)
        pos = torch.tensor([t for _, t in at], device=cuda)
        return rope.forward_store_latent(pos, query_rope, proj[:, :512], proj[:, 512:], cache, slots,
                                         norm, query_out, scale)

    old = [0, 0, 0]
    for new in bounds:
        n = [z - a for a, z in zip(old, new)]
        q = torch.randn(sum(n), heads, 192, generator=g, device=cuda).to(BF)
        store(old, new, q[:, :, 128:])  # rotated in place
        cu_q, cu_k = cu_of(n, cuda), cu_of(new, cuda)
        rows = torch.empty(sum(new), 576, dtype=BF, device=cuda)
        ops.gather_latent(rows, cache, bt, cu_k, scale)
        c = rows[:, :512].float()
        key = torch.empty(sum(new), heads, 192, dtype=BF, device=cuda)
        key[:, :, :128] = (c @ up.flatten(0, 1).t()).unflatten(1, (heads, 128))
        key[:, :, 128:] = rows[:, None, 512:]
        value = (c @ up_v.flatten(0, 1).t()).unflatten(1, (heads, 128)).to(BF)
        out = torch.empty(sum(n), heads, 128, dtype=BF, device=cuda)
        ops.varlen_prefill(out, q, key, value, cu_q, cu_k, max(n), s, max_seqlen_k=max(new))
        k64, v64, q64 = f64(key), f64(value), f64(q)
        for b in range(3):
            for i in range(n[b]):
                t, z = int(cu_q[b]) + i, int(cu_k[b]) + new[b] - n[b] + i + 1
                x = s * np.matmul(k64[int(cu_k[b]):z].transpose(1, 0, 2), q64[t][:, :, None])[:, :, 0]
                w = np.exp(x - x.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                v = v64[int(cu_k[b]):z].transpose(1, 0, 2)
                want = np.matmul(w[:, None], v)[:, 0]
                mean = np.matmul(w[:, None], np.abs(v))[:, 0]
                tol = attn_tolerance(want, mean, np.abs(x).max() + 60, 192) + 300 * E24 * mean
                assert (np.abs(f64(out[t]) - want) <= tol).all()
        old = new
    for rows in ([1, 1, 1], [3, 1, 4], [0, 4, 2]):
        new = [a + r for a, r in zip(old, rows)]
        q = torch.randn(sum(rows), heads, 576, generator=g, device=cuda).to(BF)
        raw = torch.randn(sum(rows), heads, 64, generator=g, device=cuda).to(BF)
        store(old, new, raw, q[:, :, 512:])
        cu = cu_of(rows, cuda)
        got = attn(q, cache, int32(new, cuda), bt, scale, cu, 4)
        want = ref.latent_decode(f64(q), dense(cache, scale), bt.cpu().numpy(), new, s,
                                 cu_seqlens_q=cu.tolist())
        assert check(got, None, *want, 300).all()
        old = new
    # the first 96 keys and the others apart, merged by their log-sum-exps
    b, q = 2, torch.randn(1, heads, 576, generator=g, device=cuda).to(BF)
    o = [torch.empty(1, heads, 512, dtype=BF, device=cuda) for _ in range(3)]
    lse = [torch.empty(heads, 1, device=cuda) for _ in range(2)]
    ops.latent_decode(o[0], q, cache, bt[b:b + 1, :6], int32([96], cuda), s, scale, lse=lse[0])
    ops.latent_decode(o[1], q, cache, bt[b:b + 1, 6:], int32([old[b] - 96], cuda), s, scale, lse=lse[1])
    ops.merge_attn_states(o[2], o[0], lse[0], o[1], lse[1])
    out, mean, mag, _ = ref.latent_decode(f64(q), dense(cache, scale), bt[b:b + 1].cpu().numpy(),
                                          [old[b]], s)
    tol = 2 * attn_tolerance(out, mean, mag, 576) + U * mean  # the parts' roundings, and the result's
    assert (np.abs(f64(o[2]) - out) <= tol).all()


@pytest.mark.parametrize("kv,heads", [("bf16", 128), ("fp8", 16)])
def test_in_graphs(cuda, kv, heads):
    """Two steps captured on one module, replayed in turn with eager work in between as the
    lengths grow, against the eager result."""
    g = torch.Generator(device=cuda).manual_seed(4)
    cache, scale = make_cache(g, 200, 16, kv, cuda), scale_of(kv, cuda)
    bt = torch.randperm(200, generator=g, device=cuda).to(torch.int32).view(4, 50)
    q = torch.randn(8, heads, 576, generator=g, device=cuda).to(BF)
    proj = torch.randn(4, 576, generator=g, device=cuda).to(BF)
    raw = torch.randn(4, heads, 64, generator=g, device=cuda).to(BF)
    ctx, slots = int32([1, 20, 300, 0], cuda), int32([0, 1, 2, 3], cuda)
    pos, cu = torch.arange(4, device=cuda), int32([0, 2, 5, 6, 8], cuda)
    rope = load("rotary_emb", "RotaryEmbedding")(64, 512, 10000.0).to(cuda)
    attn = load("latent_attn", "LatentAttnDecode")(heads, 0.05)

    def one():
        rope.forward_store_latent(pos, raw, proj[:, :512], proj[:, 512:], cache, slots,
                                  query_out=q[:4, :, 512:], cache_scale=scale)
        return attn(q[:4], cache, ctx, bt, scale)

    def drafts():
        return attn(q, cache, ctx, bt, scale, cu, 3)

    one(), drafts()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (one, drafts):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(f())
        graphs.append(graph)
    for i, lens in enumerate(([1, 20, 300, 0], [800, 0, 2, 799], [33, 64, 65, 500])):
        ctx.copy_(int32(lens, cuda))
        pos.copy_(torch.tensor([i, 3, 500, 511], device=cuda))
        slots.copy_(int32([7 * i, 300 + i, -1, 900 - i], cuda))
        for graph in graphs:  # (the store first; stored again, the rows stay as they are)
            graph.replay()
        got = [o.clone() for o in outs]
        want = [one(), drafts()]
        torch.cuda.synchronize()
        for graph in graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(got, want, outs):
            assert torch.equal(a, b) and torch.equal(c, b)


def test_streams_and_compile(cuda):
    """Calls that overlap on two streams, and under torch.compile: the same bits."""
    g = torch.Generator(device=cuda).manual_seed(5)
    cache = make_cache(g, 100, 64, "bf16", cuda)
    bt = torch.randperm(100, generator=g, device=cuda).to(torch.int32).view(4, 25)
    attn = load("latent_attn", "LatentAttnDecode")(128, 0.05)
    q = torch.randn(4, 128, 576, generator=g, device=cuda).to(BF)
    ctxs = [int32(x, cuda) for x in ([1500, 3, 900, 64], [10, 1600, 1, 0])]

    def step(q, ctx):
        return attn(q, cache, ctx, bt)

    want = [step(q, c) for c in ctxs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ctxs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(q, ctxs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for r, w in zip(got, want) for x in r)
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    for c, w in zip(ctxs, want):
        assert torch.equal(compiled(q, c), w)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_compiled_step(cuda, kv):
    """A store into a view of the queries and the attention behind it under torch.compile: the bits
    of the eager step, in the cache, the queries and the result."""
    g = torch.Generator(device=cuda).manual_seed(6)
    cache, scale = make_cache(g, 20, 16, kv, cuda), scale_of(kv, cuda)
    bt = torch.randperm(20, generator=g, device=cuda).to(torch.int32).view(2, 10)
    q = torch.randn(2, 16, 576, generator=g, device=cuda).to(BF)
    raw = torch.randn(2, 16, 64, generator=g, device=cuda).to(BF)
    proj = torch.randn(2, 576, generator=g, device=cuda).to(BF)
    pos, ctx = torch.tensor([8, 100], device=cuda), int32([9, 101], cuda)
    slots = torch.stack([bt[0, 0] * 16 + 8, bt[1, 6] * 16 + 4]).long()
    rope = load("rotary_emb", "RotaryEmbedding")(64, 512, 10000.0).to(cuda)
    norm = load("rms_norm", "RMSNorm")(512).to(cuda, BF)
    attn = load("latent_attn", "LatentAttnDecode")(16, 0.05)

    def step(cache, q):
        rope.forward_store_latent(pos, raw, proj[:, :512], proj[:, 512:], cache, slots, norm,
                                  q[:, :, 512:], scale)
        return attn(q, cache, ctx, bt, scale)

    got = []
    for f in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        c, x = cache.clone(), q.clone()
        out = f(c, x)
        got.append((out, x, c.view(torch.uint8) if kv == "fp8" else c.view(torch.int16)))
    assert not torch.equal(got[0][1], q)
    for a, b in zip(*got):
        assert torch.equal(a, b)
