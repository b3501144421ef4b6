"""The 4-bit cache (GPU): store, read-back and decode attention against float64 definitions
(``oracle.small_cache``), and a run of them together.

Tolerances.  Scales and codes are exact, and so is the read-back (a code times a power of two is a
bf16 value).  The attention's operands are exact too: its output differs as that of a bf16 cache
does (each weight rounded to bf16, the result once more, the logits' float32 sums), and by the
float32 sums over the keys, 2^-24 of the average of |v| for each of them.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import small_cache as ref
from test_gpu_sparse import attn_tolerance, cu_of, f64, int32, load, tables

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def check(out, want, mean, mag, keys, factor=1.0):
    """NaN in `want`: not compared.  Returns where it is a number."""
    got, seen = f64(out), ~np.isnan(want)
    assert np.isfinite(got[seen]).all()
    tol = factor * attn_tolerance(want, mean, mag, want.shape[2]) + keys * 2.0 ** -24 * mean
    err = (np.abs(got - want) - tol)[seen]
    assert err.size == 0 or err.max() <= 0, f"beyond the tolerance by {err.max()}"
    return seen


def random_cache(g, nb, page, hk, d, dev):
    """Random codes under scales of 2^-4 to 2^1."""
    from fastkernels_amd import ops

    c = ops.new_mxfp4_cache(nb, page, hk, d, dev)
    for t, (lo, hi) in zip(c, ((0, 256), (0, 256), (123, 129), (123, 129))):
        t.copy_(torch.randint(lo, hi, t.shape, generator=g, device=dev))
    return c


def values(cache):
    return ref.mxfp4_cache_values(*(t.cpu().numpy() for t in cache))


def poison(cache, bt, lens, page):
    """NaN scales wherever no sequence has a token."""
    nb = cache.k_scales.shape[0]
    used = torch.zeros(nb, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(-(-n // page)):
            if int(bt[b, j]) >= 0:
                used[int(bt[b, j]), :min(page, n - j * page)] = True
    free = (~used).to(cache.k_scales.device)[:, None, None].expand(cache.k_scales.shape)
    cache.k_scales[free] = 255
    cache.v_scales[free] = 255


# ---------------------------------------------------------------------------
# store and read-back
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, BF])
@pytest.mark.parametrize("hk,d,page,n,i64", [(8, 128, 16, 37, False), (1, 64, 32, 1, True),
                                             (3, 256, 16, 300, True), (5, 64, 256, 65, False),
                                             (20, 128, 64, 9, True)])
def test_store(cuda, dtype, hk, d, page, n, i64):
    """Every slot's scales and codes, skipped and out-of-range slots, rows inside wider ones, and
    everything else left as it was."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(n + d)
    nb = -(-n // page) + 2
    cache = random_cache(g, nb, page, hk, d, cuda)
    before = [t.clone() for t in cache]
    off = 3 if n % 2 else 8  # an odd offset: rows that are not 16-byte aligned
    wide = torch.randn(n, 2 * hk * d + 2 * off, generator=g, device=cuda)
    # blocks of all magnitudes that the type has, zeros among them
    mag = torch.randint(-130, 100, (n, wide.shape[1] // 32 + 1), generator=g, device=cuda)
    if dtype == torch.float16:
        mag = mag.clamp(-22, 13)
    wide *= (2.0 ** mag.double()).repeat_interleave(32, 1)[:, :wide.shape[1]].float()
    wide[0, off:off + 64] = 0
    wide = wide.to(dtype)
    key = wide[:, off:off + hk * d].unflatten(1, (hk, d))
    value = wide[:, off + hk * d:off + 2 * hk * d].unflatten(1, (hk, d))
    if n > 4:
        key[1, 0, 3], value[2, hk - 1, d - 1], value[3, 0, 40] = float("nan"), float("inf"), \
            float("-inf")
    slots = torch.randperm(nb * page, generator=g, device=cuda)[:n]
    if n > 8:
        slots[4], slots[6], slots[7] = -1, nb * page, -7
    if n > 8 and i64:
        slots[8] = (1 << 40) + 3
    ops.store_kvcache_mxfp4(key, value, *cache, slots if i64 else slots.to(torch.int32))
    k, v = (x.copy() for x in ref.mxfp4_cache_values(*(t.cpu().numpy() for t in before)))
    wide64 = [x.double().cpu().numpy() for x in (key, value)]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < nb * page:
            for c, x in zip((k, v), wide64):
                c[s // page, s % page] = ref.mxfp4_values(*ref.mxfp4_blocks(x[t]))
    got = values(cache)
    for name, a, b in zip("kv", got, (k, v)):
        assert np.array_equal(a, b, equal_nan=True), name
    for t, s in enumerate(slots.tolist()):  # the scales themselves, where zeros would hide them
        if 0 <= s < nb * page:
            for c, x in zip((cache.k_scales, cache.v_scales), wide64):
                want = ref.mxfp4_blocks(x[t])[0]
                assert np.array_equal(c[s // page, :, :, s % page].cpu().numpy(), want)


def test_store_every_rounding(cuda):
    """All bf16 magnitudes beside a greatest value that fixes the scale, of both signs."""
    from fastkernels_amd import ops

    x = (torch.arange(1 << 15, dtype=torch.int32, device=cuda) << 16).view(torch.float32)
    x = x[x.isfinite()]
    rows = []
    for top in (1.0, 1.75, 3.0, 2.0 ** -126, 2.0 ** -133, 3.0e38):
        y = x[x <= top]
        y = torch.cat([y, y.new_zeros(-y.numel() % 31)]).view(-1, 31)
        rows.append(torch.cat([y, y.new_full((y.shape[0], 1), top)], 1))
    x = torch.cat(rows)
    x = torch.cat([x, -x])
    n = -(-x.shape[0] // 2)
    key = torch.cat([x, x.new_zeros(2 * n - x.shape[0], 32)]).view(n, 1, 64).to(BF)
    cache = ops.new_mxfp4_cache(-(-n // 256), 256, 1, 64, cuda)
    ops.store_kvcache_mxfp4(key, key, *cache, torch.arange(n, device=cuda))
    want = ref.mxfp4_values(*ref.mxfp4_blocks(f64(key)))[:, 0]
    for got in values(cache):
        assert np.array_equal(got.reshape(-1, 64)[:n], want)


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_greatest_magnitudes_stay_finite(cuda, dtype, d):
    """Blocks whose greatest value is next to the type's end, of both signs: what is read back is
    finite, and what the definition says."""
    from fastkernels_amd import ops

    tops = [1.2 * 2.0 ** 127, 1.74 * 2.0 ** 127, 1.75 * 2.0 ** 127, 1.9 * 2.0 ** 127, 3.0e38,
            float(torch.finfo(dtype).max), 1.74 * 2.0 ** 126, 1.75 * 2.0 ** 126]
    n = len(tops)
    x = torch.rand(n, 1, d // 32, 32, device=cuda) * 1.5
    x[..., 5], x[..., 6] = 1.0, -1.0
    x = (x.clamp(-1, 1) * torch.tensor(tops, device=cuda).view(n, 1, 1, 1)).flatten(2).to(dtype)
    assert bool(x.isfinite().all())
    cache = ops.new_mxfp4_cache(1, 16, 1, d, cuda)
    ops.store_kvcache_mxfp4(x, -x, *cache, torch.arange(n, device=cuda))
    key = torch.empty(n, 1, d, dtype=BF, device=cuda)
    value = torch.empty_like(key)
    ops.gather_kvcache_mxfp4(key, value, *cache, int32([[0]], cuda), int32([0, n], cuda))
    want = ref.mxfp4_values(*ref.mxfp4_blocks(x.double().cpu().numpy()))
    assert np.isfinite(f64(key)).all() and np.isfinite(f64(value)).all()
    assert np.array_equal(f64(key), want) and np.array_equal(f64(value), -want)


@pytest.mark.parametrize("hk,d,page,lens", [(8, 128, 16, [17, 0, 1, 300]), (1, 64, 32, [1]),
                                            (3, 256, 64, [64, 65, 200]),
                                            (20, 64, 256, [255, 257, 0]), (40, 128, 16, [33]),
                                            (2, 64, 16, [1500, 0, 1601]),
                                            (1, 128, 64, [9000, 1, 8001])])
def test_gather(cuda, hk, d, page, lens):
    """The rows in between, those of masked pages zero, those of no sequence left alone."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(hk + d)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = random_cache(g, pool, page, hk, d, cuda)
    poison(cache, bt, lens, page)
    longest = max(range(len(lens)), key=lambda b: lens[b])
    if lens[longest] > page:
        bt[longest, 0] = -1
    if len(lens) > 2 and lens[-1] > page:
        bt[-1, 1] = pool  # outside the cache
    cu = cu_of(lens, cuda) + 2
    total = sum(lens) + 7
    wide = torch.full((total, 2 * hk * d + 16), 9.0, dtype=BF, device=cuda)
    key = wide[:, :hk * d].unflatten(1, (hk, d))
    value = wide[:, hk * d + 8:2 * hk * d + 8].unflatten(1, (hk, d))
    ops.gather_kvcache_mxfp4(key, value, *cache, bt, cu)
    for got, c in zip((key, value), values(cache)):
        want = ref.gather(c, bt.cpu().numpy(), cu.tolist(), total)
        want[:2], want[2 + sum(lens):] = 9.0, 9.0
        assert np.array_equal(f64(got), want)
    assert bool((wide[:, hk * d:hk * d + 8] == 9.0).all())
    assert bool((wide[:, 2 * hk * d + 8:] == 9.0).all())


@pytest.mark.parametrize("d", [64, 128, 256])
def test_gather_every_scale(cuda, d):
    """All codes under all scale bytes: exact, from 2^-128 to the greatest bf16, and infinities for
    what is beyond."""
    from fastkernels_amd import ops

    cache = ops.new_mxfp4_cache(1, 256, 1, d, cuda)
    code = torch.arange(16, dtype=torch.uint8, device=cuda)
    pairs = (code[0::2] | code[1::2] << 4).repeat(d // 16)
    cache.k_cache[:] = pairs
    cache.v_cache[:] = pairs.view(1, 1, 1, 16, 1, d // 32)
    cache.k_scales[:] = torch.arange(256, dtype=torch.uint8, device=cuda)
    cache.v_scales[:] = torch.arange(256, dtype=torch.uint8, device=cuda).flip(0)
    key = torch.empty(256, 1, d, dtype=BF, device=cuda)
    value = torch.empty_like(key)
    ops.gather_kvcache_mxfp4(key, value, *cache, int32([[0]], cuda), int32([0, 256], cuda))
    for got, want in zip((key, value), values(cache)):
        want = want.reshape(256, 1, d)
        big = np.abs(want) >= 2.0 ** 128
        assert np.array_equal(big.any((1, 2)), np.isin(want[:, 0, 1], [2.0 ** 125, 2.0 ** 126]))
        want[big] = np.copysign(np.inf, want[big])
        assert np.array_equal(f64(got), want, equal_nan=True)


# ---------------------------------------------------------------------------
# decode attention
# ---------------------------------------------------------------------------
SHAPES = [(32, 8, 128, 16), (16, 2, 256, 16), (20, 20, 64, 32), (64, 8, 128, 64), (64, 8, 64, 256),
          (8, 1, 128, 16), (40, 2, 256, 128), (34, 2, 128, 16), (128, 1, 64, 16)]
BATCHES = {
    "one": ([1], None), "zeros": ([0, 0], None), "short": ([31, 33, 0, 1, 16], None),
    "mixed": ([700, 5, 0, 1300, 64, 63, 65], None),
    "drafts": ([300, 3, 40, 1, 900], [4, 3, 1, 1, 5]),
    "holes": ([300, 2, 0, 70], [0, 3, 2, 2]),  # more rows than tokens: the first see none
    "many": ([17 * i % 90 for i in range(70)], None),
    "negative": ([40, -3, 20], None),  # a length below zero is none
}


@pytest.mark.parametrize("name", list(BATCHES))
@pytest.mark.parametrize("hq,hk,d,page", SHAPES)
def test_decode(cuda, hq, hk, d, page, name):
    from fastkernels_amd import ops

    lens, rows = BATCHES[name]
    g = torch.Generator(device=cuda).manual_seed(hq + d + page + len(lens))
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = random_cache(g, pool, page, hk, d, cuda)
    poison(cache, bt, lens, page)
    n = len(lens) if rows is None else sum(rows)
    spare = 0 if rows is None else 3
    wide = torch.randn(n + spare, hq + 1, d, generator=g, device=cuda).to(BF)
    q = wide[:, :hq]
    out = torch.full((n + spare, hq + 2, d), 9.0, dtype=BF, device=cuda)
    cu = None if rows is None else cu_of(rows, cuda)
    ops.mxfp4_paged_decode(out[:, :hq], q, *cache, bt, int32(lens, cuda), d ** -0.5,
                           cu_seqlens_q=cu, max_seqlen_q=None if rows is None else max(rows))
    want, mean, mag = ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), lens, d ** -0.5,
                                       cu_seqlens_q=None if cu is None else cu.tolist())
    check(out[:n, :hq], want[:n], mean[:n], mag[:n], max(lens))
    assert bool((out[:, hq:] == 9.0).all()) and bool((out[n:] == 9.0).all())


@pytest.mark.parametrize("window", [0, 1, 15, 40, 600, 100000])
@pytest.mark.parametrize("hq,hk,d,page,rows", [(32, 8, 128, 16, None), (24, 2, 64, 32, [3, 1, 4]),
                                               (12, 4, 256, 16, [2, 5, 1]),
                                               (64, 8, 128, 64, [4, 4, 4])])
def test_decode_windows_and_sinks(cuda, hq, hk, d, page, rows, window):
    """Windows over contexts whose other keys are NaN, with sinks, among them -inf."""
    from fastkernels_amd import ops

    lens = [900, 130, 2500]
    g = torch.Generator(device=cuda).manual_seed(window % 97 + d)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = random_cache(g, pool, page, hk, d, cuda)
    poison(cache, bt, lens, page)
    most = 1 if rows is None else max(rows)
    for b, n in enumerate(lens):  # keys before every row's window
        for t in range(max(0, n - (1 if rows is None else rows[b]) - window)):
            p = int(bt[b, t // page])
            cache.k_scales[p, :, :, t % page] = 255
            cache.v_scales[p, :, :, t % page] = 255
    n = 3 if rows is None else sum(rows)
    q = torch.randn(n, hq, d, generator=g, device=cuda).to(BF)
    sinks = torch.randn(hq, generator=g, device=cuda) * 3
    sinks[1], sinks[2] = float("-inf"), 40.0
    cu = None if rows is None else cu_of(rows, cuda)
    out = torch.empty_like(q)
    ops.mxfp4_paged_decode(out, q, *cache, bt, int32(lens, cuda), d ** -0.5, window, sinks, cu,
                           most)
    want = ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), lens, d ** -0.5, window,
                            f64(sinks), None if cu is None else cu.tolist())
    assert check(out, *want, min(window + 1, 2500)).all()


@pytest.mark.parametrize("scale", [-0.11, 0.0, 0.3])
@pytest.mark.parametrize("hq,hk,d", [(16, 2, 128), (9, 3, 64), (16, 1, 256)])
def test_decode_of_odd_arguments(cuda, hq, hk, d, scale):
    """Masked pages (the first, some in between, all), lengths past the table, a bound that is too
    large, scales that are not positive."""
    from fastkernels_amd import ops

    page, lens, rows = 16, [500, 90, 64, 1000], [2, 1, 3, 1]
    g = torch.Generator(device=cuda).manual_seed(d)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = random_cache(g, pool, page, hk, d, cuda)
    poison(cache, bt, lens, page)
    bt[0, :5], bt[0, 9], bt[0, 11:13], bt[1, 4] = -1, pool, -5, -1
    bt[2, :] = -1
    bt = bt[:, :40]  # the last sequence is longer than its table
    q = torch.randn(7, hq, d, generator=g, device=cuda).to(BF)
    out, cu = torch.empty_like(q), cu_of(rows, cuda)
    ops.mxfp4_paged_decode(out, q, *cache, bt, int32(lens, cuda), scale, cu_seqlens_q=cu,
                           max_seqlen_q=60)
    want = ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), lens, scale,
                            cu_seqlens_q=cu.tolist())
    assert check(out, *want, 1000).all()
    assert bool((out[3:6] == 0).all())


@pytest.mark.parametrize("hq,hk,d", [(8, 2, 128), (16, 1, 64), (8, 2, 256), (24, 1, 128)])
def test_decode_nan_stays_with_the_rows_that_see_it(cuda, hq, hk, d):
    """A NaN block of V shows in its dims, one of K in its heads, of the rows that see it."""
    from fastkernels_amd import ops

    page, lens, rows = 16, [70, 100, 45], [4, 4, 2]
    g = torch.Generator(device=cuda).manual_seed(d)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = random_cache(g, pool, page, hk, d, cuda)
    q = torch.randn(10, hq, d, generator=g, device=cuda).to(BF)
    t = lens[0] - 2  # seen by rows 2 and 3 of the first sequence
    cache.v_scales[int(bt[0, t // page]), 0, 1, t % page] = 255
    t = lens[1] - 1  # seen by the last row of the second
    cache.k_scales[int(bt[1, t // page]), hk - 1, 0, t % page] = 255
    out, cu = torch.empty_like(q), cu_of(rows, cuda)
    ops.mxfp4_paged_decode(out, q, *cache, bt, int32(lens, cuda), d ** -0.5, cu_seqlens_q=cu,
                           max_seqlen_q=4)
    want = ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), lens, d ** -0.5,
                            cu_seqlens_q=cu.tolist())
    seen = check(out, *want, 100)
    assert np.array_equal(np.isnan(f64(out)), ~seen)
    gqa, nan = hq // hk, np.zeros(out.shape, bool)
    nan[2:4, :gqa, 32:64] = True
    nan[7, hq - gqa:] = True
    assert np.array_equal(~seen, nan)


@pytest.mark.parametrize("byte,code", [(253, 6), (253, 15), (254, 4), (254, 14)])
@pytest.mark.parametrize("hq,hk,d,page", [(8, 2, 128, 16), (16, 1, 64, 64), (8, 2, 256, 16),
                                          (24, 1, 128, 32)])
def test_decode_infinities_stay_with_the_rows_that_see_them(cuda, hq, hk, d, page, byte, code):
    """A value of 2^128 or more in V, which bf16 does not have, at keys that the last rows of a
    sequence see: infinite there, in its dim alone."""
    from fastkernels_amd import ops

    lens, rows = [70, 100, 45], [4, 4, 2]
    g = torch.Generator(device=cuda).manual_seed(d)
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = random_cache(g, pool, page, hk, d, cuda)
    q = torch.randn(10, hq, d, generator=g, device=cuda).to(BF)
    t = lens[0] - 2  # seen by rows 2 and 3 of the first sequence
    p, s = int(bt[0, t // page]), t % page
    cache.v_scales[p, 0, 1, s] = byte  # of dims 32 .. 63: their codes 0, but for dim 32's
    first = 32 // (d // 16)
    cache.v_cache[p, 0, s // 4, first:2 * first, s % 4] = 0
    cache.v_cache[p, 0, s // 4, first, s % 4, 0] = code
    assert abs(values(cache)[1][p, s, 0, 32]) >= 2.0 ** 128
    out, cu = torch.empty_like(q), cu_of(rows, cuda)
    ops.mxfp4_paged_decode(out, q, *cache, bt, int32(lens, cuda), d ** -0.5, cu_seqlens_q=cu,
                           max_seqlen_q=4)
    want, mean, mag = ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), lens, d ** -0.5,
                                       cu_seqlens_q=cu.tolist())
    inf = np.zeros(out.shape, bool)
    inf[2:4, :hq // hk, 32] = True
    assert np.array_equal(f64(out)[inf], np.where(code & 8, -np.inf, np.inf).repeat(inf.sum()))
    want[inf] = np.nan
    assert np.array_equal(check(out, want, mean, mag, 100), ~inf)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("power", [96, -100])
def test_decode_of_great_and_small_magnitudes(cuda, d, power):
    """Logits of 2^90 and more, where the greatest alone counts; and values of 2^-100."""
    from fastkernels_amd import ops

    hq, hk, page, n = 4, 2, 16, 150
    g = torch.Generator(device=cuda).manual_seed(d)
    cache = random_cache(g, 10, page, hk, d, cuda)
    bt, ctx = int32([list(range(10))] * 2, cuda), int32([n, n], cuda)
    q = torch.randn(2, hq, d, generator=g, device=cuda).to(BF)
    if power > 0:
        cache.k_cache.fill_(0x22)  # all ones
        cache.k_scales.fill_(127)
        q = (q.float().abs() + 0.1) * 2.0 ** power
        q[1] *= -1
        q = q.to(BF)
        cache.k_scales[4, :, :, 3] = 129
        cache.k_scales[8, :, :, 9] = 125
        v = values(cache)[1]
        want = torch.tensor(np.stack([v[4, 3], v[8, 9]])).repeat_interleave(hq // hk, 1)
    else:
        cache.v_scales.fill_(127 + power)
    out = torch.empty_like(q)
    ops.mxfp4_paged_decode(out, q, *cache, bt, ctx, 0.1)
    if power > 0:
        assert torch.equal(out.cpu().double(), want)
    else:
        check(out, *ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), [n, n], 0.1), n)


@pytest.mark.parametrize("hq,hk,d,page,n,rows", [(32, 8, 128, 16, 33001, 1), (8, 8, 64, 256, 20000, 2),
                                                 (16, 2, 256, 64, 9000, 3)])
def test_decode_of_one_long_sequence(cuda, hq, hk, d, page, n, rows):
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(n)
    bt, pool = tables(g, [-(-n // page)], cuda)
    cache = random_cache(g, pool, page, hk, d, cuda)
    q = torch.randn(rows, hq, d, generator=g, device=cuda).to(BF)
    out, cu = torch.empty_like(q), int32([0, rows], cuda)
    ops.mxfp4_paged_decode(out, q, *cache, bt, int32([n], cuda), d ** -0.5, cu_seqlens_q=cu,
                           max_seqlen_q=rows)
    want = ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), [n], d ** -0.5,
                            cu_seqlens_q=[0, rows])
    assert check(out, *want, n).all()


@pytest.mark.parametrize("batch", [257, 1500])
def test_decode_of_many_sequences(cuda, batch):
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(batch)
    hq, hk, d, page = 4, 1, 64, 16
    lens = torch.randint(0, 40, (batch,), generator=g, device=cuda).tolist()
    rows = torch.randint(0, 4, (batch,), generator=g, device=cuda).tolist()
    bt, pool = tables(g, [-(-n // page) for n in lens], cuda)
    cache = random_cache(g, pool, page, hk, d, cuda)
    poison(cache, bt, lens, page)
    q = torch.randn(sum(rows), hq, d, generator=g, device=cuda).to(BF)
    out, cu = torch.full_like(q, 9.0), cu_of(rows, cuda)
    ops.mxfp4_paged_decode(out, q, *cache, bt, int32(lens, cuda), d ** -0.5, cu_seqlens_q=cu,
                           max_seqlen_q=3)
    want = ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), lens, d ** -0.5,
                            cu_seqlens_q=cu.tolist())
    assert check(out, *want, 40).all()


def test_caches_past_4_gib(cuda):
    """Pages whose byte offsets pass 32 bits, against the same pages in a small cache."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(3)
    hq, hk, d, page = 16, 8, 128, 256
    nb = (5 << 30) // (page * hk * d // 2)
    at = [0, nb - 1, nb // 2 + 1, nb - 2]
    small, big = random_cache(g, 4, page, hk, d, cuda), ops.new_mxfp4_cache(nb, page, hk, d, cuda)
    new = torch.randn(40, hk, d, generator=g, device=cuda).to(BF)
    q = torch.randn(3, hq, d, generator=g, device=cuda).to(BF)
    ctx, got = int32([1000, 1024, 700], cuda), []
    for x, y in zip(big, small):
        for i, p in enumerate(at):
            x[p] = y[i]
    for cache, pages in ((small, [0, 1, 2, 3]), (big, at)):
        bt = int32([pages] * 3, cuda)
        slots = torch.tensor([p * page + 3 * i for p in pages for i in range(10)], device=cuda)
        ops.store_kvcache_mxfp4(new, new.flip(0), *cache, slots)
        key = torch.empty(1024, hk, d, dtype=BF, device=cuda)
        value, out = torch.empty_like(key), torch.empty_like(q)
        ops.gather_kvcache_mxfp4(key, value, *cache, bt[1:2], int32([0, 1024], cuda))
        ops.mxfp4_paged_decode(out, q, *cache, bt, ctx, d ** -0.5)
        got.append((key, value, out))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("hk,d", [(8, 128), (1, 64)])
def test_decode_of_small_pages_past_4_gib(cuda, hk, d):
    """Pages of 16 tokens, two of them to a step, on both sides of the byte offset 2^32."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(4)
    nb = (5 << 30) // (16 * hk * d // 2)
    at = [nb - 1, 0, nb * 4 // 5 - 1, nb * 4 // 5 + 1, nb // 2, nb - 2]
    small, big = random_cache(g, 6, 16, hk, d, cuda), ops.new_mxfp4_cache(nb, 16, hk, d, cuda)
    for x, y in zip(big, small):
        for i, p in enumerate(at):
            x[p] = y[i]
    q = torch.randn(3, 2 * hk, d, generator=g, device=cuda).to(BF)
    got = []
    for cache, pages in ((small, range(6)), (big, at)):
        out = torch.empty_like(q)
        ops.mxfp4_paged_decode(out, q, *cache, int32([list(pages)] * 3, cuda),
                               int32([96, 33, 70], cuda), d ** -0.5)
        got.append(out)
    assert torch.equal(*got)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("hq,hk,d,page", [(32, 8, 128, 16), (16, 2, 256, 64), (8, 8, 64, 16)])
def test_prompt_in_chunks_then_steps(cuda, hq, hk, d, page):
    """Prompts stored in two chunks, the second attending to the read-back of its context; then
    decode steps, one of them checking drafted tokens: everything against the float64 attention
    over the cache's values."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(d)
    final, chunks = [130, 47, 300], ([64, 40, 200], [126, 41, 290])
    bt, pool = tables(g, [-(-n // page) for n in final], cuda)
    cache = ops.new_mxfp4_cache(pool, page, hk, d, cuda)
    put = load("store_kvcache", "StoreKVCacheMxfp4")()
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)
    scale = d ** -0.5

    def store(old, new):
        at = [(b, t) for b, (a, z) in enumerate(zip(old, new)) for t in range(a, z)]
        slots = torch.tensor([int(bt[b, t // page]) * page + t % page for b, t in at], device=cuda)
        kv = torch.randn(2, len(at), hk, d, generator=g, device=cuda).to(BF)
        put(kv[0], kv[1], cache, slots)

    old = [0, 0, 0]
    for new in chunks:
        store(old, new)
        n = [z - a for a, z in zip(old, new)]
        q = torch.randn(sum(n), hq, d, generator=g, device=cuda).to(BF)
        cu_q, cu_k = cu_of(n, cuda), cu_of(new, cuda)
        key = torch.empty(sum(new), hk, d, dtype=BF, device=cuda)
        value = torch.empty_like(key)
        ops.gather_kvcache_mxfp4(key, value, *cache, bt, cu_k)
        out = torch.empty_like(q)
        ops.varlen_prefill(out, q, key, value, cu_q, cu_k, max(n), scale, max_seqlen_k=max(new))
        want = ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), new, scale,
                                cu_seqlens_q=cu_q.tolist())
        check(out, *want, 300)
        # the last rows of the chunk by the decode kernel
        last = min(min(n), 4)
        pick = torch.cat([torch.arange(z - last, z) for z in np.cumsum(n).tolist()]).to(cuda)
        got = attn.forward_mxfp4(q[pick].flatten(1), cache, int32(new, cuda),
                                 cu_of([last] * 3, cuda), last, block_table=bt)
        check(got, *(x[pick.cpu().numpy()] for x in want), 300)
        old = new
    for rows in ([1, 1, 1], [3, 1, 4], [0, 4, 2]):
        new = [a + r for a, r in zip(old, rows)]
        store(old, new)
        q = torch.randn(sum(rows), hq, d, generator=g, device=cuda).to(BF)
        cu = cu_of(rows, cuda)
        got = attn.forward_mxfp4(q, cache, int32(new, cuda), cu, 4, block_table=bt,
                                 max_seq_len=300, causal=True)
        want = ref.paged_decode(f64(q), *values(cache), bt.cpu().numpy(), new, scale,
                                cu_seqlens_q=cu.tolist())
        assert check(got, *want, 300).all()
        old = new


def test_in_graphs(cuda):
    """Two steps captured on one module, replayed in turn with eager work in between as the
    lengths grow, against the eager result."""
    hq, hk, d, page = 32, 8, 128, 16
    g = torch.Generator(device=cuda).manual_seed(4)
    cache = random_cache(g, 200, page, hk, d, cuda)
    bt = torch.randperm(200, generator=g, device=cuda).to(torch.int32).view(4, 50)
    q = torch.randn(8, hq, d, generator=g, device=cuda).to(BF)
    new = torch.randn(2, 4, hk, d, generator=g, device=cuda).to(BF)
    ctx, slots = int32([1, 20, 300, 0], cuda), int32([0, 1, 2, 3], cuda)
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)
    put = load("store_kvcache", "StoreKVCacheMxfp4")()
    cu = int32([0, 2, 5, 6, 8], cuda)

    def one():
        put(new[0], new[1], cache, slots)
        return attn.forward_mxfp4(q[:4], cache, ctx, block_table=bt)

    def drafts():
        return attn.forward_mxfp4(q, cache, ctx, cu, 3, block_table=bt)

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
    hq, hk, d, page = 64, 8, 128, 64
    g = torch.Generator(device=cuda).manual_seed(5)
    cache = random_cache(g, 100, page, hk, d, cuda)
    bt = torch.randperm(100, generator=g, device=cuda).to(torch.int32).view(4, 25)
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)
    q = torch.randn(4, hq, d, generator=g, device=cuda).to(BF)
    ctxs = [int32(x, cuda) for x in ([1500, 3, 900, 64], [10, 1600, 1, 0])]

    def step(q, ctx):
        return attn.forward_mxfp4(q, cache, ctx, block_table=bt, s_aux=None, window_size=(999, 0))

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


def test_compiled_step(cuda):
    """A store, the read-back and the attention under torch.compile: the bits of the eager step."""
    hq, hk, d, page = 16, 2, 128, 16
    g = torch.Generator(device=cuda).manual_seed(6)
    cache = random_cache(g, 20, page, hk, d, cuda)
    bt = torch.randperm(20, generator=g, device=cuda).to(torch.int32).view(2, 10)
    q = torch.randn(2, hq, d, generator=g, device=cuda).to(BF)
    new = torch.randn(2, 2, hk, d, generator=g, device=cuda).to(BF)
    ctx, cu = int32([9, 101], cuda), int32([0, 9, 110], cuda)
    slots = torch.stack([bt[0, 0] * 16 + 8, bt[1, 6] * 16 + 4]).long()
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)
    put = load("store_kvcache", "StoreKVCacheMxfp4")()

    def step(k, v, ks, vs, q):
        put(new[0], new[1], (k, v, ks, vs), slots)
        key = torch.zeros(110, hk, d, dtype=BF, device=q.device)
        value = torch.zeros_like(key)
        torch.ops.fastkernels_amd.gather_kvcache_mxfp4(key, value, k, v, ks, vs, bt, cu)
        return attn.forward_mxfp4(q, (k, v, ks, vs), ctx, block_table=bt), key, value

    got = []
    for f in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        c = [t.clone() for t in cache]
        got.append((*f(*c, q), *c))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    want = ref.mxfp4_values(*ref.mxfp4_blocks(f64(new[0])))
    assert np.array_equal(f64(got[1][1][[8, 109]]), want)
