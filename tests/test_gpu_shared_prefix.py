"""Decode attention of a batch in groups that share a prefix (GPU), against the float64
definition (``oracle.partial``).  The tolerance is that of tests/test_gpu_sparse.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import partial as ref
from test_gpu_sparse import attn_tolerance, check_attn, cu_of, f64, int32, load, make_cache, poison

pytestmark = pytest.mark.gpu


def shared_tables(g, groups, dev, page):
    """groups: list of (prefix, [own tokens per row] ), a row's length being their sum or, for
    a negative entry, the positive length of a row shorter than the prefix; prefix None: rows
    outside any group.  Only the first row of a group lists the prefix's whole pages."""
    rows, pool = [], 0
    for prefix, own in groups:
        start = len(rows)
        for t in own:
            n = (prefix or 0) + t if t >= 0 else -t
            rows.append((start, prefix or 0, n))
    pages = max(-(-max(n, p) // page) for _, p, n in rows) + 1
    bt = torch.full((len(rows), pages), -1, dtype=torch.int32)
    pool = 0
    for b, (start, prefix, n) in enumerate(rows):
        whole = prefix // page if b != start else 0
        for j in range(whole, -(-max(n, prefix if b == start else 0) // page)):
            bt[b, j] = pool
            pool += 1
    perm = torch.randperm(pool + 3, generator=g, device=dev).to(torch.int32).cpu()
    bt = torch.where(bt >= 0, perm[bt.clamp(min=0).long()], bt)
    return bt.to(dev), pool + 3, [n for _, _, n in rows]


def build(cuda, kv, hq, hk, d, page, groups, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed + hq + d + page)
    bt, pool, lens = shared_tables(g, groups, cuda, page)
    k = make_cache(g, pool, page, hk, d, kv, cuda)
    v = make_cache(g, pool, page, hk, d, kv, cuda)
    real = [(p, o) for p, o in groups if p is not None]
    cu = cu_of([len(o) for _, o in real], cuda)
    pre = int32([p for p, _ in real], cuda)
    # a prefix that ends inside a page: rows keep their own copy of that page, whose positions
    # below the prefix hold other values; they are not read
    at = 0
    used = torch.zeros(pool, page, dtype=torch.bool, device=cuda)
    for p, own in groups:
        for i in range(len(own)):
            n = lens[at + i]
            for j in range(-(-n // page)):
                lo = 0 if i == 0 else max(0, min(page, (p or 0) - j * page))
                pg = int(bt[at + i, j])
                if pg >= 0:
                    used[pg, lo:max(0, min(page, n - j * page))] = True
        if p:
            most = min(p, max(lens[at:at + len(own)], default=0))
            for j in range(-(-most // page)):
                used[int(bt[at, j]), :min(page, most - j * page)] = True
        at += len(own)
    for c in (k, v):
        poison(c, ~used)
    ks = vs = None
    if kv == "fp8":
        ks = torch.linspace(0.1, 0.3, hk, device=cuda)
        vs = torch.linspace(0.2, 0.4, hk, device=cuda)
    q = torch.randn(len(lens), hq, d, generator=g, device=cuda).to(torch.bfloat16)
    return g, q, k, v, bt, lens, cu, pre, ks, vs


GROUPS = {
    "one": [(200, [5, 40, 1, 0, 300])],
    "ragged": [(333, [7, 0, -1, 20]), (64, [1]), (1000, [100, 3, -500, 250, 16, 17]),
               (None, [90, 0, 16])],
    "none": [(None, [30, 700, 0])],
    "zero": [(0, [10, 0]), (0, [129])],
    "wide": [(513, [3 + i for i in range(40)])],
    "short": [(5, [1, 2, 3]), (15, [0, 1])],
    "empty": [(100, []), (48, [1, 2]), (100, [])],
    "long": [(9000, [60, 1, 2500])],
}


@pytest.mark.parametrize("name", list(GROUPS))
@pytest.mark.parametrize("kv,hq,hk,d,page", [
    ("bf16", 32, 8, 128, 16), ("fp8", 16, 2, 128, 64), ("bf16", 8, 1, 256, 16),
    ("bf16", 10, 10, 64, 32), ("fp8", 40, 2, 64, 16), ("fp8", 12, 4, 256, 128),
])
def test_shared_prefix(cuda, kv, hq, hk, d, page, name):
    from fastkernels_amd import ops

    g, q, k, v, bt, lens, cu, pre, ks, vs = build(cuda, kv, hq, hk, d, page, GROUPS[name])
    out = torch.full_like(q, 9.0)
    ops.shared_prefix_decode(out, q, k, v, bt, int32(lens, cuda), cu, pre, d ** -0.5, ks, vs,
                             max_prefix_len=0 if name == "ragged" else
                             max([1, *pre.tolist()]))
    want = ref.shared_prefix_decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), lens,
                                    cu.cpu().numpy(), pre.cpu().numpy(), d ** -0.5, f64(ks),
                                    f64(vs))
    check_attn(out, *want)


@pytest.mark.parametrize("bound", [1, 16, 100, 500])
def test_shared_prefix_bound(cuda, bound):
    """Prefixes longer than max_prefix_len are shared up to there."""
    from fastkernels_amd import ops

    g, q, k, v, bt, lens, cu, pre, ks, vs = build(cuda, "bf16", 32, 8, 128, 16, GROUPS["ragged"])
    out = torch.full_like(q, 9.0)
    ops.shared_prefix_decode(out, q, k, v, bt, int32(lens, cuda), cu, pre, 128 ** -0.5,
                             max_prefix_len=bound)
    want = ref.shared_prefix_decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), lens,
                                    cu.cpu().numpy(), pre.cpu().numpy(), 128 ** -0.5)
    check_attn(out, *want)


@pytest.mark.parametrize("window", [0, 15, 100, 600, 5000])
@pytest.mark.parametrize("kv,hq,hk,d,page", [("bf16", 32, 8, 128, 16), ("fp8", 24, 2, 64, 32)])
def test_shared_prefix_window_and_sinks(cuda, kv, hq, hk, d, page, window):
    from fastkernels_amd import ops

    g, q, k, v, bt, lens, cu, pre, ks, vs = build(cuda, kv, hq, hk, d, page, GROUPS["ragged"])
    sinks = torch.randn(hq, generator=g, device=cuda)
    wide = torch.full((len(lens), hq + 3, d), 9.0, dtype=torch.bfloat16, device=cuda)
    ops.shared_prefix_decode(wide[:, :hq], q, k, v, bt, int32(lens, cuda), cu, pre, d ** -0.5, ks,
                             vs, window, sinks)
    want = ref.shared_prefix_decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), lens,
                                    cu.cpu().numpy(), pre.cpu().numpy(), d ** -0.5, f64(ks),
                                    f64(vs), window, f64(sinks))
    check_attn(wide[:, :hq], *want)
    assert bool((wide[:, hq:] == 9.0).all())


def test_shared_prefix_is_decode(cuda):
    """FlashAttnDecode.forward_shared_prefix beside forward, the tables listing every page."""
    hq, hk, d, page = 32, 8, 128, 16
    g = torch.Generator(device=cuda).manual_seed(4)
    pre, own = 96 * page, [5, 300, 1, 44, 17, 900]
    bt = torch.full((6, 160), -1, dtype=torch.int32, device=cuda)
    perm = torch.randperm(1000, generator=g, device=cuda).to(torch.int32)
    at = 96
    for b, t in enumerate(own):
        n = -(-t // page)
        bt[b, :96], bt[b, 96:96 + n] = perm[:96], perm[at:at + n]
        at += n
    k, v = (make_cache(g, 1000, page, hk, d, "bf16", cuda) for _ in range(2))
    q = torch.randn(6, hq * d, generator=g, device=cuda).to(torch.bfloat16)
    ctx = int32([pre + t for t in own], cuda)
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)
    got = attn.forward_shared_prefix(q, k, v, ctx, int32([0, 4, 6], cuda), int32([pre, pre], cuda),
                                     block_table=bt, max_prefix_len=pre)
    dense = attn(q, k, v, ctx, block_table=bt)
    assert got.shape == dense.shape
    want = ref.shared_prefix_decode(f64(q).reshape(6, hq, d), f64(k), f64(v), bt.cpu().numpy(),
                                    ctx.tolist(), [0, 4, 6], [pre, pre], d ** -0.5)
    check_attn(got, *want)
    check_attn(dense, *want)


def test_shared_prefix_in_graphs(cuda):
    """Two graphs of different groups captured on one module and replayed in turn, as the
    lengths and the prefixes change, against the eager result."""
    hq, hk, d, page = 32, 8, 128, 16
    _, q, k, v, bt, lens, cu, pre, _, _ = build(cuda, "bf16", hq, hk, d, page, GROUPS["one"])
    k, v = k.nan_to_num(1.0), v.nan_to_num(1.0)
    bt[:] = bt[:1].clamp(min=0)
    ctx = int32(lens, cuda)
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)
    two = int32([0, 2, 5], cuda)
    two_pre = int32([64, 160], cuda)

    def steps():
        return (attn.forward_shared_prefix(q, k, v, ctx, cu, pre, block_table=bt),
                attn.forward_shared_prefix(q, k, v, ctx, two, two_pre, block_table=bt))

    steps()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for args in ((cu, pre), (two, two_pre)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attn.forward_shared_prefix(q, k, v, ctx, *args, block_table=bt))
        graphs.append(graph)
    for i, new in enumerate((lens, [205, 240, 201, 200, 0], [1, 2, 3, 170, 190])):
        ctx.copy_(int32(new, cuda))
        two_pre.copy_(int32([64 - 16 * i, 160 - i], cuda))
        for graph in (graphs[i % 2], graphs[1 - i % 2]):
            graph.replay()
        got = [o.clone() for o in outs]
        want = steps()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_streams_at_once(cuda):
    """Shared-prefix and sparse calls that overlap on two streams, against the same calls one
    after the other: results depend on nothing but the arguments."""
    from fastkernels_amd import ops

    hq, hk, d, page = 32, 8, 128, 16
    calls = []
    for seed in range(2):
        g, q, k, v, bt, lens, cu, pre, _, _ = build(cuda, "bf16", hq, hk, d, page,
                                                    GROUPS["ragged"], seed)
        ctx, n = int32(lens, cuda), len(lens)
        idx = torch.randint(-1, 60, (n, hk, 20), generator=g, device=cuda, dtype=torch.int32)

        def call(out, args=(q, k, v, bt, ctx), cu=cu, pre=pre, idx=idx):
            ops.shared_prefix_decode(out[0], *args, cu, pre, d ** -0.5)
            ops.sparse_paged_decode(out[1], *args, idx, d ** -0.5)

        calls.append((call, (2, *q.shape)))
    want = [torch.zeros(s, dtype=torch.bfloat16, device=cuda) for _, s in calls]
    for (call, _), out in zip(calls, want):
        call(out)
    got = [[torch.zeros(s, dtype=torch.bfloat16, device=cuda) for _ in range(6)] for _, s in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(6):
        for (call, _), outs, stream in zip(calls, got, streams):
            with torch.cuda.stream(stream):
                call(outs[i])
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        for out in outs:
            assert torch.equal(out.view(torch.int16), w.view(torch.int16))


# Rows of a group whose prefix is longer than some of them: (prefix, length of each row).
SHORT_ROWS = {
    "padding": (100, [150, 40, 0, 100, 98, 130]),
    "first": (333, [0, 340, 333, 200, 1, 700]),
    "many": (700, [0 if i % 7 == 3 else 13 * i + 1 for i in range(60)]),
    "beyond": (5000, [1000, 1001, 1002, 999]),
}


@pytest.mark.parametrize("name", list(SHORT_ROWS))
@pytest.mark.parametrize("kv,hq,hk,d,page,bad", [
    ("bf16", 32, 8, 128, 16, "nan"), ("bf16", 32, 8, 128, 16, "inf"),
    ("bf16", 40, 2, 128, 32, "-inf"), ("fp8", 16, 2, 128, 64, "nan"),
    ("bf16", 8, 1, 256, 16, "inf"), ("bf16", 10, 10, 64, 32, "-inf"),
    ("fp8", 12, 4, 256, 128, "nan"), ("fp8", 40, 1, 64, 16, "nan"),
])
def test_values_that_a_shorter_row_does_not_see(cuda, kv, hq, hk, d, page, name, bad):
    """Keys and values of the prefix that only its longer rows see are not finite: rows that do
    not see them are as ever, and so are the dims of the others whose values are finite."""
    from fastkernels_amd import ops

    prefix, lens = SHORT_ROWS[name]
    g = torch.Generator(device=cuda).manual_seed(d + len(lens))
    pages = -(-max(prefix, *lens) // page)
    bt = torch.stack([torch.randperm(pages, generator=g, device=cuda) for _ in lens])
    bt[:, :-(-prefix // page)] = bt[0, :-(-prefix // page)]
    bt = (bt + 1).to(torch.int32)
    k = make_cache(g, pages + 1, page, hk, d, kv, cuda)
    v = make_cache(g, pages + 1, page, hk, d, kv, cuda)
    # behind each length that ends inside the prefix: one value of V; a key behind the median
    ends = sorted(n for n in set(lens) if 0 <= n < min(prefix, max(lens)))
    for i, n in enumerate(ends):
        at = (int(bt[0, n // page]), n % page, i % hk, (7 * i) % d)
        v.view(torch.uint8 if kv == "fp8" else v.dtype)[at] = 0x7F if kv == "fp8" else float(bad)
    mid = ends[len(ends) // 2]
    poison(k, (int(bt[0, mid // page]), mid % page, 0, 3))
    q = torch.randn(len(lens), hq, d, generator=g, device=cuda).to(torch.bfloat16)
    ks = vs = None
    if kv == "fp8":
        ks, vs = torch.linspace(0.1, 0.3, hk, device=cuda), torch.linspace(0.2, 0.4, hk,
                                                                          device=cuda)
    sinks = torch.randn(hq, generator=g, device=cuda)
    cu, pre = int32([0, len(lens)], cuda), int32([prefix], cuda)
    out = torch.full((len(lens), hq + 1, d), 9.0, dtype=torch.bfloat16, device=cuda)[:, :hq]
    ops.shared_prefix_decode(out, q, k, v, bt, int32(lens, cuda), cu, pre, d ** -0.5, ks, vs, -1,
                             sinks)
    with np.errstate(invalid="ignore"):
        want, mean, mag = ref.shared_prefix_decode(
            f64(q), f64(k), f64(v), bt.cpu().numpy(), lens, [0, len(lens)], [prefix], d ** -0.5,
            f64(ks), f64(vs), -1, f64(sinks))
    got, finite = f64(out), np.isfinite(want)
    assert finite[lens.index(min(lens))].all()
    assert not np.isfinite(got[~finite]).any()
    assert np.isfinite(got[finite]).all()
    want, mean, mag = want[finite], mean[finite], mag[finite]
    err = (np.abs(got[finite] - want) - attn_tolerance(want, mean, mag, d)).max()
    assert err <= 0, f"beyond the tolerance by {err}"


def test_no_groups_without_arrays(cuda):
    """The C ABI with num_groups 0 takes NULL for the groups' arrays."""
    from fastkernels_amd import _native as N

    hq, hk, d, page = 32, 8, 128, 16
    _, q, k, v, bt, lens, _, _, _, _ = build(cuda, "bf16", hq, hk, d, page, GROUPS["none"])
    nbytes = N.shared_prefix_bytes(len(lens), 0, 0, hq, hk, d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=cuda)
    out, ctx = torch.full_like(q, 9.0), int32(lens, cuda)
    N.call("fk_shared_prefix_decode", out.data_ptr(), hq * d, q.data_ptr(), hq * d, k.data_ptr(),
           v.data_ptr(), N.FK_DTYPE_BF16, None, None, bt.data_ptr(), bt.stride(0), bt.shape[1],
           ctx.data_ptr(), len(lens), None, None, 0, 0, hq, hk, d, page, k.shape[0], d ** -0.5, -1,
           None, ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
    want = ref.shared_prefix_decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), lens, [0], [],
                                    d ** -0.5)
    check_attn(out, *want)


@pytest.mark.parametrize("kv,hq,hk,d,page", [("bf16", 4, 2, 64, 16), ("fp8", 8, 1, 128, 32),
                                             ("bf16", 2, 2, 256, 16)])
def test_many_groups_and_rows(cuda, kv, hq, hk, d, page):
    """More groups than a wave has lanes and more rows than a work-group has threads: groups of
    every small size, empty and single ones among them, and rows outside any group behind."""
    groups = []
    for i in range(150):
        rows = (3, 0, 8, 1, 5, 2, 9)[i % 7]
        groups.append(((37 * i) % 250, [(11 * i + 29 * r) % 90 for r in range(rows)]))
    groups.append((None, [(17 * r) % 70 for r in range(40)]))
    from fastkernels_amd import ops

    _, q, k, v, bt, lens, cu, pre, ks, vs = build(cuda, kv, hq, hk, d, page, groups)
    assert len(lens) > 600 and int(cu[-1]) > 512
    out = torch.full_like(q, 9.0)
    ops.shared_prefix_decode(out, q, k, v, bt, int32(lens, cuda), cu, pre, d ** -0.5, ks, vs)
    want = ref.shared_prefix_decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), lens,
                                    cu.cpu().numpy(), pre.cpu().numpy(), d ** -0.5, f64(ks),
                                    f64(vs))
    check_attn(out, *want)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_entry_points(cuda, backend):
    """forward_sparse and forward_shared_prefix under torch.compile give what they give eagerly."""
    hq, hk, d, page = 32, 8, 128, 16
    g, q, k, v, bt, lens, cu, pre, _, _ = build(cuda, "bf16", hq, hk, d, page, GROUPS["one"])
    k, v = k.nan_to_num(1.0), v.nan_to_num(1.0)
    bt[:] = bt[:1].clamp(min=0)
    ctx = int32(lens, cuda)
    bounds = torch.randn(k.shape[0], hk, 2, d, generator=g, device=cuda).sort(dim=2).values.to(
        torch.bfloat16)
    attn = load("flash_attn_decode", "FlashAttnDecode")(hq, hk, d)

    def step(q, ctx):
        return (attn.forward_sparse(q, k, v, bounds, ctx, 9, block_table=bt, max_seq_len=512),
                attn.forward_shared_prefix(q, k, v, ctx, cu, pre, block_table=bt))

    compiled = torch.compile(step, backend=backend, fullgraph=True)
    for shift in (0, 1):
        want = step(q, ctx - shift)
        got = compiled(q, ctx - shift)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("scale", [-0.11, 0.0])
def test_shared_prefix_of_odd_arguments(cuda, kv, scale):
    """Rows before the first group, prefixes of any length, lengths past the table, masked pages,
    a scale that is not positive, key scales of either sign."""
    from fastkernels_amd import ops

    g = torch.Generator(device=cuda).manual_seed(12)
    hq, hk, d, page, width = 16, 2, 128, 16, 12
    lens = [40, 150, 180, 250, 10 ** 6, 0, 2 ** 31 - 1, 100, 33]
    bt = torch.stack([torch.randperm(40, generator=g, device=cuda)[:width] for _ in lens])
    bt = bt.to(torch.int32)
    cu, pre = int32([2, 4, 7, 8], cuda), int32([100, 2 ** 31 - 1, 50], cuda)
    bt[3, :6], bt[5:7] = bt[2, :6], bt[4]
    bt[1, 0], bt[2, 1], bt[3, 9], bt[4, 3] = -1, 10 ** 6, -1, -2 ** 31
    k, v = (make_cache(g, 40, page, hk, d, kv, cuda) for _ in range(2))
    q = torch.randn(len(lens), hq, d, generator=g, device=cuda).to(torch.bfloat16)
    ks = vs = None
    if kv == "fp8":
        ks, vs = torch.tensor([0.2, -0.3], device=cuda), torch.tensor([-0.1, 0.4], device=cuda)
    out = torch.full_like(q, 9.0)
    ops.shared_prefix_decode(out, q, k, v, bt, int32(lens, cuda), cu, pre, scale, ks, vs)
    seen = [min(n, width * page) for n in lens]  # (the definition counts tokens one by one)
    want, mean, mag = ref.shared_prefix_decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), seen,
                                               cu.tolist(), pre.tolist(), scale, f64(ks), f64(vs))
    check_attn(out, want, np.abs(mean), np.abs(mag))


def test_most_groups(cuda):
    """As many groups as a launch takes, of none to three rows each."""
    from fastkernels_amd import ops

    groups = [((5 * i) % 40, [(3 * i + r) % 20 for r in range((1, 2, 0, 3)[i % 4])])
              for i in range(2048)]
    _, q, k, v, bt, lens, cu, pre, _, _ = build(cuda, "bf16", 2, 1, 64, 16, groups)
    out = torch.full_like(q, 9.0)
    ops.shared_prefix_decode(out, q, k, v, bt, int32(lens, cuda), cu, pre, 0.125)
    want = ref.shared_prefix_decode(f64(q), f64(k), f64(v), bt.cpu().numpy(), lens,
                                    cu.cpu().numpy(), pre.cpu().numpy(), 0.125)
    check_attn(out, *want)


def test_most_rows(cuda):
    """As many rows as a launch takes, each with up to a page of its own behind a page that groups
    of 40 share, of which sparse decode lists the second: against dense float64."""
    from fastkernels_amd import ops

    n, d, page = 65535, 64, 16
    g = torch.Generator(device=cuda).manual_seed(6)
    k, v = (make_cache(g, 4096, page, 1, d, "bf16", cuda) for _ in range(2))
    own = torch.randint(0, 4096, (n,), generator=g, device=cuda, dtype=torch.int32)
    group = torch.arange(n, device=cuda) // 40
    bt = torch.stack([(group % 1024).to(torch.int32), own], 1)
    tail = torch.arange(n, device=cuda, dtype=torch.int32) % 17
    ctx = tail + page
    q = torch.randn(n, 2, d, generator=g, device=cuda).to(torch.bfloat16)
    last = int(group[-1]) + 1
    cu = torch.arange(last + 1, device=cuda, dtype=torch.int32).mul_(40).clamp_(max=n)
    prefix, sparse = torch.full_like(q, 9.0), torch.full_like(q, 9.0)
    ops.shared_prefix_decode(prefix, q, k, v, bt, ctx, cu,
                             torch.full((last,), page, dtype=torch.int32, device=cuda), d ** -0.5)
    idx = torch.ones(n, 1, 1, dtype=torch.int32, device=cuda)
    rows = torch.arange(n + 1, device=cuda, dtype=torch.int32)
    ops.sparse_paged_decode(sparse, q, k, v, bt, ctx, idx, d ** -0.5, cu_seqlens_q=rows)
    for out, pages in ((prefix, 2), (sparse, 1)):
        at = bt[:, 2 - pages:].long()
        kk, vv = (x[at].view(n, pages * page, d).double() for x in (k, v))
        seen = torch.arange(pages * page, device=cuda) < (ctx - (2 - pages) * page).unsqueeze(1)
        x = (q.double() @ kk.transpose(1, 2).contiguous()) * d ** -0.5
        w = torch.where(seen.unsqueeze(1), x, -float("inf")).softmax(2).nan_to_num(0.0)
        want, mean = w @ vv, w @ vv.abs()
        mag = (q.double().abs() @ kk.abs().transpose(1, 2).contiguous()).amax((1, 2)) * d ** -0.5
        tol = attn_tolerance(*(t.cpu().numpy() for t in (want, mean, mag.view(-1, 1, 1))), d)
        assert (np.abs(f64(out) - want.cpu().numpy()) <= tol).all()
