"""Attention that reads part of a paged cache, without a GPU: what the entry points refuse,
the C ABI's own checks, and the definitions of ``oracle.partial`` against dense attention."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import partial as ref
from fastkernels_amd import _native as N
from fastkernels_amd import ops

BF, FP8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


def args():
    """A valid call's tensors (CPU: a call that passes its checks raises RuntimeError)."""
    return dict(q=torch.zeros(3, 8, 128, dtype=BF), k=torch.zeros(5, 16, 2, 128, dtype=BF),
                bt=torch.zeros(3, 4, dtype=I32), ctx=torch.ones(3, dtype=I32),
                kb=torch.zeros(5, 2, 2, 128, dtype=BF), sc=torch.zeros(3, 2, 4),
                idx=torch.zeros(3, 2, 2, dtype=I32), cu=torch.tensor([0, 1, 2, 3], dtype=I32),
                gr=torch.tensor([0, 3], dtype=I32), pre=torch.tensor([16], dtype=I32))


def bounds(**kw):
    a = {**args(), **kw}
    ops.update_key_bounds(a["kb"], a["k"], a["bt"], a["ctx"], a.get("cuq"), 1)


def scores(**kw):
    a = {**args(), **kw}
    ops.block_scores(a["sc"], a["q"], a["kb"], a["bt"], a["ctx"], 16, a.get("ks"), a.get("cuq"), 1)


def select(**kw):
    a = {**args(), **kw}
    ops.select_blocks(a["idx"], a["sc"], a["ctx"], 16, a.get("first", 0), a.get("last", 1),
                      a.get("cuq"))


def sparse(**kw):
    a = {**args(), **kw}
    ops.sparse_paged_decode(a.get("out", torch.empty_like(a["q"])), a["q"], a["k"],
                            a.get("v", a["k"]), a["bt"], a["ctx"], a["idx"], 0.1, a.get("ks"),
                            a.get("vs"), a.get("sinks"), a.get("cuq"))


def prefix(**kw):
    a = {**args(), **kw}
    ops.shared_prefix_decode(a.get("out", torch.empty_like(a["q"])), a["q"], a["k"],
                             a.get("v", a["k"]), a["bt"], a["ctx"], a["gr"], a["pre"], 0.1,
                             a.get("ks"), a.get("vs"), a.get("window", -1), a.get("sinks"),
                             a.get("most", 0))


@pytest.mark.parametrize("call", [bounds, scores, select, sparse, prefix])
def test_a_valid_call_reaches_the_device_check(call):
    with pytest.raises(RuntimeError, match="GPU only"):
        call()


BAD = [
    (bounds, dict(kb=torch.zeros(5, 2, 2, 128)), ValueError),
    (bounds, dict(kb=torch.zeros(4, 2, 2, 128, dtype=BF)), ValueError),
    (bounds, dict(kb=torch.zeros(5, 2, 128, dtype=BF)), ValueError),
    (bounds, dict(k=torch.zeros(5, 2, 16, 128, dtype=BF).transpose(1, 2)), ValueError),
    (bounds, dict(k=torch.zeros(5, 16, 2, 128), kb=torch.zeros(5, 2, 2, 128)), TypeError),
    (bounds, dict(ctx=torch.ones(3, dtype=torch.int64)), TypeError),
    (bounds, dict(cuq=torch.zeros(4, dtype=torch.int64)), TypeError),
    (bounds, dict(cuq=torch.zeros(5, dtype=I32)), TypeError),
    (bounds, dict(bt=torch.zeros(2, 4, dtype=I32)), ValueError),
    (scores, dict(q=torch.zeros(3, 8, 128)), ValueError),
    (scores, dict(q=torch.zeros(3, 7, 128, dtype=BF)), ValueError),
    (scores, dict(q=torch.zeros(3, 8, 256, dtype=BF)[:, :, ::2]), ValueError),
    (scores, dict(sc=torch.zeros(3, 2, 4, dtype=BF)), ValueError),
    (scores, dict(sc=torch.zeros(3, 8, 4)), ValueError),
    (scores, dict(sc=torch.zeros(3, 2, 8)[:, :, ::2]), ValueError),
    (scores, dict(ks=torch.ones(3)), ValueError),
    (scores, dict(bt=torch.zeros(3, 4, dtype=torch.int64)), TypeError),
    (scores, dict(bt=torch.zeros(3, 8, dtype=I32)[:, ::2]), TypeError),
    (select, dict(idx=torch.zeros(3, 2, 2, dtype=torch.int64)), ValueError),
    (select, dict(idx=torch.zeros(2, 2, 2, dtype=I32)), ValueError),
    (select, dict(first=2, last=1), ValueError),
    (select, dict(first=-1), ValueError),
    (select, dict(sc=torch.zeros(3, 2, 4, dtype=torch.float64)), ValueError),
    (select, dict(ctx=torch.ones(2, dtype=I32)), TypeError),
    (sparse, dict(out=torch.zeros(3, 4, 128, dtype=BF)), ValueError),
    (sparse, dict(v=torch.zeros(5, 16, 2, 64, dtype=BF)), ValueError),
    (sparse, dict(v=torch.zeros(5, 16, 2, 128).to(FP8)), TypeError),
    (sparse, dict(idx=torch.zeros(3, 8, 2, dtype=I32)), ValueError),
    (sparse, dict(sinks=torch.zeros(4)), ValueError),
    (sparse, dict(vs=torch.zeros(2, dtype=BF)), ValueError),
    (sparse, dict(k=torch.zeros(5, 16, 2, 128, dtype=torch.float16)), TypeError),
    (prefix, dict(gr=torch.tensor([0, 3])), TypeError),
    (prefix, dict(gr=torch.tensor([0, 1, 3], dtype=I32)), ValueError),
    (prefix, dict(gr=torch.zeros(0, dtype=I32)), ValueError),
    (prefix, dict(pre=torch.tensor([16])), TypeError),
    (prefix, dict(window=-2), ValueError),
    (prefix, dict(most=-1), ValueError),
    (prefix, dict(ctx=torch.ones(6, dtype=I32)[::2]), TypeError),
    (prefix, dict(out=torch.zeros(3, 8, 128)), ValueError),
]


@pytest.mark.parametrize("i", range(len(BAD)))
def test_refused(i):
    call, kw, error = BAD[i]
    with pytest.raises(error):
        call(**kw)


def test_empty_batches_return():
    e = dict(q=torch.zeros(0, 8, 128, dtype=BF), ctx=torch.zeros(0, dtype=I32),
             bt=torch.zeros(0, 4, dtype=I32), sc=torch.zeros(0, 2, 4),
             idx=torch.zeros(0, 2, 2, dtype=I32), gr=torch.zeros(1, dtype=I32))
    for call in (bounds, scores, select, sparse, prefix):
        call(**e)


def last_error():
    return N.lib().fk_last_error().decode()


def test_c_abi_refusals():
    """The library's own checks, before any launch (pointers that are never read)."""
    lib, p = N.lib(), ctypes.c_void_p(0x100000)

    def kb(batch=1, most=1, hk=2, d=128, page=16, blocks=4, cu=None, tag=N.FK_DTYPE_BF16,
           ptr=p):
        return lib.fk_update_key_bounds(ptr, p, tag, p, 4, 4, p, cu, batch, most, hk, d, page,
                                        blocks, None)

    assert kb(batch=0) == N.FK_OK
    for kw in (dict(batch=-1), dict(batch=65536), dict(most=2), dict(hk=0), dict(page=24),
               dict(page=8), dict(blocks=0), dict(tag=N.FK_DTYPE_F16), dict(ptr=None),
               dict(ptr=ctypes.c_void_p(0x100008))):
        assert kb(**kw) == N.FK_ERR_INVALID_ARG, kw
        assert last_error().startswith("fk_update_key_bounds")
    assert kb(d=96) == N.FK_ERR_UNSUPPORTED

    def bs(hq=8, hk=2, width=4, rows=1, batch=1, most=1, cu=None, qstride=1024):
        return lib.fk_block_scores(p, 8, 4, width, p, qstride, p, N.FK_DTYPE_BF16, None, p, 4, 4,
                                   p, cu, batch, rows, most, hq, hk, 128, 16, 4, None)

    assert bs(batch=0) == N.FK_OK
    for kw in (dict(hq=7), dict(width=-1), dict(rows=-1), dict(most=2), dict(qstride=1025),
               dict(batch=65535, rows=65535, most=100, cu=p), dict(batch=2)):
        assert bs(**kw) == N.FK_ERR_INVALID_ARG, kw

    def sb(keep=2, first=0, last=1, page=16, rows=1, hk=2):
        return lib.fk_select_blocks(p, 4, 2, keep, p, 8, 4, 4, p, None, 1, rows, hk, page, first,
                                    last, None)

    assert sb(keep=0, last=0) == N.FK_OK and sb(rows=0) == N.FK_OK
    for kw in (dict(first=2), dict(first=-1), dict(page=12), dict(rows=-1), dict(hk=0),
               dict(keep=-1), dict(first=2 ** 31 - 1, last=2 ** 31 - 1)):
        assert sb(**kw) == N.FK_ERR_INVALID_ARG, kw

    def sp(hq=8, hk=2, d=128, rows=1, batch=1, keep=2, page=16, stride=1024):
        return lib.fk_sparse_paged_decode(p, stride, p, stride, p, p, N.FK_DTYPE_BF16, None, None,
                                          p, 4, 4, p, None, batch, rows, p, 4, 2, keep, hq, hk, d,
                                          page, 4, 0.1, None, None, 0, None)

    assert sp(rows=0) == N.FK_OK
    for kw in (dict(hq=9), dict(rows=2), dict(rows=65536, batch=65535), dict(keep=-1),
               dict(keep=2 ** 30, page=64), dict(page=100), dict(stride=4)):
        assert sp(**kw) == N.FK_ERR_INVALID_ARG, kw
    assert sp(d=72) == N.FK_ERR_UNSUPPORTED

    def sh(batch=1, groups=1, most=0, window=-1, d=128, hq=8):
        return lib.fk_shared_prefix_decode(p, 1024, p, 1024, p, p, N.FK_DTYPE_BF16, None, None, p,
                                           4, 4, p, batch, p, p, groups, most, hq, 2, d, 16, 4,
                                           0.1, window, None, None, 0, None)

    assert sh(batch=0) == N.FK_OK
    for kw in (dict(groups=-1), dict(most=-1), dict(window=-2), dict(hq=9), dict(batch=70000)):
        assert sh(**kw) == N.FK_ERR_INVALID_ARG, kw
    assert sh(d=80) == N.FK_ERR_UNSUPPORTED


def test_flash_attn_decode_entry_points_refuse():
    from fastkernels_amd.candidate.L1.flash_attn_decode import FlashAttnDecode

    a, attn = args(), FlashAttnDecode(8, 2, 128)
    with pytest.raises(ValueError, match="block_table"):
        attn.forward_sparse(a["q"], a["k"], a["k"], a["kb"], a["ctx"], 2)
    with pytest.raises(NotImplementedError, match="window"):
        attn.forward_sparse(a["q"], a["k"], a["k"], a["kb"], a["ctx"], 2, block_table=a["bt"],
                            window_size=(7, 0))
    with pytest.raises(TypeError, match="num_splits"):
        attn.forward_shared_prefix(a["q"], a["k"], a["k"], a["ctx"], a["gr"], a["pre"],
                                   block_table=a["bt"], num_splits=4)
    with pytest.raises(RuntimeError, match="GPU only"):
        attn.forward_shared_prefix(a["q"], a["k"], a["k"], a["ctx"], a["gr"], a["pre"],
                                   block_table=a["bt"])


def test_custom_ops_trace():
    """The ops are registered with in-place annotations and fake implementations."""
    a = {k: v.to("meta") for k, v in args().items()}
    o = torch.ops.fastkernels_amd
    o.update_key_bounds(a["kb"], a["k"], a["bt"], a["ctx"])
    o.block_scores(a["sc"], a["q"], a["kb"], a["bt"], a["ctx"], 16)
    o.select_blocks(a["idx"], a["sc"], a["ctx"], 16)
    o.sparse_paged_decode(a["q"], a["q"], a["k"], a["k"], a["bt"], a["ctx"], a["idx"], 0.1)
    o.shared_prefix_decode(a["q"], a["q"], a["k"], a["k"], a["bt"], a["ctx"], a["gr"], a["pre"],
                           0.1)


# ---------------------------------------------------------------------------
# the definitions
# ---------------------------------------------------------------------------
def test_definitions_agree_with_dense_attention():
    rng = np.random.default_rng(0)
    nb, page, hk, g, d = 9, 16, 2, 3, 64
    k, v = rng.standard_normal((2, nb, page, hk, d))
    q = rng.standard_normal((3, hk * g, d))
    bt = np.array([[3, 1, 7, 0], [3, 1, 5, -1], [2, 8, 4, 6]])
    lens = [55, 40, 20]
    every = np.tile(np.arange(4), (3, hk, 1))
    a = ref.sparse_paged_decode(q, k, v, bt, lens, every, d ** -0.5)[0]
    b = ref.shared_prefix_decode(q, k, v, bt, lens, [0, 2, 3], [32, 7], d ** -0.5)[0]
    assert np.allclose(a, b, atol=1e-12)
    for r in range(3):
        kk = k[bt[r]].reshape(-1, hk, d)[:lens[r]]
        vv = v[bt[r]].reshape(-1, hk, d)[:lens[r]]
        for h in range(hk * g):
            x = kk[:, h // g] @ q[r, h] * d ** -0.5
            w = np.exp(x - x.max())
            assert np.allclose(a[r, h], w @ vv[:, h // g] / w.sum(), atol=1e-12)


def test_selection_keeps_what_the_bounds_promise():
    """No block left out has a key with a larger logit than its score says."""
    rng = np.random.default_rng(1)
    nb, page, hk, d, n = 12, 16, 2, 64, 180
    k = rng.standard_normal((nb, page, hk, d))
    q = rng.standard_normal((1, 4, d))
    bt = rng.permutation(nb)[None]
    kb = ref.update_key_bounds(np.zeros((nb, hk, 2, d)), k, bt, [n], [0, n])
    s, _ = ref.block_scores(q, kb, bt, [n], page, 12)
    x = np.einsum("hgd,pthd->hpgt", q[0].reshape(hk, 2, d), k[bt[0]])
    assert (s[0] >= np.where(np.arange(12)[None, :] < 11, x.max((2, 3)), -np.inf) - 1e-12).all()
    idx = ref.select_blocks(s, [n], page, 5, 1, 2)
    assert (idx[:, :, 0] == 0).all() and (idx[:, :, -2:] == [10, 11]).all()


def test_prefix_bound_keeps_the_workspace_small():
    N = pytest.importorskip("fastkernels_amd._native")
    size = lambda bound, batch=8, groups=1: N.shared_prefix_bytes(batch, groups, bound, 32, 8, 128)
    assert size(128) < size(1500) < size(0)
    assert size(1 << 40) == size(0)
    assert size(1500, 0) == 0
    assert size(64, 64, 64) < size(64, 4096, 1000)
    with pytest.raises(N.FkError):
        size(-1)


def test_c_abi_refuses_groups_without_arrays():
    """NULL cu_groups or prefix_lens with a group (GPU: with none they are not read)."""
    lib, p = N.lib(), ctypes.c_void_p(0x100000)
    for cu, pre in ((None, p), (p, None), (None, None)):
        rc = lib.fk_shared_prefix_decode(p, 1024, p, 1024, p, p, N.FK_DTYPE_BF16, None, None, p, 4,
                                         4, p, 2, cu, pre, 1, 0, 8, 2, 128, 16, 4, 0.1, -1, None,
                                         p, 1 << 40, None)
        assert rc == N.FK_ERR_INVALID_ARG and "null pointer" in last_error()


def test_rows_of_sequences_need_their_bound():
    """cu_seqlens_q without max_seqlen_q is refused: rows past a bound of one would be left out."""
    from fastkernels_amd.candidate.L1.flash_attn_decode import FlashAttnDecode

    a, attn = args(), FlashAttnDecode(8, 2, 128)
    for call in (
            lambda **kw: ops.update_key_bounds(a["kb"], a["k"], a["bt"], a["ctx"], **kw),
            lambda **kw: ops.block_scores(a["sc"], a["q"], a["kb"], a["bt"], a["ctx"], 16, **kw),
            lambda **kw: attn.forward_sparse(a["q"], a["k"], a["k"], a["kb"], a["ctx"], 2,
                                             block_table=a["bt"], **kw)):
        with pytest.raises(ValueError, match="max_seqlen_q"):
            call(cu_seqlens_q=a["cu"])
        for kw in (dict(cu_seqlens_q=a["cu"], max_seqlen_q=1), {}):
            with pytest.raises(RuntimeError, match="GPU only"):
                call(**kw)
    m = {k: v.to("meta") for k, v in a.items()}
    o = torch.ops.fastkernels_amd
    o.update_key_bounds(m["kb"], m["k"], m["bt"], m["ctx"], m["cu"], 2)
    o.block_scores(m["sc"], m["q"], m["kb"], m["bt"], m["ctx"], 16, None, m["cu"], 2)


@pytest.mark.parametrize("how", ["sparse", "prefix"])
def test_entry_points_compile(how):
    """Under torch.compile each method is its custom ops, with no graph break."""
    from fastkernels_amd.candidate.L1.flash_attn_decode import FlashAttnDecode

    a, attn, calls = args(), FlashAttnDecode(8, 2, 128), []

    def backend(gm, _):
        calls.extend(str(n.target) for n in gm.graph.nodes if n.op == "call_function")
        return lambda *_: [torch.zeros(3, 8, 128)]

    def step(q):
        if how == "sparse":
            return attn.forward_sparse(q, a["k"], a["k"], a["kb"], a["ctx"], 2,
                                       block_table=a["bt"], max_seq_len=64)
        return attn.forward_shared_prefix(q, a["k"], a["k"], a["ctx"], a["gr"], a["pre"],
                                          block_table=a["bt"])

    torch.compile(step, backend=backend, fullgraph=True)(a["q"])
    ops_called = [c.split(".")[1] for c in calls if c.startswith("fastkernels_amd.")]
    assert ops_called == (["block_scores", "select_blocks", "sparse_paged_decode"]
                          if how == "sparse" else ["shared_prefix_decode"])


def test_more_groups_than_a_launch_takes_are_refused():
    lib, p = N.lib(), ctypes.c_void_p(0x100000)
    rc = lib.fk_shared_prefix_decode(p, 1024, p, 1024, p, p, N.FK_DTYPE_BF16, None, None, p, 4, 4, p,
                                     3000, p, p, 2049, 0, 8, 2, 128, 16, 4, 0.1, -1, None, p,
                                     1 << 40, None)
    assert rc == N.FK_ERR_INVALID_ARG and "2049 groups" in last_error()
