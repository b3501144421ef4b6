"""Caches that hold a token in few bytes, without a GPU: what the entry points refuse, the C
ABI's own checks, and the definitions of ``oracle.small_cache`` against plain ones."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import small_cache as ref
from fastkernels_amd import _native as N
from fastkernels_amd import ops

BF, F32, FP8, I32, I64 = (torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int32,
                          torch.int64)


def args():
    """A valid call's tensors (CPU: a call that passes its checks raises RuntimeError)."""
    return dict(cache=ops.new_mxfp4_cache(5, 16, 2, 128, "cpu"),
                key=torch.zeros(3, 2, 128, dtype=BF), q=torch.zeros(3, 8, 128, dtype=BF),
                slots=torch.zeros(3, dtype=I32), bt=torch.zeros(3, 4, dtype=I32),
                ctx=torch.ones(3, dtype=I32), cu=torch.tensor([0, 1, 2, 3], dtype=I32),
                lat=torch.zeros(5, 16, 576, dtype=BF), c=torch.zeros(3, 512, dtype=BF),
                kr=torch.zeros(3, 64, dtype=BF), qr=torch.zeros(3, 16, 64, dtype=BF),
                pos=torch.zeros(3, dtype=I64), cs=torch.zeros(32, 64),
                lq=torch.zeros(3, 16, 576, dtype=BF), lo=torch.zeros(3, 16, 512, dtype=BF))


def merged(kw):
    a = {**args(), **kw}
    a["cache"] = list(a["cache"])
    for i in range(4):
        a["cache"][i] = a.get(f"cache{i}", a["cache"][i])
    return a


def store(**kw):
    a = merged(kw)
    ops.store_kvcache_mxfp4(a["key"], a.get("value", a["key"]), *a["cache"], a["slots"])


def gather(**kw):
    a = merged(kw)
    ops.gather_kvcache_mxfp4(a["key"], a.get("value", a["key"]), *a["cache"], a["bt"], a["cu"])


def decode(**kw):
    a = merged(kw)
    ops.mxfp4_paged_decode(a.get("out", torch.empty_like(a["q"])), a["q"], *a["cache"], a["bt"],
                           a["ctx"], 0.1, a.get("window", -1), a.get("sinks"), a.get("cuq"),
                           a.get("most"))


def lstore(**kw):
    a = merged(kw)
    ops.latent_norm_rope_store(a["lat"], a["slots"], a["pos"], a["c"], a["kr"], a["cs"], False,
                               a.get("w"), 1e-6, a.get("scale"), a.get("qin", a["qr"]),
                               a.get("qout", a["qr"]), a.get("c_out"), a.get("k_out"))


def lgather(**kw):
    a = merged(kw)
    ops.gather_latent(a.get("rows", torch.zeros(3, 576, dtype=BF)), a["lat"], a["bt"], a["cu"],
                      a.get("scale"))


def ldecode(**kw):
    a = merged(kw)
    ops.latent_decode(a["lo"], a["lq"], a["lat"], a["bt"], a["ctx"], 0.1, a.get("scale"),
                      a.get("cuq"), a.get("most"), a.get("lse"))


CALLS = [store, gather, decode, lstore, lgather, ldecode]


@pytest.mark.parametrize("call", CALLS)
def test_a_valid_call_reaches_the_device_check(call):
    with pytest.raises(RuntimeError, match="GPU only"):
        call()


def u8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8)


BAD = [
    *[(f, kw, ValueError) for f in (store, gather, decode) for kw in (
        dict(cache0=u8(5, 2, 16 * 64)), dict(cache0=torch.zeros(5, 2, 16, 64)),
        dict(cache0=u8(5, 2, 32, 64)[:, :, ::2]), dict(cache1=u8(5, 2, 16, 64)),
        dict(cache1=u8(5, 2, 4, 16, 4, 8)), dict(cache2=u8(5, 2, 4, 32)),
        dict(cache3=u8(5, 2, 16, 4)), dict(cache3=u8(4, 2, 4, 16)),
        dict(cache=ops.new_mxfp4_cache(5, 16, 4, 64, "cpu"),
             cache2=u8(5, 4, 4, 16)))],
    (store, dict(key=torch.zeros(3, 256, dtype=BF)), ValueError),
    (store, dict(key=torch.zeros(3, 2, 64, dtype=BF)), ValueError),
    (store, dict(value=torch.zeros(2, 2, 128, dtype=BF)), ValueError),
    (store, dict(value=torch.zeros(3, 2, 128)), TypeError),
    (store, dict(key=torch.zeros(3, 2, 128, dtype=torch.float64)), TypeError),
    (store, dict(key=torch.zeros(3, 2, 256, dtype=BF)[:, :, ::2]), ValueError),
    (store, dict(key=torch.zeros(3, 4, 128, dtype=BF)[:, ::2]), ValueError),
    (store, dict(slots=torch.zeros(2, dtype=I32)), ValueError),
    (store, dict(slots=torch.zeros(3)), TypeError),
    (store, dict(slots=torch.zeros(6, dtype=I32)[::2]), TypeError),
    (gather, dict(key=torch.zeros(3, 2, 128)), ValueError),
    (gather, dict(key=torch.zeros(3, 4, 128, dtype=BF)), ValueError),
    (gather, dict(value=torch.zeros(4, 2, 128, dtype=BF)), ValueError),
    (gather, dict(cu=torch.zeros(4, dtype=I64)), TypeError),
    (gather, dict(cu=torch.zeros(0, dtype=I32)), TypeError),
    (gather, dict(bt=torch.zeros(2, 4, dtype=I32)), ValueError),
    (gather, dict(bt=torch.zeros(3, 4, dtype=I64)), TypeError),
    (decode, dict(q=torch.zeros(3, 8, 128)), ValueError),
    (decode, dict(q=torch.zeros(3, 7, 128, dtype=BF)), ValueError),
    (decode, dict(q=torch.zeros(3, 8, 64, dtype=BF)), ValueError),
    (decode, dict(out=torch.zeros(3, 4, 128, dtype=BF)), ValueError),
    (decode, dict(window=-2), ValueError),
    (decode, dict(sinks=torch.zeros(4)), ValueError),
    (decode, dict(ctx=torch.ones(3, dtype=I64)), TypeError),
    (decode, dict(ctx=torch.ones(2, dtype=I32)), TypeError),
    (decode, dict(cuq=torch.zeros(4, dtype=I32)), ValueError),  # without max_seqlen_q
    (decode, dict(cuq=torch.zeros(4, dtype=I64), most=1), TypeError),
    *[(f, kw, e) for f in (lstore, lgather, ldecode) for kw, e in (
        (dict(lat=torch.zeros(5, 16, 576)), TypeError),
        (dict(lat=torch.zeros(5, 16, 576, dtype=torch.float16)), TypeError),
        (dict(lat=torch.zeros(5, 9216, dtype=BF)), ValueError),
        (dict(lat=torch.zeros(5, 16, 640, dtype=BF)), ValueError),
        (dict(lat=torch.zeros(5, 32, 576, dtype=BF)[:, ::2]), ValueError),
        (dict(scale=torch.ones(1)), ValueError),  # of a bf16 cache
        (dict(lat=torch.zeros(5, 16, 576).to(FP8), scale=torch.ones(2)), ValueError),
        (dict(lat=torch.zeros(5, 16, 576).to(FP8), scale=torch.ones(1, dtype=BF)), ValueError))],
    (lstore, dict(c=torch.zeros(3, 512)), ValueError),
    (lstore, dict(c=torch.zeros(2, 512, dtype=BF)), ValueError),
    (lstore, dict(c=torch.zeros(3, 1, 512, dtype=BF)), ValueError),
    (lstore, dict(c=torch.zeros(3, 1024, dtype=BF)[:, ::2]), ValueError),
    (lstore, dict(kr=torch.zeros(2, 64, dtype=BF)), ValueError),
    (lstore, dict(pos=torch.zeros(3, dtype=I32)), TypeError),
    (lstore, dict(pos=torch.zeros(2, dtype=I64)), TypeError),
    (lstore, dict(cs=torch.zeros(32, 32)), ValueError),
    (lstore, dict(cs=torch.zeros(32, 64, dtype=torch.float16)), ValueError),
    (lstore, dict(w=torch.zeros(512)), ValueError),
    (lstore, dict(w=torch.zeros(576, dtype=BF)), ValueError),
    (lstore, dict(qin=None), ValueError),
    (lstore, dict(qout=None), ValueError),
    (lstore, dict(qout=torch.zeros(3, 8, 64, dtype=BF)), ValueError),
    (lstore, dict(qin=torch.zeros(3, 16, 32, dtype=BF)), ValueError),
    (lstore, dict(c_out=torch.zeros(3, 512)), ValueError),
    (lstore, dict(k_out=torch.zeros(3, 512, dtype=BF)), ValueError),
    (lstore, dict(slots=torch.zeros(2, dtype=I64)), ValueError),
    (lgather, dict(rows=torch.zeros(3, 512, dtype=BF)), ValueError),
    (lgather, dict(rows=torch.zeros(3, 576)), ValueError),
    (lgather, dict(rows=torch.zeros(3, 1, 576, dtype=BF)), ValueError),
    (lgather, dict(cu=torch.zeros(4)), TypeError),
    (lgather, dict(bt=torch.zeros(2, 4, dtype=I32)), ValueError),
    (ldecode, dict(lq=torch.zeros(3, 16, 512, dtype=BF)), ValueError),
    (ldecode, dict(lq=torch.zeros(3, 16, 576)), ValueError),
    (ldecode, dict(lo=torch.zeros(3, 16, 576, dtype=BF)), ValueError),
    (ldecode, dict(lo=torch.zeros(3, 8, 512, dtype=BF)), ValueError),
    (ldecode, dict(lse=torch.zeros(3, 16)), ValueError),
    (ldecode, dict(lse=torch.zeros(16, 3, dtype=BF)), ValueError),
    (ldecode, dict(lse=torch.zeros(3, 16).t()), ValueError),
    (ldecode, dict(cuq=torch.zeros(4, dtype=I32)), ValueError),
    (ldecode, dict(ctx=torch.ones(2, dtype=I32)), TypeError),
    (ldecode, dict(bt=torch.zeros(3, 8, dtype=I32)[:, ::2]), TypeError),
]


@pytest.mark.parametrize("i", range(len(BAD)))
def test_refused(i):
    call, kw, error = BAD[i]
    with pytest.raises(error):
        call(**kw)


def test_new_cache_refuses():
    for kw in (dict(head_dim=96), dict(block_size=8), dict(block_size=24)):
        with pytest.raises(ValueError):
            ops.new_mxfp4_cache(**{**dict(num_blocks=2, block_size=16, num_kv_heads=1,
                                          head_dim=64, device="cpu"), **kw})
    c = ops.new_mxfp4_cache(3, 32, 2, 256, "cpu")
    assert sum(t.numel() for t in c) == 3 * 32 * 2 * (256 + 256 // 16)


def test_empty_batches_return():
    e = dict(key=torch.zeros(0, 2, 128, dtype=BF), q=torch.zeros(0, 8, 128, dtype=BF),
             ctx=torch.zeros(0, dtype=I32), slots=torch.zeros(0, dtype=I32),
             bt=torch.zeros(0, 4, dtype=I32), cu=torch.zeros(1, dtype=I32),
             c=torch.zeros(0, 512, dtype=BF), kr=torch.zeros(0, 64, dtype=BF),
             qr=torch.zeros(0, 16, 64, dtype=BF), pos=torch.zeros(0, dtype=I64),
             lq=torch.zeros(0, 16, 576, dtype=BF), lo=torch.zeros(0, 16, 512, dtype=BF),
             rows=torch.zeros(0, 576, dtype=BF))
    for call in CALLS:
        call(**e)
    ldecode(lq=torch.zeros(3, 0, 576, dtype=BF), lo=torch.zeros(3, 0, 512, dtype=BF))


def test_c_abi_refusals():
    """The library's own checks, before any launch (pointers that are never read)."""
    lib, p = N.lib(), ctypes.c_void_p(0x100000)
    odd, bf, fp8 = ctypes.c_void_p(0x100008), N.FK_DTYPE_BF16, N.FK_DTYPE_FP8_E4M3FN

    def refuses(f, bad, name, error=N.FK_ERR_INVALID_ARG):
        for kw in bad:
            assert f(**kw) == error, kw
            assert N.lib().fk_last_error().decode().startswith(name), kw

    def st(tokens=1, tag=bf, hk=2, d=128, page=16, nb=4, cache=p, key=p):
        return lib.fk_store_kvcache_mxfp4(key, 256, p, 256, tag, cache, p, p, p, p, 0, tokens, hk,
                                          d, page, nb, None)

    assert st(tokens=0) == N.FK_OK
    refuses(st, [dict(tokens=-1), dict(tokens=1 << 40), dict(hk=0), dict(hk=70000), dict(page=24),
                 dict(page=8), dict(nb=0), dict(nb=1 << 31), dict(cache=odd), dict(cache=None),
                 dict(key=None)], "fk_store_kvcache_mxfp4")
    refuses(st, [dict(d=96), dict(tag=fp8)], "fk_store_kvcache_mxfp4", N.FK_ERR_UNSUPPORTED)

    def ga(rows=1, batch=1, key=p, stride=256, width=4, bts=4, d=128, cu=p):
        return lib.fk_gather_kvcache_mxfp4(key, stride, p, 256, p, p, p, p, p, bts, width, cu,
                                           batch, rows, 2, d, 16, 4, None)

    assert ga(rows=0) == N.FK_OK and ga(batch=0) == N.FK_OK
    refuses(ga, [dict(rows=-1), dict(rows=1 << 31), dict(batch=-1), dict(key=odd),
                 dict(stride=257), dict(width=-1), dict(bts=-1), dict(cu=None)],
            "fk_gather_kvcache_mxfp4")
    refuses(ga, [dict(d=512)], "fk_gather_kvcache_mxfp4", N.FK_ERR_UNSUPPORTED)

    def de(rows=1, batch=1, most=1, hq=8, hk=2, d=128, page=16, nb=4, window=-1, scales=p, ws=p,
           size=1 << 40, stride=1024, cu=None):
        return lib.fk_mxfp4_paged_decode(p, stride, p, stride, p, p, scales, p, p, 4, 4, p, cu,
                                         batch, rows, most, hq, hk, d, page, nb, 0.1, window,
                                         None, ws, size, None)

    assert de(rows=0) == N.FK_OK and de(batch=0) == N.FK_OK
    refuses(de, [dict(rows=-1), dict(rows=65536), dict(batch=65536), dict(most=0),
                 dict(most=65536), dict(hq=9), dict(hk=0), dict(page=24), dict(nb=0),
                 dict(nb=1 << 30), dict(window=-2), dict(scales=odd), dict(scales=None),
                 dict(ws=odd), dict(stride=1025), dict(page=1 << 29, nb=1)],
            "fk_mxfp4_paged_decode")
    refuses(de, [dict(d=96)], "fk_mxfp4_paged_decode", N.FK_ERR_UNSUPPORTED)
    refuses(de, [dict(ws=None), dict(size=1000)], "fk_mxfp4_paged_decode", N.FK_ERR_WORKSPACE)

    def ls(tokens=1, heads=16, slots=64, tag=bf, r=512, pe=64, lat=p, stride=512, cs=N.FK_DTYPE_F32,
           q=p, mp=32):
        return lib.fk_latent_norm_rope_store(p, tag, None, p, 0, slots, p, lat, stride, p, 64, None,
                                             1e-6, p, cs, mp, 0, q, 1024, 64, heads, p, 1024, 64,
                                             None, 0, None, 0, tokens, r, pe, None)

    assert ls(tokens=0) == N.FK_OK
    refuses(ls, [dict(tokens=-1), dict(tokens=1 << 31), dict(heads=-1), dict(heads=65536),
                 dict(slots=-1), dict(mp=-1), dict(tag=N.FK_DTYPE_F16), dict(lat=odd),
                 dict(stride=513), dict(cs=N.FK_DTYPE_F16), dict(q=None), dict(lat=None)],
            "fk_latent_norm_rope_store")
    refuses(ls, [dict(r=256), dict(pe=32)], "fk_latent_norm_rope_store", N.FK_ERR_UNSUPPORTED)

    def lg(rows=1, batch=1, out=p, stride=576, page=16, nb=4, width=4, r=512, cu=p, tag=bf,
           scale=None):
        return lib.fk_gather_latent(out, stride, p, tag, scale, p, 4, width, cu, batch, rows, r, 64,
                                    page, nb, None)

    assert lg(rows=0) == N.FK_OK and lg(batch=0) == N.FK_OK
    refuses(lg, [dict(rows=-1), dict(rows=1 << 31), dict(batch=-1), dict(out=odd),
                 dict(stride=577), dict(page=17), dict(nb=0), dict(width=-1), dict(cu=None),
                 dict(tag=N.FK_DTYPE_F32), dict(scale=p)], "fk_gather_latent")
    refuses(lg, [dict(r=448)], "fk_gather_latent", N.FK_ERR_UNSUPPORTED)

    def ld(rows=1, batch=1, most=1, heads=16, tag=bf, page=16, nb=4, r=512, ws=p, size=1 << 40,
           q=p, head_stride=576, cu=None, scale=None):
        return lib.fk_latent_decode(p, 8192, 512, q, 9216, head_stride, p, tag, scale, p, 4, 4, p,
                                    cu, batch, rows, most, heads, r, 64, page, nb, 0.1, None, 0,
                                    ws, size, None)

    assert ld(rows=0) == N.FK_OK and ld(batch=0) == N.FK_OK
    refuses(ld, [dict(rows=-1), dict(rows=65536), dict(batch=65536), dict(most=0),
                 dict(most=65536), dict(heads=0), dict(heads=65536), dict(page=48), dict(nb=0),
                 dict(tag=N.FK_DTYPE_F16), dict(q=odd), dict(q=None), dict(head_stride=577),
                 dict(ws=odd), dict(scale=p)], "fk_latent_decode")
    refuses(ld, [dict(r=256)], "fk_latent_decode", N.FK_ERR_UNSUPPORTED)
    refuses(ld, [dict(ws=None), dict(size=1000)], "fk_latent_decode", N.FK_ERR_WORKSPACE)

    size = ctypes.c_int64()
    for f, good in ((lib.fk_mxfp4_paged_decode_plan, (4, 1, 8, 2, 128)),
                    (lib.fk_latent_decode_plan, (4, 1, 16, 512))):
        assert f(*good, ctypes.byref(size)) == N.FK_OK and size.value > 0
        assert f(0, *good[1:], ctypes.byref(size)) == N.FK_OK and size.value == 0
        for bad in ((-1, *good[1:]), (4, 0, *good[2:]), (70000, *good[1:])):
            assert f(*bad, ctypes.byref(size)) == N.FK_ERR_INVALID_ARG
        assert f(*good, None) == N.FK_ERR_INVALID_ARG


def test_c_abi_refuses_more_than_a_launch_takes():
    """A grid has fewer than 2^32 threads: refused by the arguments' checks, before a launch."""
    lib, p = N.lib(), ctypes.c_void_p(0x100000)

    def st(tokens, hk, d):
        return lib.fk_store_kvcache_mxfp4(p, hk * d, p, hk * d, N.FK_DTYPE_BF16, p, p, p, p, p, 0,
                                          tokens, hk, d, 16, 4, None)

    def ga(rows):
        return lib.fk_gather_kvcache_mxfp4(p, 64, p, 64, p, p, p, p, p, 4, 4, p, 1, rows, 1, 64, 16,
                                           4, None)

    def ls(tokens):
        return lib.fk_latent_norm_rope_store(p, N.FK_DTYPE_BF16, None, p, 0, 64, p, p, 512, p, 64,
                                             None, 1e-6, p, N.FK_DTYPE_F32, 32, 0, None, 0, 0, 0,
                                             None, 0, 0, None, 0, None, 0, tokens, 512, 64, None)

    def lg(rows):
        return lib.fk_gather_latent(p, 576, p, N.FK_DTYPE_BF16, None, p, 4, 4, p, 1, rows, 512, 64,
                                    16, 4, None)

    for f, bad in ((lambda n: st(n, 8, 128), 1 << 24), (lambda n: st(n, 1, 64), 1 << 28),
                   (lambda n: st(n, 65535, 256), 1025), (ga, 1 << 29), (ls, 1 << 24),
                   (lg, 1 << 29)):
        assert f(bad) == N.FK_ERR_INVALID_ARG
        assert str(bad) in lib.fk_last_error().decode()


@pytest.mark.parametrize("page,hk,nb", [(16, 2, 1 << 28), (16, 1, (1 << 31) - 1), (64, 8, 1 << 27),
                                        (1 << 20, 1, 4104)])
def test_c_abi_takes_every_cache_that_fits_a_gpu(page, hk, nb):
    """2^32 tokens and more of a head of 64 are 272 GiB; with pages counted in 32 bits there is
    room for all."""
    lib, p = N.lib(), ctypes.c_void_p(0x100000)

    def de(nb):
        return lib.fk_mxfp4_paged_decode(p, 64, p, 64, p, p, p, p, p, 4, 4, p, None, 0, 1, 1, hk, hk,
                                         64, page, nb, 0.1, -1, None, p, 1 << 40, None)

    assert de(nb) == N.FK_OK, lib.fk_last_error().decode()
    assert de((1 << 31) // hk) == N.FK_ERR_INVALID_ARG


def test_modules_refuse():
    from fastkernels_amd.candidate.L1.flash_attn_decode import FlashAttnDecode
    from fastkernels_amd.candidate.L1.latent_attn import LatentAttnDecode

    a, attn = args(), FlashAttnDecode(8, 2, 128)
    with pytest.raises(TypeError, match="scale"):
        attn.forward_mxfp4(a["q"], a["cache"], a["ctx"], block_table=a["bt"], k_scale=0.5)
    with pytest.raises(TypeError, match="num_splits"):
        attn.forward_mxfp4(a["q"], a["cache"], a["ctx"], block_table=a["bt"], num_splits=2)
    with pytest.raises(ValueError, match="max_seqlen_q"):
        attn.forward_mxfp4(a["q"], a["cache"], a["ctx"], a["cu"], block_table=a["bt"])
    with pytest.raises(RuntimeError, match="GPU only"):
        attn.forward_mxfp4(a["q"].view(3, -1), a["cache"], a["ctx"], block_table=a["bt"])
    with pytest.raises(NotImplementedError):
        LatentAttnDecode(16, 0.1, latent_size=256)
    lat = LatentAttnDecode(16, 0.1)
    with pytest.raises(ValueError, match="16"):
        lat(a["lq"][:, :8], a["lat"], a["ctx"], a["bt"])
    with pytest.raises(RuntimeError, match="GPU only"):
        lat(a["lq"], a["lat"], a["ctx"], a["bt"])


def test_entry_points_compile():
    """Under torch.compile each method is its custom op, with no graph break."""
    from fastkernels_amd.candidate.L1.flash_attn_decode import FlashAttnDecode
    from fastkernels_amd.candidate.L1.latent_attn import LatentAttnDecode
    from fastkernels_amd.candidate.L1.rms_norm import RMSNorm
    from fastkernels_amd.candidate.L1.rotary_emb import RotaryEmbedding
    from fastkernels_amd.candidate.L1.store_kvcache import StoreKVCacheMxfp4

    a, calls = args(), []
    attn, lat, put = FlashAttnDecode(8, 2, 128), LatentAttnDecode(16, 0.1), StoreKVCacheMxfp4()
    rope = RotaryEmbedding(64, 32, 10000.0)
    norm = RMSNorm(512).to(BF)

    def backend(gm, _):
        calls.extend(str(n.target) for n in gm.graph.nodes if n.op == "call_function")
        outs = [n for n in gm.graph.nodes if n.op == "output"][0].args[0]
        return lambda *_: [torch.zeros(3, 8, 128)] * len(outs)

    def step(q, c, lq):
        put(a["key"], a["key"], a["cache"], a["slots"])
        o = attn.forward_mxfp4(q, a["cache"], a["ctx"], block_table=a["bt"])
        rope.forward_store_latent(a["pos"], a["qr"], c, a["kr"], a["lat"], a["slots"], norm,
                                  lq[:, :, 512:])
        return o, lat(lq, a["lat"], a["ctx"], a["bt"])

    torch.compile(step, backend=backend, fullgraph=True)(a["q"], a["c"], a["lq"])
    names = [c.split(".")[1] for c in calls if c.startswith("fastkernels_amd.")]
    assert names == ["store_kvcache_mxfp4", "mxfp4_paged_decode", "latent_norm_rope_store",
                     "latent_decode"]


def test_custom_ops_trace():
    """The ops are registered with in-place annotations and fake implementations."""
    a = {k: v.to("meta") for k, v in args().items() if k != "cache"}
    cache = [t.to("meta") for t in args()["cache"]]
    o = torch.ops.fastkernels_amd
    o.store_kvcache_mxfp4(a["key"], a["key"], *cache, a["slots"])
    o.gather_kvcache_mxfp4(a["key"], a["key"], *cache, a["bt"], a["cu"])
    o.mxfp4_paged_decode(a["q"], a["q"], *cache, a["bt"], a["ctx"], 0.1)
    o.latent_norm_rope_store(a["lat"], a["slots"], a["pos"], a["c"], a["kr"], a["cs"], True)
    o.gather_latent(torch.zeros(3, 576, dtype=BF, device="meta"), a["lat"], a["bt"], a["cu"])
    o.latent_decode(a["lo"], a["lq"], a["lat"], a["bt"], a["ctx"], 0.1)


# ---------------------------------------------------------------------------
# the definitions
# ---------------------------------------------------------------------------
def test_blocks_are_nearest():
    """No value is off by more than half a step of the grid at it (a quarter of the block's
    unit at least), and no other scale's grid of the same reach does better at the greatest."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 256)) * 2.0 ** rng.integers(-140, 120, (50, 1))
    x = x.astype(np.float32).astype(np.float64)
    x[0, :32] = 0
    s, c = ref.mxfp4_blocks(x)
    y = ref.mxfp4_values(s, c)
    unit = np.repeat(2.0 ** (s.astype(np.float64) - 127), 32, -1)
    a = np.abs(x) / unit
    assert (a.max() <= 7) and s[0, 0] == 0 and (y[0, :32] == 0).all()
    half = np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1.0))
    assert (np.abs(x - y) <= half * unit).all()
    every = np.abs(x[..., None]) / unit[..., None] - ref.GRID
    assert np.allclose(np.abs(every).min(-1) * unit, np.abs(x - y), atol=0)
    # a block's unit is the largest power of two that its greatest value fills: a quarter of the
    # value's power of two, after it is rounded to two significant bits
    for top, e in ((4.0, 127), (5.9, 127), (6.9, 127), (7.0, 128), (3.5, 127), (3.4, 126),
                   (1.0, 125), (2.0 ** -124, 1), (2.0 ** -130, 0)):
        assert ref.mxfp4_blocks(np.array([top] + [0.0] * 31))[0][0] == e
    # ties go to the even code; infinities and NaN take the whole block, and no other
    t = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] + [0.0] * 24)
    s, c = ref.mxfp4_blocks(np.concatenate([t, -t]))
    assert ref.mxfp4_values(s, c)[:8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6]
    assert ref.mxfp4_values(s, c)[32:39].tolist() == [0, -1, -1, -2, -2, -4, -4]
    for bad in (np.inf, -np.inf, np.nan):
        y = ref.mxfp4_values(*ref.mxfp4_blocks(np.concatenate([t, [bad], t[1:]])))
        assert np.isnan(y[32:]).all() and not np.isnan(y[:32]).any()


def test_greatest_blocks_stay_finite():
    """From 1.75 2^127 on values become 1.5 2^127: the next value of a greater scale is 2^128."""
    for top, scale, want in ((1.25 * 2.0 ** 127, 252, 1.0), (1.74 * 2.0 ** 127, 252, 1.5),
                             (1.75 * 2.0 ** 127, 252, 1.5), (3.0e38, 252, 1.5),
                             (float(np.finfo(np.float32).max), 252, 1.5),
                             (1.74 * 2.0 ** 126, 251, 0.75), (1.75 * 2.0 ** 126, 252, 1.0)):
        s, c = ref.mxfp4_blocks(np.array([top, -top] + [0.0] * 30))
        assert s[0] == scale and ref.mxfp4_values(s, c)[:2].tolist() == [want * 2.0 ** 127,
                                                                         -want * 2.0 ** 127]


def test_layouts():
    """The arrays of a cache, byte by byte."""
    rng = np.random.default_rng(1)
    nb, hk, page, d = 2, 3, 16, 128
    c = [rng.integers(0, 256, t.shape, np.uint8).astype(np.uint8)
         for t in ops.new_mxfp4_cache(nb, page, hk, d, "cpu")]
    c[2][1, 2, 3, 4] = 255
    k, v = ref.mxfp4_cache_values(*c)
    assert k.shape == v.shape == (nb, page, hk, d) and np.isnan(k[1, 4, 2, 96:]).all()
    for p, h, t, i in rng.integers(0, [nb, hk, page, d], (200, 4)):
        for x, byte, scale in ((k, c[0][p, h, t, i // 2], c[2][p, h, i // 32, t]),
                               (v, c[1][p, h, t // 4, i // 8, t % 4, i % 8 // 2],
                                c[3][p, h, i // 32, t])):
            code = int(byte >> 4 if i % 2 else byte & 15)
            want = (-1) ** (code >> 3) * ref.GRID[code & 7] * 2.0 ** (float(scale) - 127)
            assert x[p, t, h, i] == want or scale == 255


def test_definitions_agree_with_dense_attention():
    rng = np.random.default_rng(2)
    nb, page, hk, g, d = 9, 16, 2, 3, 64
    k, v = rng.standard_normal((2, nb, page, hk, d))
    bt = np.array([[3, 1, 7, 0], [8, -1, 4, 6]])
    q = rng.standard_normal((5, hk * g, d))
    out, _, _ = ref.paged_decode(q, k, v, bt, [55, 40], 0.1, 20, None, [0, 3, 4])
    assert np.isnan(out[4]).all()
    for t, b, hi in ((0, 0, 53), (1, 0, 54), (2, 0, 55), (3, 1, 40)):
        at = np.arange(max(0, hi - 21), hi)
        at = at[bt[b, at // page] >= 0]
        for h in range(hk * g):
            x = 0.1 * k[bt[b, at // page], at % page, h // g] @ q[t, h]
            w = np.exp(x) / np.exp(x).sum()
            assert np.allclose(out[t, h], w @ v[bt[b, at // page], at % page, h // g], atol=1e-12)
    # latent attention is that of one kv head whose values are the keys' first dims
    cache = rng.standard_normal((nb, page, 96))
    lq = rng.standard_normal((5, 4, 96))
    a, _, _, lse = ref.latent_decode(lq, cache, bt, [55, 40], 0.1, 64, [0, 3, 4])
    b, _, _ = ref.paged_decode(lq, cache[:, :, None], cache[:, :, None], bt, [55, 40], 0.1, -1,
                               None, [0, 3, 4])
    assert np.allclose(a, b[:, :, :64], atol=1e-12, equal_nan=True)
    x = 0.1 * lq[3] @ np.concatenate([cache[8], cache[4, :8]]).T
    assert np.allclose(lse[:, 3], np.log(np.exp(x).sum(1)), atol=1e-12)


def test_rows_and_rotations():
    rng = np.random.default_rng(3)
    cs = np.concatenate([np.cos(np.outer(np.arange(9), [1, .1])),
                         np.sin(np.outer(np.arange(9), [1, .1]))], 1)
    x = rng.standard_normal((3, 4))
    for neox in (False, True):
        y = ref.rotate(x, 5, cs, neox)
        pair = (lambda z, i: z[:, i] + 1j * z[:, i + 2]) if neox else \
            (lambda z, i: z[:, 2 * i] + 1j * z[:, 2 * i + 1])
        for i, f in enumerate([1, .1]):
            assert np.allclose(pair(y, i), pair(x, i) * np.exp(5j * f))
        assert (ref.rotate(x, 9, cs, neox) == x).all() and (ref.rotate(x, -1, cs, neox) == x).all()
    c, _ = ref.latent_rows(x, x, [0, 0, 0], cs, False, np.full(4, 2.0), 0.0)
    assert np.allclose((c ** 2).mean(-1), 4.0)
    cache = np.arange(2 * 16.0).reshape(2, 16, 1)
    got = ref.gather(cache, np.array([[1, 0], [-1, 1]]), [1, 19, 37], 40)
    assert np.isnan(got[[0, 37, 38, 39]]).all() and got[1, 0] == 16 and got[17, 0] == 0
    assert (got[19:35] == 0).all() and got[35, 0] == 16
