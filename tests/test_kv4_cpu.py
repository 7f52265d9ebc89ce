"""No-GPU checks of the 4-bit K/V cache: the entry points refuse bad arguments before any launch, the Python wrappers
refuse tensors of the wrong kind, and the oracle's format agrees with the NVFP4 codec pinned to the reference."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import kv4_ref as K
from oracle import nvfp4_ref as N


@pytest.fixture(scope="module")
def lib():
    from muse_spark_open_challenge_b200 import build, _lib
    build.build()
    return _lib.load()


FAKE, NULL = ctypes.c_void_p(1 << 20), None


def test_oracle_quantiser_is_the_nvfp4_codec_and_rounds_to_nearest_even():
    g = torch.Generator().manual_seed(0)
    z = torch.randn((50, 3, 64), generator=g, dtype=torch.float64)
    codes, sf = K.quantise(z, 0.37)
    back = K.dequantise(codes, sf, 0.37)
    theirs = N.dequantize(codes.numpy(), sf.view(torch.uint8).numpy(), 0.37)
    assert np.allclose(back.numpy(), theirs, rtol=2 ** -22)
    # every code is the nearest grid point: the error is at most half the gap around it (1 at the top: 4 .. 6)
    unit = (sf.double() * 0.37).repeat_interleave(16, -1)
    assert ((back - z).abs() <= unit * (1 + 1e-12)).all()
    # ties go to the even code: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -6.0])
    codes, sf = K.quantise(ties.double()[None], 1.0)
    assert float(sf.double()) == 1.0
    assert K.dequantise(codes, sf, 1.0)[0].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 0, -1, -1, -2, -2, -4, -4, -6]
    codes, sf = K.quantise(torch.full((1, 16), 2.0 ** -14).double(), 1.0)       # below half the smallest scale: all zero
    assert int(codes.max()) == 0 and int(sf.view(torch.uint8)) == 0


def test_page_plan_refuses(lib):
    def call(**kw):
        a = dict(new=FAKE, seq=FAKE, table=FAKE, max_pages=4, free=FAKE, n_free=4, head=FAKE, out=ctypes.c_void_p(4096),
                 batch=2, page=16, tokens=8, cu=FAKE, pos=FAKE, loc=FAKE)
        a.update(kw)
        return lib.msl_page_plan(a["new"], a["seq"], a["table"], a["max_pages"], a["free"], a["n_free"], a["head"],
                                 a["out"], a["batch"], a["page"], a["tokens"], a["cu"], a["pos"], a["loc"], NULL, NULL)
    for name in ("new", "seq", "table", "free", "head", "out", "cu", "pos", "loc"):
        assert call(**{name: NULL}) == -1, name
    assert call(batch=0) == -1 and call(page=0) == -1 and call(max_pages=0) == -1 and call(tokens=-1) == -1
    assert call(n_free=-1) == -1 and call(out=FAKE) == -1            # the new head must be another word
    assert call(batch=16385) == -7


def test_store_refuses(lib):
    def call(**kw):
        a = dict(qkv=FAKE, ld=12 * 64, pos=FAKE, loc=FAKE, ks=FAKE, vs=FAKE, q=FAKE, k=FAKE, kf=FAKE, v=FAKE, vf=FAKE,
                 tokens=3, hq=8, hkv=2, dim=64, rows=64)
        a.update(kw)
        return lib.msl_qk_rope_store_kv4(a["qkv"], a["ld"], a["pos"], a["loc"], NULL, a["ks"], a["vs"], a["q"], a["k"],
                                         a["kf"], a["v"], a["vf"], a["tokens"], a["hq"], a["hkv"], a["dim"], a["rows"],
                                         NULL, NULL)
    for name in ("qkv", "pos", "loc", "ks", "vs", "q", "k", "kf", "v", "vf"):
        assert call(**{name: NULL}) == -1, name
    assert call(ld=12 * 64 - 8) == -1 and call(tokens=-1) == -1 and call(hq=0) == -1 and call(rows=0) == -1
    assert call(dim=96) == -7 and call(ld=12 * 64 + 4) == -2 and call(qkv=ctypes.c_void_p((1 << 20) + 8)) == -2
    assert call(tokens=0) == 0


def test_rows_refuses(lib):
    def call(**kw):
        a = dict(codes=FAKE, sf=FAKE, scale=FAKE, rows=FAKE, n=4, width=128, have=64, mode=0, out=FAKE)
        a.update(kw)
        return lib.msl_kv4_rows(a["codes"], a["sf"], a["scale"], a["rows"], a["n"], a["width"], a["have"], a["mode"],
                                a["out"], NULL, NULL)
    for name in ("codes", "sf", "scale", "rows", "out"):
        assert call(**{name: NULL}) == -1, name
    assert call(n=-1) == -1 and call(mode=2) == -1 and call(width=24) == -2 and call(have=0) == -1 and call(n=0) == 0


def attention_call(lib, **kw):
    a = dict(q=FAKE, ld_q=512, k=FAKE, kf=FAKE, v=FAKE, vf=FAKE, table=FAKE, max_pages=4, seq=FAKE, cu=FAKE, ks=FAKE,
             vs=FAKE, scale=0.125, batch=2, longest=3, tokens=6, hq=8, hkv=2, dim=64, page=16, window=0, rows=64, out=FAKE, ld_out=512,
             gate=NULL, ld_gate=0, work=FAKE, bytes=None)
    a.update(kw)
    if a["bytes"] is None:
        a["bytes"] = lib.msl_attention_kv4_workspace(a["batch"], a["longest"], a["tokens"], a["hq"], a["hkv"], a["dim"],
                                                     a["max_pages"], a["page"], a["window"])
    return lib.msl_attention_kv4(a["q"], a["ld_q"], a["k"], a["kf"], a["v"], a["vf"], a["table"], a["max_pages"], a["seq"],
                                 a["cu"], a["ks"], a["vs"], a["scale"], a["batch"], a["longest"], a["tokens"], a["hq"],
                                 a["hkv"], a["dim"], a["page"], a["window"], a["rows"], a["out"], a["ld_out"], a["gate"],
                                 a["ld_gate"], a["work"], a["bytes"], NULL, NULL)


def test_attention_refuses(lib):
    for name in ("q", "k", "kf", "v", "vf", "table", "seq", "cu", "ks", "vs", "out", "work"):
        assert attention_call(lib, **{name: NULL}) == -1, name
    for name, bad in (("batch", 0), ("longest", 0), ("tokens", -1), ("hq", 7), ("hkv", 0), ("page", 0), ("window", -1),
                      ("rows", 0), ("rows", 1 << 31), ("max_pages", 0), ("ld_q", 504), ("ld_out", 504), ("scale", 0.0), ("scale", -1.0),
                      ("scale", float("nan"))):
        assert attention_call(lib, bytes=1 << 30, **{name: bad}) == -1, name
    assert attention_call(lib, gate=FAKE, ld_gate=504) == -1
    assert attention_call(lib, dim=96, bytes=1 << 30, ld_q=768, ld_out=768) == -7
    assert attention_call(lib, hq=258, ld_q=258 * 64, ld_out=258 * 64) == -7            # 129 query heads a KV head
    odd = ctypes.c_void_p((1 << 20) + 4)
    for name in ("q", "k", "v", "kf", "vf", "out", "work"):
        assert attention_call(lib, **{name: odd}) == -2, name
    assert attention_call(lib, ld_q=516) == -2 and attention_call(lib, ld_out=516) == -2
    assert attention_call(lib, bytes=15) == -6
    assert attention_call(lib, tokens=0) == 0


def test_wrappers_refuse_cpu_tensors():
    from muse_spark_open_challenge_b200 import ops
    from muse_spark_open_challenge_b200._lib import MslError
    i32, one = torch.zeros(4, dtype=torch.int32), torch.ones(())
    with pytest.raises(MslError):
        ops.page_plan(i32, i32, i32.view(4, 1), i32, i32[:1], 16, 8)
    codes, sf = torch.zeros((4, 16, 2, 32), dtype=torch.uint8), torch.zeros((4, 16, 2, 4)).to(K.FP8)
    with pytest.raises(MslError):
        ops.kv4_rows(codes, sf, one, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(MslError):
        ops.qk_rope_store_kv4(torch.zeros((1, 768)).bfloat16(), torch.zeros(1).long(), torch.zeros(1).long(), None, one,
                              one, codes, sf, codes, sf, 8, 2, 64)
    with pytest.raises(MslError):
        ops.attention_kv4(torch.zeros((1, 8, 64)).bfloat16(), codes, sf, codes, sf, i32.view(1, 4), i32[:1], i32[:2], one,
                          one, 0.1, 1, 1, 8, 2, 64, 16, 0)


def test_synthetic_cache_has_the_documented_layout():
    from muse_spark_open_challenge_b200 import synth
    c = synth.kv4_cache(synth.TINY, 5, 16, seed=3)
    assert c["k_cache"].shape == (5, 16, 2, 32) and c["k_cache_sf"].shape == (5, 16, 2, 4)
    assert c["v_cache_sf"].dtype == torch.float8_e4m3fn and torch.isfinite(c["v_cache_sf"].float()).all()
    v = K.dequantise(c["v_cache"], c["v_cache_sf"], 1.0)
    assert 0.5 < float(v.std()) < 2.0


@pytest.mark.parametrize("what", ["codes with scales", "codes alone", "one cache of codes", "half a cache"])
def test_c_host_binding_refuses_what_is_not_an_fp8_cache(what):
    """`clayer.kernel_fn` passes addresses on: an FP8 store into 4-bit codes, or into fewer rows than the configuration
    says, would write past the caches.  The state is empty, so anything but the refusal would be another error."""
    from muse_spark_open_challenge_b200 import clayer, synth
    from muse_spark_open_challenge_b200._lib import MslError
    shape = synth.TINY
    data = synth.make_input(shape, [3], [5], seed=1, page=16)
    config = clayer.Config()
    config.hkv, config.head_dim = shape.hkv, shape.head_dim
    config.cache_rows = data["k_cache"].numel() // (shape.hkv * shape.head_dim)
    with pytest.raises(KeyError):                    # this one is taken, as far as the empty state
        clayer.kernel_fn(data, {}, config)
    codes = synth.kv4_cache(shape, data["k_cache"].shape[0], 16, seed=1)
    if what == "codes with scales":
        data.update(codes)
    elif what == "codes alone":
        data["k_cache"], data["v_cache"] = codes["k_cache"], codes["v_cache"]
    elif what == "one cache of codes":
        data["v_cache"] = codes["v_cache"]
    else:
        data["v_cache"] = data["v_cache"][:data["v_cache"].shape[0] // 2]
    with pytest.raises(MslError, match="cache"):
        clayer.kernel_fn(data, {}, config)
