"""CPU tests of the 4-bit KV cache: the format's oracle against its definition, the op
schemas and fakes, the cache's allocation, argument errors of the launchers and of the C
entry points, and the attention's launch plan."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import fxpr_vllm  # noqa: F401
from fxpr_vllm import _hip, _lib
from fxpr_vllm._kernels import mx4
from oracle import mx4 as O

OPS = ("reshape_and_cache_mx4", "gather_cache_mx4", "unified_attention_mx4_fxp")


@pytest.mark.parametrize("d", mx4.HEAD_SIZES)
def test_oracle_pack_roundtrip(d):
    codes = np.random.default_rng(d).integers(0, 16, (7, d)).astype(np.uint8)
    data = O.pack(codes)
    assert data.shape == (7, d // 2) and np.array_equal(O.unpack(data), codes)
    # lane group kg's chunks 4 j + kg are its D / 8 consecutive bytes
    words = data.view("<u4")
    for c in range(d // 8):
        u = words[:, (c % 4) * (d // 32) + c // 4]
        for i in range(8):
            assert np.array_equal((u >> (4 * i)) & 15, codes[:, 8 * c + i])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_oracle_rounding(dtype):
    # a block pinned at scale 1 by a 6: every midpoint goes to the even code
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    want = [0, 2, 2, 4, 4, 6, 6]
    x = np.zeros((1, 64))
    x[0, 0] = 6.0
    x[0, 1:8], x[0, 8:15] = mids, [-m for m in mids]
    x[0, 15], x[0, 16], x[0, 17], x[0, 18] = np.nan, 7.0, np.nextafter(0.25, 1), np.nextafter(5.0, 6)
    codes, b = O.quantise(x, dtype)
    assert b[0, 0] == 127 and codes[0, 0] == 7
    assert codes[0, 1:8].tolist() == want and codes[0, 8:15].tolist() == [c | 8 for c in want]
    assert codes[0, 15] == 0 and codes[0, 16] == 7 and codes[0, 17] == 1 and codes[0, 18] == 7
    # the scale: amax / s in (3.5, 7]
    for amax, s in [(3.5, 0.5), (3.500001, 1.0), (7.0, 1.0), (7.00001, 2.0), (1.0, 0.25)]:
        x = np.full((1, 32), amax)
        assert 2.0 ** (int(O.quantise(x, dtype)[1][0, 0]) - 127) == s
    lo, hi = O.BYTES[dtype]
    assert O.quantise(np.full((1, 32), 0.0), dtype)[1][0, 0] == lo
    assert O.quantise(np.full((1, 32), np.inf), dtype)[1][0, 0] == hi
    # every value a writer can leave is one of the type
    t = {"f16": np.float16, "f32": np.float32}.get(dtype)
    all_codes = np.tile(np.arange(16, dtype=np.uint8), (hi - lo + 1, 2))
    v = O.values(all_codes, np.arange(lo, hi + 1, dtype=np.uint8)[:, None], dtype)
    assert np.isfinite(v).all()
    if t is not None:
        assert np.array_equal(v.astype(t).astype(np.float64), v)
    else:
        assert torch.equal(torch.from_numpy(v).to(torch.bfloat16).double(), torch.from_numpy(v))
    assert np.array_equal(O.values(all_codes[:1], np.array([[255]], np.uint8), dtype), v[-1:])


def test_schemas_and_fakes():
    for op in OPS:
        assert torch._C._dispatch_has_kernel_for_dispatch_key("fxpr::" + op, "CUDA")
    assert str(torch.ops.fxpr.unified_attention_mx4_fxp.default._schema) == (
        "fxpr::unified_attention_mx4_fxp(Tensor q, Tensor kv_codes, Tensor kv_scales, Tensor(a!) o, "
        "Tensor query_start_loc, Tensor seq_lens, Tensor block_table, int max_query_len, Tensor? alibi_slopes, "
        "bool is_causal, float? softmax_scale, int fxp_int_bits, int fxp_frac_bits, float logit_softcap, "
        "int window_size, int num_kv_splits) -> ()")
    codes, scales = mx4.empty_cache(4, 16, 2, 128, "meta")
    slots = torch.empty(5, dtype=torch.int64, device="meta")
    k, v = torch.ops.fxpr.gather_cache_mx4(codes, scales, slots, torch.float16)
    assert k.shape == v.shape == (5, 2, 128) and k.dtype == v.dtype == torch.float16
    rows = torch.empty(5, 2, 128, device="meta")
    assert torch.ops.fxpr.reshape_and_cache_mx4(rows, rows, codes, scales, slots) is None


@pytest.mark.parametrize("d", mx4.HEAD_SIZES)
def test_empty_cache(d):
    codes, scales = mx4.empty_cache(3, 32, 4, d, "cpu")
    assert codes.shape == (3, 2, 32, 4, d // 2) and scales.shape == (3, 2, 32, 4, d // 32)
    assert codes.stride(4) == scales.stride(4) == 1
    assert codes.untyped_storage().nbytes() == 3 * 2 * 32 * 4 * d * 17 // 32
    assert codes.untyped_storage().data_ptr() == scales.untyped_storage().data_ptr()
    # no byte belongs to two rows
    codes.fill_(0)
    scales.fill_(1)
    assert int(codes.sum()) == 0 and int(scales.sum()) == scales.numel()
    assert all(s % 16 == 0 for s in codes.stride()[:4]) and all(s % (d // 32) == 0 for s in scales.stride()[:4])
    for bad in ((3, 32, 4, 96), (3, 24, 4, d), (3, 32, 0, d), (-1, 32, 4, d)):
        with pytest.raises(ValueError):
            mx4.empty_cache(*bad, "cpu")


def test_launchers_refuse_host_tensors():
    codes, scales = mx4.empty_cache(4, 16, 2, 64, "cpu")
    x = torch.zeros(3, 2, 64)
    slots = torch.arange(3)
    i32 = torch.zeros(4, dtype=torch.int32)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        _lib._reshape_and_cache_mx4_cuda(x, x, codes, scales, slots)
    with pytest.raises(RuntimeError, match="CUDA"):
        _lib._gather_cache_mx4_cuda(codes, scales, slots, torch.float32)
    with pytest.raises(RuntimeError, match="CUDA"):
        _lib._unified_attention_mx4_fxp_cuda(q, codes, scales, q, i32, i32[:3], i32, 1, None, True, None, 32, 16, 0.0, 0, 0)
    with pytest.raises(ValueError, match="int_bits"):
        _lib._unified_attention_mx4_fxp_cuda(q, codes, scales, q, i32, i32[:3], i32, 1, None, True, None, 24, 16, 0.0, 0, 0)


P = ctypes.c_void_p(256)


def _attn(**kw):
    a = dict(q=P, codes=P, scales=P, o=P, dt=1, qsl=P, sl=P, bt=P, alibi=None, reqs=1, tokens=1, hq=8, hk=2, d=128,
             page=16, mq=1, mb=4, nb=8, sqt=1024, sqh=128, scb=4096, sch=2048, scs=128, scd=64, ssb=256, ssh=128, sss=8,
             ssd=4, sot=1024, soh=128, sbt=4, causal=1, scale=1.0, cap=0.0, win=0, ib=32, fb=16, splits=0, ws=None,
             wsb=0, st=None)
    a.update(kw)
    return _hip.load().fxpr_unified_attention_mx4(*a.values())


def test_c_abi_refusals_attention():
    # every refusal comes before any launch (there is no device here)
    assert _attn(reqs=0) == 0 and _attn(tokens=0) == 0
    assert _attn(ib=24) == -2 and _attn(fb=64) == -2 and _attn(fb=-1) == -2
    assert _attn(dt=2) == -1 and _attn(dt=9) == -1
    for bad in (dict(d=96), dict(d=32), dict(page=8), dict(page=48), dict(hk=3), dict(hk=0), dict(reqs=-1),
                dict(tokens=-1), dict(splits=-1), dict(mb=0), dict(nb=0), dict(page=1 << 20, mb=1 << 12),
                dict(tokens=1 << 31), dict(tokens=1 << 30, hq=1 << 12, hk=1)):
        assert _attn(**bad) == -3, bad
    for bad in (dict(q=None), dict(codes=None), dict(scales=None), dict(o=None), dict(qsl=None), dict(sl=None),
                dict(bt=None), dict(sqt=1020), dict(sqh=4), dict(scb=4100), dict(scs=8), dict(ssb=258), dict(scs=-16),
                dict(scb=1 << 33), dict(scs=1 << 28), dict(q=ctypes.c_void_p(264)), dict(codes=ctypes.c_void_p(264)),
                dict(scales=ctypes.c_void_p(258))):
        assert _attn(**bad) == -5, bad
    # a split launch without its workspace
    need = _hip.load().fxpr_attention_mx4_plan(1, 1, 8, 2, 128, 16, 1, 4096, 0, 32, 4, None)
    assert need > 0
    assert _attn(mb=4096, splits=4) == -4
    assert _attn(mb=4096, splits=4, ws=P, wsb=need - 1) == -4


def test_c_abi_refusals_cache():
    lib = _hip.load()

    def write(**kw):
        a = dict(k=P, v=P, c=P, s=P, dt=1, slots=P, t=4, h=2, d=128, page=16, nb=8, skt=256, skh=128, svt=256, svh=128,
                 cb=4096, ch=2048, cs=128, cd=64, sb=256, sh=128, ss=8, sd=4, st=None)
        a.update(kw)
        return lib.fxpr_reshape_and_cache_mx4(*a.values())

    def gather(**kw):
        a = dict(c=P, s=P, k=P, v=P, dt=1, slots=P, t=4, h=2, d=128, page=16, nb=8, cb=4096, ch=2048, cs=128, cd=64,
                 sb=256, sh=128, ss=8, sd=4, st=None)
        a.update(kw)
        return lib.fxpr_gather_cache_mx4(*a.values())

    for f in (write, gather):
        assert f(t=0) == 0
        assert f(dt=3) == -1 and f(dt=4) == -1
        for bad in (dict(d=32), dict(d=96), dict(d=512), dict(h=0), dict(page=0), dict(t=-1), dict(nb=-1), dict(t=1 << 40)):
            assert f(**bad) == -3, bad
        for bad in (dict(k=None), dict(v=None), dict(c=None), dict(s=None), dict(slots=None), dict(cb=8), dict(cd=4),
                    dict(ss=2), dict(k=ctypes.c_void_p(264)), dict(c=ctypes.c_void_p(260))):
            assert f(**bad) == -5, bad
    assert write(skt=129) == -5 and write(svh=4) == -5
    assert write(nb=0) == 0  # no slot exists: every one is padding


def test_c_abi_refuses_what_its_indices_do_not_hold():
    lib = _hip.load()
    for t, h in (((1 << 30) + 1, 1), ((1 << 29) + 1, 2), ((1 << 26) + 1, 16)):
        assert lib.fxpr_gather_cache_mx4(P, P, P, P, 1, P, t, h, 128, 16, 8, 4096, 2048, 128, 64, 256, 128, 8, 4, None) == -3
        assert lib.fxpr_reshape_and_cache_mx4(P, P, P, P, 1, P, t, h, 128, 16, 8, 0, 0, 0, 0, 4096, 2048, 128, 64, 256, 128,
                                              8, 4, None) == -3
    need = lib.fxpr_attention_mx4_plan(1, 1, 8, 2, 128, 16, 1, 4096, 0, 32, 4, None)
    assert _attn(mb=4096, splits=4, ws=ctypes.c_void_p(264), wsb=need) == -4  # not 16-byte aligned


def plan(reqs, tokens, hq, hk, d, page, mq, mb, window=0, bits=32, splits=0):
    out = (ctypes.c_int32 * 4)()
    n = _hip.load().fxpr_attention_mx4_plan(reqs, tokens, hq, hk, d, page, mq, mb, window, bits, splits, out)
    return n, tuple(out)


def test_plan():
    # nothing for what the launch refuses
    assert plan(1, 1, 8, 3, 128, 16, 1, 4) == (0, (0, 0, 0, 0))
    assert plan(1, 1, 8, 2, 96, 16, 1, 4)[0] == 0 and plan(0, 0, 8, 2, 128, 16, 1, 4)[0] == 0
    # one short request: no split, no workspace
    n, p = plan(1, 1, 32, 8, 128, 16, 1, 4)
    assert n == 0 and p == (0, 1, 1, 0)
    # an explicit count is capped at the chunks a table row holds; its records fit the workspace
    n, p = plan(2, 2, 32, 8, 128, 16, 1, 128, splits=1000)
    assert p[2] == 4 and n >= 2 * 32 * (8 + 4 * (4 + 4 + 4 * 128))
    # prompts: 64-row workgroups; only short requests' tokens keep records where those alone are split
    n, p = plan(33, 32 + 4096, 32, 8, 128, 16, 4096, 2048)
    assert p[0] == 1
    if p[1] == 1 and p[2] > 1:
        assert 1 <= p[3] <= 11 and n <= 33 * p[3] * 32 * (8 + 64 * (8 + 512)) + 1024
    # the workspace never passes 1 GiB
    for reqs in (1, 16, 256, 4096):
        for mb in (64, 1024, 65536):
            for mq in (1, 7, 100, 3000):
                assert plan(reqs, reqs * mq, 64, 8, 128, 16, mq, mb)[0] <= 1 << 30
