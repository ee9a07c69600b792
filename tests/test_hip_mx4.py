"""GPU tests of the KV cache in 4 bits: the quantising write and the read back bit for bit
against the oracle, attention against the formula in 64 bits (within bounds derived from
the roundings it makes) and bit for bit against unified_attention_fxp over a cache of the
values the codes stand for."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import fxpr_vllm  # noqa: F401
from fxpr_vllm._kernels import mx4
from oracle import mx4 as O

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
NAME = {HF: "f16", BF: "bf16", FP: "f32"}
ops = torch.ops.fxpr


def randn(*shape, seed=0, dtype=FP):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def new_cache(blocks, page, heads, d, order="heads", seed=None):
    """A cache on the GPU: every byte random where a seed is given (whatever a fresh page may hold), else zeros."""
    if order == "heads":
        c, s = mx4.empty_cache(blocks, page, heads, d, "cuda")
    else:  # slots before heads, each tensor contiguous
        c = torch.empty(blocks, 2, page, heads, d // 2, dtype=torch.uint8, device="cuda")
        s = torch.empty(blocks, 2, page, heads, d // 32, dtype=torch.uint8, device="cuda")
    if seed is None:
        c.zero_()
        s.zero_()
    else:
        g = torch.Generator().manual_seed(seed)
        c.copy_(torch.randint(0, 256, c.shape, generator=g, dtype=torch.uint8))
        s.copy_(torch.randint(0, 256, s.shape, generator=g, dtype=torch.uint8))
    return c, s


def awkward(t, dtype):
    """Rows with zeros, one outlier, infinities, NaN, the type's extremes and subnormals among normal ones."""
    x = t.clone()
    f = torch.finfo(dtype)
    flat = x.view(-1, x.shape[-1])
    n = flat.shape[0]
    special = [0.0, -0.0, math.inf, -math.inf, math.nan, f.max, f.min, f.tiny, f.tiny * f.eps, 6.5, 7.0]
    for i, v in enumerate(special):
        flat[i % n, (5 * i) % flat.shape[1]] = v
    flat[(len(special)) % n] = 0.0
    flat[(len(special) + 1) % n] *= f.tiny
    flat[(len(special) + 2) % n] *= 2.0 ** 12
    return x.to(dtype)


# ---------------------------------------------------------------------------
# Write and read back.


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("d,heads,page,tokens,order", [(128, 8, 16, 37, "heads"), (64, 3, 32, 1, "slots"),
                                                       (256, 2, 16, 130, "heads"), (128, 1, 24, 65, "slots"),
                                                       (64, 16, 64, 300, "heads")])
def test_write_is_the_oracles_bytes(dtype, d, heads, page, tokens, order):
    blocks = tokens // page + 3
    codes, scales = new_cache(blocks, page, heads, d, order, seed=5)
    c0, s0 = codes.cpu(), scales.cpu()
    g = torch.Generator().manual_seed(tokens)
    slots = torch.randperm(blocks * page, generator=g)[:tokens]
    if tokens > 4:  # padding and slots past the cache leave everything as it is
        slots[1], slots[tokens // 2], slots[-1] = -1, blocks * page, 1 << 40
    key, value = (awkward(randn(tokens, heads, d, seed=i, dtype=dtype), dtype) for i in (1, 2))
    ops.reshape_and_cache_mx4(key.cuda(), value.cuda(), codes, scales, slots.cuda())
    live = (slots >= 0) & (slots < blocks * page)
    blk, off = slots[live] // page, slots[live] % page
    for half, x in enumerate((key, value)):
        want_c, want_s = O.quantise(x[live].double().numpy(), NAME[dtype])
        c0[blk, half, off] = torch.from_numpy(O.pack(want_c))
        s0[blk, half, off] = torch.from_numpy(want_s)
    # (the codes of zeros may carry either sign: -0 is a zero)
    assert torch.equal(scales.cpu(), s0)
    got, want = O.unpack(codes.cpu().numpy()), O.unpack(c0.numpy())
    assert np.array_equal(np.where(got == 8, 0, got), np.where(want == 8, 0, want))
    # read back: exactly the values, zeros for slots outside the cache
    k, v = ops.gather_cache_mx4(codes, scales, slots.cuda(), dtype)
    for half, y in enumerate((k, v)):
        w = np.zeros((tokens, heads, d))
        w[live.numpy()] = O.values(O.unpack(c0[blk, half, off].numpy()), s0[blk, half, off].numpy(), NAME[dtype])
        assert np.array_equal(y.cpu().double().numpy(), w)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_read_back_of_every_byte(dtype):
    # every code under every scale byte, in both nibbles
    codes, scales = new_cache(16, 16, 1, 64)
    c = torch.arange(256, dtype=torch.uint8).view(16, 16)
    codes[:, 0, :, 0, :] = c[:, :, None].expand(16, 16, 32).cuda()
    codes[:, 1] = codes[:, 0].flip(0)
    scales[:, 0, :, 0, :] = torch.arange(256, dtype=torch.uint8).view(16, 16, 1).expand(16, 16, 2).cuda()
    for b in range(0, 256, 5):
        scales[:, 1] = b
        k, v = ops.gather_cache_mx4(codes, scales, torch.arange(256, device="cuda"), dtype)
        for half, y in enumerate((k, v)):
            want = O.values(O.unpack(codes[:, half].reshape(256, 1, 32).cpu().numpy()),
                            scales[:, half].reshape(256, 1, 2).cpu().numpy(), NAME[dtype])
            got = y.cpu()
            assert bool(torch.isfinite(got).all())
            assert torch.equal(got.double(), torch.from_numpy(want).to(dtype).double())


def test_write_takes_views_and_flat_rows():
    d, heads, page, tokens = 128, 4, 16, 21
    qkv = randn(tokens, 12 * d, seed=3, dtype=BF).cuda()
    key, value = qkv[:, 4 * d : 8 * d], qkv[:, 8 * d :]
    slots = torch.arange(tokens, dtype=torch.int32, device="cuda") * 2
    want = new_cache(4, page, heads, d)
    ops.reshape_and_cache_mx4(key.reshape(tokens, heads, d).contiguous(), value.reshape(tokens, heads, d).contiguous(),
                              *want, slots)
    odd = torch.empty(tokens, heads, d + 1, dtype=BF, device="cuda")  # rows off 16 bytes
    odd[..., 1:] = key.reshape(tokens, heads, d)
    t = value.reshape(tokens, heads, d).transpose(1, 2).contiguous().transpose(1, 2)  # no unit stride along a row
    for k, v in ((key, value), (key.view(tokens, heads, d), value.view(tokens, heads, d)), (odd[..., 1:], t)):
        got = new_cache(4, page, heads, d)
        ops.reshape_and_cache_mx4(k, v, *got, slots)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_empty_and_all_padding():
    codes, scales = new_cache(2, 16, 2, 64, seed=1)
    c0, s0 = codes.clone(), scales.clone()
    x = randn(5, 2, 64, dtype=HF).cuda()
    ops.reshape_and_cache_mx4(x[:0], x[:0], codes, scales, torch.empty(0, dtype=torch.int64, device="cuda"))
    ops.reshape_and_cache_mx4(x, x, codes, scales, torch.full((9,), -1, device="cuda"))
    assert torch.equal(codes, c0) and torch.equal(scales, s0)
    k, v = ops.gather_cache_mx4(codes, scales, torch.empty(0, dtype=torch.int64, device="cuda"), HF)
    assert k.shape == v.shape == (0, 2, 64)
    k, v = ops.gather_cache_mx4(codes, scales, torch.full((3,), -1, device="cuda"), FP)
    assert not k.any() and not v.any()
    none = mx4.empty_cache(0, 16, 2, 64, "cuda")
    ops.reshape_and_cache_mx4(x, x, *none, torch.arange(5, device="cuda"))
    k, v = ops.gather_cache_mx4(*none, torch.arange(5, device="cuda"), BF)
    assert k.shape == (5, 2, 64) and not k.any() and not v.any()


def test_offsets_past_32_bits():
    # a cache of over 4 GiB of codes: its last blocks hold what a small one would
    heads, d, page = 8, 256, 16
    blocks = (5 << 30) // (2 * heads * page * d // 2)
    codes, scales = mx4.empty_cache(blocks, page, heads, d, "cuda")
    small = mx4.empty_cache(4, page, heads, d, "cuda")
    x, y = randn(40, heads, d, seed=1, dtype=BF).cuda(), randn(40, heads, d, seed=2, dtype=BF).cuda()
    at = torch.arange(40, device="cuda")
    far = at + (blocks - 4) * page
    ops.reshape_and_cache_mx4(x, y, codes, scales, far)
    ops.reshape_and_cache_mx4(x, y, *small, at)
    for a, b in zip(ops.gather_cache_mx4(codes, scales, far, BF), ops.gather_cache_mx4(*small, at, BF)):
        assert torch.equal(a, b)
    q = randn(2, 16, d, seed=3, dtype=BF).cuda()
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    outs = []
    for cache, first in (((codes, scales), blocks - 4), (small, 0)):
        o = torch.zeros_like(q)
        bt = (torch.arange(3, dtype=torch.int32, device="cuda") + first).repeat(2, 1)
        ops.unified_attention_mx4_fxp(q, *cache, o, i(0, 1, 2), i(40, 17), bt, 1, None, True, None, 32, 16, 0.0, 0, 0)
        outs.append(o)
    assert torch.equal(outs[0], outs[1]) and bool(outs[0].any())


# ---------------------------------------------------------------------------
# Attention.


class Batch:
    """Requests of (new tokens, context) over a filled cache, on the GPU; the values it stands for, on the CPU."""

    def __init__(self, reqs, hq, hk, d, page=16, dtype=BF, order="heads", seed=0, spare=3, garbage=True):
        self.reqs, self.hq, self.hk, self.d, self.page, self.dtype = reqs, hq, hk, d, page, dtype
        g = torch.Generator().manual_seed(seed)
        need = [-(-max(c, 1) // page) for _, c in reqs]
        self.width = max(need)
        blocks = sum(need) + spare
        # unwritten rows hold any bytes
        self.codes, self.scales = new_cache(blocks, page, hk, d, order, seed=seed + 1 if garbage else None)
        perm = torch.randperm(blocks, generator=g)
        self.table = torch.randint(-5, blocks + 5, (len(reqs), self.width), generator=g).to(torch.int32)
        slots, at = [], 0
        for r, (_, ctx) in enumerate(reqs):
            self.table[r, : need[r]] = perm[at : at + need[r]]
            at += need[r]
            p = torch.arange(ctx)
            slots.append(self.table[r].long()[p // page] * page + p % page)
        self.slots = slots
        n = sum(c for _, c in reqs)
        self.key = torch.randn(n, hk, d, generator=g).to(dtype)
        self.value = (torch.randn(n, hk, d, generator=g) + 0.1).to(dtype)
        if n:
            ops.reshape_and_cache_mx4(self.key.cuda(), self.value.cuda(), self.codes, self.scales, torch.cat(slots).cuda())
        starts = [0]
        for m, _ in reqs:
            starts.append(starts[-1] + m)
        self.qsl = torch.tensor(starts, dtype=torch.int32)
        self.lens = torch.tensor([c for _, c in reqs], dtype=torch.int32)
        self.q = torch.randn(starts[-1], hq, d, generator=g).to(dtype)
        self.max_q = max([m for m, _ in reqs] + [1])

    def values(self):
        """K and V [tokens, hk, d] float64 of each request's rows in the cache, from its bytes."""
        c, s = self.codes.cpu().numpy(), self.scales.cpu().numpy()
        out = []
        for slots in self.slots:
            blk, off = (slots // self.page).numpy(), (slots % self.page).numpy()
            out.append([O.values(O.unpack(c[blk, h, off]), s[blk, h, off], NAME[self.dtype]) for h in (0, 1)])
        return out

    def run(self, splits=0, causal=True, scale=None, softcap=0.0, window=0, slopes=None, ib=32, fb=16, max_q=None, o=None,
            q=None):
        o = torch.full(self.q.shape, 7.0, dtype=self.dtype, device="cuda") if o is None else o
        ops.unified_attention_mx4_fxp(
            self.q.cuda() if q is None else q, self.codes, self.scales, o, self.qsl.cuda(), self.lens.cuda(),
            self.table.cuda(), self.max_q if max_q is None else max_q, None if slopes is None else slopes.cuda(), causal,
            scale, ib, fb, softcap, window, splits)
        return o

    def over_floats(self, splits=0, causal=True, scale=None, softcap=0.0, window=0, slopes=None, ib=32, fb=16):
        """unified_attention_fxp over a cache of the values."""
        blocks = self.codes.shape[0]
        every = torch.arange(blocks * self.page, device="cuda")
        k, v = ops.gather_cache_mx4(self.codes, self.scales, every, self.dtype)
        kv = torch.stack([x.view(blocks, self.page, self.hk, self.d) for x in (k, v)], 1)
        o = torch.full(self.q.shape, 7.0, dtype=self.dtype, device="cuda")
        ops.unified_attention_fxp(self.q.cuda(), kv, o, self.qsl.cuda(), self.lens.cuda(), self.table.cuda(), self.max_q,
                                  None if slopes is None else slopes.cuda(), causal, scale, ib, fb, softcap, window, splits)
        return o

    def formula(self, causal=True, scale=None, softcap=0.0, window=0, slopes=None, fb=16):
        """The outputs in 64 bits, and how far the kernel's may be from them.

        With w the weights against the row's maximum (the largest is 1), S their sum and A = sum w |v| / S, the
        kernel rounds: a score's D products and D sums in 32 bits (D 2^-24 sum |q k| scale) and a few more
        operations on it (|s| 2^-22; the softcap's exp2, quotients and product: 2^-20 of the cap; ALiBi's product
        and sum: 2^-22 of its term); each weight to the type (eps / 2) for its product with V and to 2^-f / 2 for
        the sum S; each 64-key tile's product, and a chunk's sums once or twice as they are folded, to 2^-f / 2 (the
        folded terms shrink by powers of at most 1); 64 additions in 32 bits per tile (64 2^-24 A S); the quotient
        to the type. exp2 is off by 2^-22 relative."""
        d, eps, step = self.d, torch.finfo(self.dtype).eps, 2.0 ** -fb
        scale = 1.0 / math.sqrt(d) if scale is None else scale
        out, tol = (torch.zeros(self.q.shape, dtype=torch.float64) for _ in range(2))
        for r, ((m, ctx), (k, v)) in enumerate(zip(self.reqs, self.values())):
            if m == 0 or ctx == 0:
                continue
            a = int(self.qsl[r])
            rep = self.hq // self.hk
            q = self.q[a : a + m].double().permute(1, 0, 2)
            k, v = (torch.from_numpy(x).permute(1, 0, 2).repeat_interleave(rep, 0) for x in (k, v))
            x = q @ k.transpose(1, 2) * scale
            err = (q.abs() @ k.abs().transpose(1, 2) * abs(scale)) * d * 2.0 ** -24 + x.abs() * 2.0 ** -22
            if softcap:
                x = softcap * torch.tanh(x / softcap)
                err = err + softcap * 2.0 ** -20
            dist = torch.arange(ctx)[None, :] - (ctx - m + torch.arange(m))[:, None]
            if slopes is not None:
                bias = slopes.double()[:, None, None] * math.log(2.0) * dist
                x = x + bias
                err = err + (bias.abs() + x.abs()) * 2.0 ** -22
            gone = torch.zeros(m, ctx, dtype=torch.bool)
            if causal:
                gone |= dist > 0
            if window:
                gone |= dist <= -window
            x = x.masked_fill(gone, -math.inf)
            top = x.amax(-1, keepdim=True)
            w = torch.exp(x - torch.where(top.isinf(), 0.0, top))
            s = w.sum(-1, keepdim=True)
            some = s > 0
            s1 = torch.where(some, s, 1.0)
            y = (w @ v) / s1
            big = (w @ v.abs()) / s1
            e = (err.masked_fill(gone, 0).amax(-1, keepdim=True) * 2 + 2.0 ** -21 + 2.0 ** -18)
            n = (~gone).sum(-1)[None, :, None]
            tiles, chunks = ctx // 64 + 2, ctx // 512 + 2
            t = (big * (eps / 2 + e) + y.abs() * (e + n * step / 2 / s1 + 2 * chunks * step / s1)
                 + (tiles + 2 * chunks) * step / s1)
            t = t * 1.01 + (y.abs() + t) * eps / 2
            out[a : a + m] = (y * some).permute(1, 0, 2)
            tol[a : a + m] = (t * some).permute(1, 0, 2)
        return out, tol

    def check(self, o, **kw):
        want, tol = self.formula(**kw)
        used = int(self.qsl[-1])
        off = (o.cpu().double()[:used] - want[:used]).abs()
        worst = float((off - tol[:used]).max()) if used else 0.0
        assert worst <= 0, (worst, float(off.max()))


SHAPES = [
    # requests, hq, hk, d, page, dtype
    ([(1, 1)], 4, 4, 64, 16, BF),
    ([(1, 700)], 32, 8, 128, 16, BF),
    ([(1, 63), (1, 64), (1, 65), (1, 513)], 8, 2, 128, 16, HF),
    ([(1, 2), (3, 600), (11, 11), (5, 1030)], 28, 4, 128, 32, BF),
    ([(1, 17), (1, 1500), (4, 130)], 24, 8, 64, 64, HF),
    ([(1, 900), (2, 33), (30, 300)], 4, 2, 256, 16, BF),
    ([(70, 70), (1, 200), (65, 800)], 8, 2, 128, 16, BF),
    ([(129, 1100), (3, 5)], 16, 16, 64, 16, HF),
    ([(40, 560)], 16, 2, 256, 32, HF),
    ([(1, 1200), (2, 40)], 64, 1, 128, 16, BF),
]


def shape_id(s):
    reqs, hq, hk, d, page, dtype = s
    return f"{len(reqs)}req{max(m for m, _ in reqs)}x{max(c for _, c in reqs)}_{hq}_{hk}_{d}_{page}_{NAME[dtype]}"


@pytest.mark.parametrize("shape", SHAPES, ids=shape_id)
def test_attention_formula_and_float_cache_bits(shape):
    reqs, hq, hk, d, page, dtype = shape
    b = Batch(reqs, hq, hk, d, page, dtype, seed=len(reqs))
    want = b.over_floats()
    b.check(b.run())
    for splits in (0, 1, 2, 7):
        assert torch.equal(b.run(splits), want), splits


@pytest.mark.parametrize("m,ctx,window", [(12, 513, 0), (33, 1537, 0), (48, 577, 70), (129, 1100, 600), (32, 1024, 481),
                                          (70, 1664, 513), (31, 62, 3), (200, 2111, 1024), (64, 640, 65)])
def test_prompts_whose_first_and_last_chunks_are_partly_live(m, ctx, window):
    # one to eight live tiles at either end of a row tile's keys, even and odd, over one to five chunks
    b = Batch([(m, ctx), (1, 40), (m + 5, ctx + 64)], 8, 2, 128, 16, BF, seed=ctx)
    for kw in (dict(window=window), dict(window=window, causal=False), dict(window=window, softcap=5.0)):
        want = b.over_floats(**kw)
        for splits in (0, 1, 2, 3):
            assert torch.equal(b.run(splits, **kw), want), (kw, splits)


@pytest.mark.parametrize("opts", [dict(), dict(softcap=3.0), dict(alibi=True), dict(window=3500), dict(causal=False),
                                  dict(scale=-0.1)], ids=lambda o: "_".join(f"{k}{v}" for k, v in o.items()) or "plain")
@pytest.mark.parametrize("ib,fb", [(16, 8), (32, 16), (32, 32)])
@pytest.mark.parametrize("d,dtype", [(64, BF), (128, HF), (128, BF)])
def test_prompts_over_long_contexts(d, dtype, ib, fb, opts):
    # enough rows times chunks for workgroups of two row sets, ragged in both
    opts = dict(opts)
    if opts.pop("alibi", False):
        opts["slopes"] = torch.tensor([2.0 ** -(i + 1) for i in range(8)])
    b = Batch([(500, 5000), (1, 40), (77, 900), (33, 4999)], 8, 2, d, 16, dtype, seed=d)
    want = b.over_floats(ib=ib, fb=fb, **opts)
    for splits in (0, 1, 3):
        assert torch.equal(b.run(splits, ib=ib, fb=fb, **opts), want), splits


@pytest.mark.parametrize("d,dtype", [(128, HF), (256, BF)])
def test_one_prompt_beside_many_decode_steps(d, dtype):
    # requests x the longest one's row tiles are mostly empty: the grid follows the tokens instead
    b = Batch([(1, 3 + 7 * i) for i in range(90)] + [(900, 1000)] + [(1, 33), (0, 5), (40, 50)], 8, 2, d, 16, dtype, seed=8)
    want = b.over_floats()
    for splits in (0, 1, 2):
        assert torch.equal(b.run(splits), want), splits


OPTIONS = [dict(softcap=3.0), dict(window=1), dict(window=100), dict(window=700), dict(causal=False), dict(scale=0.3),
           dict(alibi=True), dict(alibi=True, softcap=20.0, window=600), dict(causal=False, window=50)]


@pytest.mark.parametrize("opts", OPTIONS, ids=lambda o: "_".join(f"{k}{v}" for k, v in o.items()))
@pytest.mark.parametrize("d,dtype", [(128, BF), (64, HF), (256, BF)])
def test_attention_options(opts, d, dtype):
    opts = dict(opts)
    b = Batch([(1, 1100), (7, 90), (50, 700), (1, 3)], 8, 2, d, 16, dtype, seed=11)
    if opts.pop("alibi", False):
        opts["slopes"] = torch.tensor([2.0 ** -(i + 1) for i in range(8)])
    want = b.over_floats(**opts)
    b.check(b.run(**opts), **opts)
    for splits in (0, 1, 3):
        assert torch.equal(b.run(splits, **opts), want), splits


@pytest.mark.parametrize("ib,fb", [(16, 8), (32, 8), (64, 16), (64, 32)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_formats(ib, fb, d):
    b = Batch([(1, 600), (20, 140), (60, 1060)], 8, 2, d, 16, BF, seed=4)
    want = b.over_floats(ib=ib, fb=fb)
    for splits in (0, 1, 2):
        assert torch.equal(b.run(splits, ib=ib, fb=fb), want)
    if ib > 16:  # (16-bit sums wrap at 128)
        b.check(b.run(ib=ib, fb=fb), fb=fb)


@pytest.mark.parametrize("opts", [dict(), dict(softcap=3.0), dict(alibi=True), dict(scale=-0.2), dict(window=600, softcap=9.0)],
                         ids=lambda o: "_".join(f"{k}{v}" for k, v in o.items()) or "plain")
@pytest.mark.parametrize("ib,fb", [(16, 8), (32, 16), (32, 32), (64, 16)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_few_rows_a_request(d, ib, fb, opts):
    # workgroups of up to 4, 8 and 16 rows, split and not, under each form of the scores and sums
    opts = dict(opts)
    if opts.pop("alibi", False):
        opts["slopes"] = torch.tensor([2.0 ** -(i + 1) for i in range(8)])
    for reqs in ([(1, 1100), (1, 513), (1, 40)], [(1, 700), (2, 1300), (2, 64)], [(4, 64), (1, 1100), (3, 600), (7, 90)],
                 [(4, 64), (7, 600), (50, 700)]):
        b = Batch(reqs, 8, 2, d, 16, BF if fb != 32 else HF, seed=d + ib)
        want = b.over_floats(ib=ib, fb=fb, **opts)
        for splits in (0, 1, 2):
            for _ in range(2):
                assert torch.equal(b.run(splits, ib=ib, fb=fb, **opts), want), (reqs, splits)


def test_rows_do_not_depend_on_the_batch():
    # a token's output: alone as a decode step, inside a prompt, beside other requests, at any max_query_len
    b = Batch([(90, 600), (1, 40), (3, 1300)], 8, 2, 128, 16, BF, seed=2)
    whole = b.run()
    for extra in (0, 13, 200):
        assert torch.equal(b.run(max_q=b.max_q + extra), whole)
    for row in (0, 31, 89):
        one = torch.empty(1, 8, 128, dtype=BF, device="cuda")
        ops.unified_attention_mx4_fxp(
            b.q[row : row + 1].cuda(), b.codes, b.scales, one, torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
            torch.tensor([600 - 90 + row + 1], dtype=torch.int32, device="cuda"), b.table[:1].cuda(), 1, None, True, None,
            32, 16, 0.0, 0, 0)
        assert torch.equal(one[0], whole[row])


def test_rows_without_keys_and_rows_past_the_last():
    # a request of length 0 and one whose window leaves nothing give zeros; rows behind the last request stay
    reqs = [(1, 20), (2, 0), (0, 30), (1, 5)]
    b = Batch(reqs, 4, 2, 64, 16, HF, seed=9)
    b.q = torch.cat([b.q, randn(6, 4, 64, dtype=HF)])
    for splits in (0, 1, 3):
        o = b.run(splits)
        assert torch.equal(o[4:], torch.full_like(o[4:], 7.0))
        assert not o[1:3].any()
        b.check(o)
    # context shorter than the new tokens: the first rows see no key
    b = Batch([(1, 600)], 4, 2, 64, 16, HF, seed=10)
    b.qsl = torch.tensor([0, 5], dtype=torch.int32)
    b.lens = torch.tensor([3], dtype=torch.int32)
    b.q, b.max_q = randn(5, 4, 64, dtype=HF), 5
    for splits in (0, 1, 2):
        o = b.run(splits)
        assert not o[:2].any() and bool(o[2:].any()) and bool(torch.isfinite(o.float()).all())


def test_masked_keys_of_any_bytes():
    # keys that the causal mask or the window hides, and a page's rows past the sequence, hold every byte pattern
    # (among them those that would stand for infinities and NaN): no output sees them
    hk, d, page = 2, 128, 16
    b = Batch([(40, 200), (1, 1000)], 8, hk, d, page, BF, seed=6)
    base = b.run(window=64)
    g = torch.Generator().manual_seed(1)
    # request 1's keys before its window
    hidden = b.slots[1][: 1000 - 64]
    # and request 0's keys after position 170 for the rows before it: compared over those rows only
    late = b.slots[0][171:]
    for slots in (hidden, late):
        blk, off = (slots // page).cuda(), (slots % page).cuda()
        shape = (len(slots), 2, hk)
        half = torch.arange(2, device="cuda")
        b.codes[blk[:, None], half, off[:, None]] = torch.randint(0, 256, (*shape, d // 2), generator=g, dtype=torch.uint8).cuda()
        b.scales[blk[:, None], half, off[:, None]] = torch.randint(250, 256, (*shape, d // 32), generator=g,
                                                                  dtype=torch.uint8).cuda()
    for splits in (0, 1, 2):
        o = b.run(splits, window=64)
        assert torch.equal(o[:11], base[:11]) and torch.equal(o[40], base[40])


def test_bad_tables_stay_inside_the_cache():
    # block numbers outside the cache, a table narrower than the sequence, more rows than tokens: finite outputs
    b = Batch([(1, 100), (60, 300)], 8, 2, 128, 16, BF, seed=7)
    for table in (torch.full_like(b.table, -(1 << 31)), torch.full_like(b.table, (1 << 31) - 1), b.table[:, :3]):
        b.table = table.contiguous()
        for splits in (0, 1, 2):
            assert bool(torch.isfinite(b.run(splits).float()).all())
    b.qsl = torch.tensor([0, 1, 500], dtype=torch.int32)
    assert bool(torch.isfinite(b.run().float()).all())


def test_a_table_shorter_than_the_sequences():
    # keys past the table's are not there, however the keys are split; lengths and starts of any value stay inside
    b = Batch([(1, 1700), (60, 900), (2, 1200)], 8, 2, 128, 16, BF, seed=13)
    b.table = b.table[:, :40].contiguous()
    want = b.run(1)
    for splits in (0, 2, 5):
        assert torch.equal(b.run(splits), want), splits
    b.lens = torch.tensor([700, 900, 700], dtype=torch.int32)  # request 2's new tokens lie past the table: 640 keys
    b.lens[2] = 640 + 2
    o = b.run(1)
    b.lens = torch.tensor([(1 << 31) - 1, 900, (1 << 31) - 1], dtype=torch.int32)
    for splits in (0, 1, 2):
        for window in (0, 100):
            assert bool(torch.isfinite(b.run(splits, window=window).float()).all())
        far = b.run(splits)
        assert torch.equal(far[1:61], o[1:61]) and torch.equal(far[61:], o[61:])  # every key of the table is seen
    b.lens = torch.tensor([-5, 900, -1000], dtype=torch.int32)
    for splits in (0, 1, 2):
        far = b.run(splits)
        assert not far[0].any() and not far[61:].any() and torch.equal(far[1:61], o[1:61])


def test_rows_of_infinities_and_nan():
    # such rows are the float cache's, and the others do not change
    b = Batch([(1, 700), (40, 600), (3, 90)], 8, 2, 128, 16, BF, seed=12)
    base = b.run()
    bad = {0: (2, math.inf), 5: (0, math.nan), 10: (7, -math.inf), 20: (3, torch.finfo(BF).max), 42: (1, math.nan)}
    for row, (head, v) in bad.items():
        b.q[row, head, :: 2 if math.isinf(v) else 1] = v
    want = b.over_floats().view(torch.int16)
    for splits in (0, 1, 2):
        o = b.run(splits)
        assert torch.equal(o.view(torch.int16), want), splits
        for row, (head, _) in bad.items():
            o[row, head] = base[row, head]
        assert torch.equal(o, base)


def test_a_strided_output_keeps_the_rows_of_no_request():
    b = Batch([(1, 20), (2, 30)], 4, 2, 64, 16, HF, seed=9)
    want = b.run()
    n = b.q.shape[0]
    b.q = torch.cat([b.q, randn(5, 4, 64, dtype=HF)])
    wide = torch.full((n + 5, 4, 128), 7.0, dtype=HF, device="cuda")
    b.run(o=wide[:, :, ::2])
    assert torch.equal(wide[:n, :, ::2], want) and bool((wide[n:] == 7).all()) and bool((wide[:, :, 1::2] == 7).all())
    wide.fill_(7.0)
    mx4.unified_attention_run(b.q.cuda(), b.codes, b.scales, wide[:, :, ::2], b.qsl.cuda(), b.lens.cuda(), b.table.cuda(),
                              b.max_q, None, True, None, 32, 16, 0.0, 0, 0)
    assert torch.equal(wide[:n, :, ::2], want) and bool((wide[n:] == 7).all())


@pytest.mark.parametrize("order", ["heads", "slots"])
def test_strides(order):
    # q, o and the table as views; the cache in another order, one layer of a stack of caches
    b = Batch([(1, 300), (55, 70), (2, 700)], 8, 2, 128, 16, HF, order=order, seed=3)
    want = b.over_floats()
    assert torch.equal(b.run(), want)
    stack_c = torch.zeros(3, *b.codes.shape, dtype=torch.uint8, device="cuda")
    stack_s = torch.zeros(*b.scales.shape[:4], 3, b.scales.shape[4], dtype=torch.uint8, device="cuda")
    stack_c[1], stack_s[:, :, :, :, 2] = b.codes, b.scales
    b.codes, b.scales = stack_c[1], stack_s[:, :, :, :, 2]
    n = b.q.shape[0]
    qkv = torch.zeros(n, 12, 128, dtype=HF, device="cuda")
    qkv[:, :8] = b.q.cuda()
    wide = torch.full((n, 8, 256), 7.0, dtype=HF, device="cuda")
    o = wide[:, :, ::2]  # no unit stride: goes through a copy
    b.run(q=qkv[:, :8], o=o)
    assert torch.equal(o, want) and bool((wide[:, :, 1::2] == 7).all())
    padded = torch.full((n, 8, 136), 7.0, dtype=HF, device="cuda")
    off = torch.zeros(n, 8, 129, dtype=HF, device="cuda")
    off[..., 1:] = b.q.cuda()
    b.table = torch.cat([b.table, torch.zeros(3, 5, dtype=torch.int32)], 1)[:, : b.width]
    b.run(q=off[..., 1:], o=padded[..., :128])
    assert torch.equal(padded[..., :128], want) and bool((padded[..., 128:] == 7).all())


def test_a_step_as_used_captured_and_replayed():
    # write the step's tokens, attend, sample of the cache read back: eager against a replayed graph whose inputs change
    heads, hk, d, page, reqs = 8, 2, 128, 16, 5
    codes, scales = new_cache(200, page, hk, d)
    ref = [x.clone() for x in (codes, scales)]
    table = torch.randperm(200, generator=torch.Generator().manual_seed(0))[: reqs * 40].view(reqs, 40).to(torch.int32).cuda()
    lens = torch.tensor([1, 30, 64, 511, 600], dtype=torch.int32, device="cuda")
    qsl = torch.arange(reqs + 1, dtype=torch.int32, device="cuda")
    q = torch.zeros(reqs, heads, d, dtype=BF, device="cuda")
    key, value = (torch.zeros(reqs, hk, d, dtype=BF, device="cuda") for _ in range(2))
    slots = torch.zeros(reqs, dtype=torch.int64, device="cuda")
    o = torch.zeros_like(q)

    def step(c, s, out):
        ops.reshape_and_cache_mx4(key, value, c, s, slots)
        ops.unified_attention_mx4_fxp(q, c, s, out, qsl, lens, table, 1, None, True, None, 32, 16, 0.0, 0, 0)
        return ops.gather_cache_mx4(c, s, slots, BF)

    def inputs(i):
        lens.add_(1)
        pos = (lens - 1).long()
        slots.copy_(table.long().gather(1, (pos // page)[:, None])[:, 0] * page + pos % page)
        for t, seed in ((q, 1), (key, 2), (value, 3)):
            t.copy_(randn(*t.shape, seed=10 * i + seed, dtype=BF))

    inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(codes, scales, o)
    torch.cuda.current_stream().wait_stream(side)
    step(*ref, torch.zeros_like(o))  # (the reference cache gets the warm-up step's tokens too)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        back = step(codes, scales, o)
    for i in range(1, 6):
        inputs(i)
        graph.replay()
        want = torch.zeros_like(o)
        k, v = step(*ref, want)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(back[0], k) and torch.equal(back[1], v), i
        x = randn(64, 64).cuda()
        (x @ x).sum().item()  # the program's own work between replays


def test_two_streams_at_once():
    a = Batch([(1, 2000), (3, 900)], 8, 2, 128, 16, BF, seed=1)
    b = Batch([(80, 700), (1, 1500)], 8, 2, 128, 16, BF, seed=2)
    want_a, want_b = a.run(3), b.run(2)
    args = {id(x): (x.q.cuda(), x.qsl.cuda(), x.lens.cuda(), x.table.cuda()) for x in (a, b)}
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [[], []]
    for _ in range(5):
        for i, (x, splits) in enumerate(((a, 3), (b, 2))):
            q, qsl, lens, table = args[id(x)]
            with torch.cuda.stream(streams[i]):
                o = torch.empty_like(q)
                ops.unified_attention_mx4_fxp(q, x.codes, x.scales, o, qsl, lens, table, x.max_q, None, True, None, 32, 16,
                                              0.0, 0, splits)
                outs[i].append(o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want_a) for o in outs[0]) and all(torch.equal(o, want_b) for o in outs[1])


@pytest.mark.parametrize("native", [True, False])
def test_refusals(native):
    from fxpr_vllm import _lib

    if native:
        write, gather, attn = ops.reshape_and_cache_mx4, ops.gather_cache_mx4, ops.unified_attention_mx4_fxp
    else:
        write, gather, attn = (_lib._reshape_and_cache_mx4_cuda, _lib._gather_cache_mx4_cuda,
                               _lib._unified_attention_mx4_fxp_cuda)
    c, s = new_cache(4, 16, 2, 128)
    x = torch.zeros(3, 2, 128, dtype=BF, device="cuda")
    slots = torch.arange(3, device="cuda")
    write(x, x, c, s, slots)
    for err, args in [
        (TypeError, (x.double(), x.double(), c, s, slots)), (TypeError, (x, x.half(), c, s, slots)),
        (TypeError, (x, x, c.char(), s, slots)), (TypeError, (x, x, c, s, slots.float())),
        (ValueError, (x[:, :1], x[:, :1], c, s, slots)), (ValueError, (x, x[:2], c, s, slots)),
        (ValueError, (x, x, c, s[:3], slots)), (ValueError, (x, x, c[0], s[0], slots)),
        (ValueError, (x, x, c, s, slots[:2])), (ValueError, (x, x, c, s, slots[None])),
        (ValueError, (x, x, c[..., :48], s[..., :3], slots)), (ValueError, (x, x, c[..., ::2], s[..., ::2], slots)),
        (RuntimeError, (x.cpu(), x, c, s, slots)), (RuntimeError, (x, x, c, s, slots.cpu())),
        (RuntimeError, (x, x, c.cpu(), s, slots)),
    ]:
        with pytest.raises(err):
            write(*args)
    for err, args in [(TypeError, (c, s, slots, torch.float64)), (ValueError, (c, s, slots[None], BF)),
                      (TypeError, (c, s.float(), slots, BF)), (RuntimeError, (c, s, slots.cpu(), BF))]:
        with pytest.raises(err):
            gather(*args)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.zeros(3, 4, 128, dtype=BF, device="cuda")
    good = dict(q=q, c=c, s=s, o=torch.empty_like(q), qsl=i(0, 1, 3), lens=i(5, 9), bt=i(0, 1).view(2, 1), mq=2, al=None,
                causal=True, scale=None, ib=32, fb=16, cap=0.0, win=0, splits=0)
    attn(*good.values())
    for err, change in [
        (TypeError, dict(q=q.float(), o=q.float())), (TypeError, dict(o=q.half())), (TypeError, dict(qsl=good["qsl"].long())),
        (TypeError, dict(lens=good["lens"].long())), (TypeError, dict(bt=good["bt"].long())),
        (TypeError, dict(al=torch.zeros(4, dtype=BF, device="cuda"))), (TypeError, dict(c=c.char())),
        (ValueError, dict(ib=8)), (ValueError, dict(fb=12)), (ValueError, dict(splits=-1)),
        (ValueError, dict(al=torch.zeros(3, device="cuda"))), (ValueError, dict(q=q[:, :3], o=q[:, :3].clone())),
        (ValueError, dict(q=q[..., :64], o=q[..., :64].clone())), (ValueError, dict(o=q[:2].clone())),
        (ValueError, dict(qsl=i(0, 3))), (ValueError, dict(bt=i(0).view(1, 1))), (ValueError, dict(q=q[0], o=q[0].clone())),
        (ValueError, dict(c=c[:, :, :8], s=s[:, :, :8])), (ValueError, dict(s=s[..., :2])),
        (RuntimeError, dict(q=q.cpu())), (RuntimeError, dict(bt=good["bt"].cpu())),
    ]:
        with pytest.raises(err):
            attn(*{**good, **change}.values())


def test_python_launchers_give_the_native_results():
    from fxpr_vllm import _lib

    b = Batch([(1, 900), (60, 100)], 8, 2, 128, 16, BF, seed=8)
    o = torch.empty_like(b.q, device="cuda")
    _lib._unified_attention_mx4_fxp_cuda(b.q.cuda(), b.codes, b.scales, o, b.qsl.cuda(), b.lens.cuda(), b.table.cuda(),
                                         b.max_q, None, True, None, 32, 16, 0.0, 0, 0)
    assert torch.equal(o, b.run())
    x = randn(9, 2, 128, dtype=HF).cuda()
    slots = torch.arange(9, device="cuda")
    one, two = new_cache(2, 16, 2, 128), new_cache(2, 16, 2, 128)
    ops.reshape_and_cache_mx4(x, x * 2, *one, slots)
    _lib._reshape_and_cache_mx4_cuda(x, x * 2, *two, slots)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    for a, c in zip(ops.gather_cache_mx4(*one, slots, FP), _lib._gather_cache_mx4_cuda(*two, slots, FP)):
        assert torch.equal(a, c)


def test_fixed_point_attention_is_near_the_unquantised_one():
    # what 4 bits cost: an element is off by at most the block's step / 2, a quarter of its largest magnitude / 3.5
    b = Batch([(1, 500)], 8, 2, 128, 16, BF, seed=12)
    k, v = ops.gather_cache_mx4(b.codes, b.scales, b.slots[0].cuda(), BF)
    for got, x in ((k, b.key), (v, b.value)):
        x = x.double()
        amax = x.unflatten(-1, (-1, 32)).abs().amax(-1).repeat_interleave(32, -1)
        assert bool(((got.cpu().double() - x).abs() <= amax / 3.5).all())
