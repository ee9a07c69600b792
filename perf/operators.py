"""The paged KV cache held in 4 bits, as calls that can be timed and checked: the quantising write, the read
back, and attention over it.

A cache row (one token, one kv head, K or V) of D elements is D / 32 blocks of 32. A block has a scale byte b,
which stands for 2^(b - 127), and an element a 4-bit code: a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6. With amax
the block's largest magnitude, 2^(b - 127) is the power of two that brings amax into (3.5, 7], limited to what
the input type can stand for; a code is x 2^(127 - b) rounded to the nearest value (ties to the even code) and
saturated, NaN as 0. Bytes of a row: 8-element chunk c is the 4-byte unit (c % 4) (D / 32) + c / 4, its element i
in bits 4 i and up.

Kinds and what `run` returns:

  write    reshape_and_cache_mx4 of a step's tokens, then gather_cache_mx4 of the same slots; the values.
  read     gather_cache_mx4 of cached tokens; the values.
  attn     unified_attention_mx4_fxp over the cache, for some cases behind the write of the step's own tokens;
           the output rows.
"""

import math
import pathlib
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
# scale bytes that leave every code a finite and exact value of the type; a byte above reads as the last
BYTES = {"bf16": (2, 252), "f16": (104, 140), "f32": (2, 252)}


def _write(tokens, kv_heads=8, head_dim=128, page=16, dtype="bf16", padding=0, **kw):
    return dict(kw, kind="write", tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype,
                padding=padding)


def _read(tokens, kv_heads=8, head_dim=128, page=16, dtype="bf16", **kw):
    return dict(kw, kind="read", tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype)


def _attn(decodes, ctx_lo, ctx_hi, prefills=0, new=0, past=0, heads=32, kv_heads=8, head_dim=128, page=16,
          dtype="bf16", window=0, softcap=0.0, alibi=False, write=False, lens=0, **kw):
    """`decodes` one-token requests with contexts in [ctx_lo, ctx_hi]; `prefills` requests of up to `new` new
    tokens each after up to `past` cached ones (the first has exactly these). `write`: the step's tokens are
    written into the cache first."""
    return dict(kw, kind="attn", decodes=decodes, ctx_lo=ctx_lo, ctx_hi=ctx_hi, prefills=prefills, new=new, past=past,
                heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, window=window,
                softcap=softcap, alibi=alibi, write=write, lens=lens)


def listed():
    return [
        # the tokens of one decode step of a full batch, padded as a captured step is
        _write(64, padding=7, name="write_decode_step"),
        # a large prompt batch's tokens in one step
        _write(8192, name="write_prompts"),
        # an odd chunk of a float16 model with heads of 64 and larger pages
        _write(777, kv_heads=16, head_dim=64, page=64, dtype="f16", name="write_chunk_f16"),
        # a shared prefix of 2041 tokens, read back for another consumer
        _read(2041, name="read_prefix"),
        # a long context handed on in float32
        _read(65536, dtype="f32", name="read_long_f32"),
        # one user's token over a short context, where latency counts
        _attn(1, 700, 700, write=True, lens=1, name="attn_one_short"),
        # one user's token over the longest context
        _attn(1, 131072, 131072, lens=2, name="attn_one_long"),
        # a serving batch in decode: 64 requests, contexts from 512 to 8192, with the write of their tokens
        _attn(64, 512, 8192, write=True, lens=3, name="attn_decode"),
        # heads of 64, float16, a sliding window and a softcap
        _attn(83, 100, 6000, heads=24, kv_heads=8, head_dim=64, page=32, dtype="f16", window=1024, softcap=50.0, lens=4,
              name="attn_decode_window_f16"),
        # four fresh prompts of up to 2048 tokens
        _attn(0, 1, 1, prefills=4, new=2048, lens=5, name="attn_prefill"),
        # continuous batching: a 512-token chunk of one long prompt beside 31 decoding requests
        _attn(31, 512, 8192, prefills=1, new=512, past=3500, dtype="f16", lens=6, name="attn_mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "attn", "attn", "attn"])
    if kind != "attn":
        kv_heads, head_dim = rng.choice([(8, 128), (4, 128), (1, 128), (16, 64), (8, 64), (8, 256)])
        page, dtype = rng.choice([16, 16, 32, 64]), rng.choice(["bf16", "bf16", "f16", "f32"])
        if kind == "write":
            tokens = _log_int(rng, 1, 8192)
            return _write(tokens, kv_heads, head_dim, page, dtype, rng.choice([0, rng.randint(0, tokens // 4)]))
        return _read(_log_int(rng, 1, 32768), kv_heads, head_dim, page, dtype)
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (28, 4, 128), (16, 16, 64), (24, 8, 64),
                                            (32, 2, 128), (16, 8, 256)])
    what = rng.choice(["decode", "decode", "prefill", "mixed"])
    hi = _log_int(rng, 64, 8192)
    decodes = 0 if what == "prefill" else _log_int(rng, 1, 64)
    prefills = 0 if what == "decode" else rng.randint(1, 2)
    new = 0 if what == "decode" else _log_int(rng, 2, 1024)
    past = 0 if rng.random() < 0.5 or not prefills else rng.randint(0, min(6000, 1500000 // new))
    window, softcap, alibi = rng.choice([(0, 0.0, False), (0, 0.0, False), (0, 0.0, False), (1024, 0.0, False),
                                         (0, 50.0, False), (0, 0.0, True)])
    return _attn(decodes, max(1, hi // 16), hi, prefills, new, past, heads, kv_heads, head_dim,
                 rng.choice([16, 16, 32, 64]), rng.choice(["bf16", "f16"]), window, softcap, alibi, rng.random() < 0.5,
                 rng.randrange(1 << 20))


# ---------------------------------------------------------------------------
# Shapes, from the case alone.


def _requests(case):
    """(new tokens, context with them) of each request: the decodes, then the prefills."""
    rng = random.Random(case["lens"])
    dec = [(1, rng.randint(case["ctx_lo"], case["ctx_hi"])) for _ in range(case["decodes"])]
    pre = []
    for i in range(case["prefills"]):
        new = case["new"] if i == 0 else rng.randint(max(1, case["new"] // 2), case["new"])
        pre.append((new, new + (case["past"] if i == 0 else rng.randint(0, case["past"]))))
    return dec, pre


def work(case):
    d, hk = case["head_dim"], case["kv_heads"]
    row = hk * (d // 2 + d // 32) * 2  # a token's cached bytes, K and V
    if case["kind"] != "attn":
        t = case["tokens"]
        values = t * hk * d * 2 * SIZE[case["dtype"]]
        if case["kind"] == "read":
            return {"bytes": t * (row + 8) + values, "flops": 0}
        live = t - case["padding"]
        return {"bytes": 2 * values + 8 * t + 2 * live * row, "flops": 0}
    dec, pre = _requests(case)
    hq, win = case["heads"], case["window"]
    tokens = sum(n for n, _ in dec + pre)
    pairs = seen = 0
    for n, ctx in dec + pre:
        first = ctx - n  # position of the first new token
        if win:
            pairs += sum(min(p + 1, win) for p in range(first, ctx))
            seen += min(ctx, n + win - 1)
        else:
            pairs += n * first + n * (n + 1) // 2
            seen += ctx
    b = seen * row + 2 * tokens * hq * d * SIZE[case["dtype"]]
    if case["write"]:
        b += tokens * (2 * hk * d * SIZE[case["dtype"]] + row + 8)
    return {"bytes": b, "flops": 4 * hq * d * pairs}


# ---------------------------------------------------------------------------
# The plain form.


def _quantise(x, dtype):
    """x [..., D] float32 -> (codes [..., D / 2], scale bytes [..., D / 32]), both uint8."""
    lo, hi = BYTES[dtype]
    x = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf)
    blocks = x.unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1)
    b = (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 2).clamp(lo, hi)
    y = blocks * ((254 - b) << 23).view(torch.float32).unsqueeze(-1)
    a = y.abs()
    level = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (level + 8 * (y < 0)).flatten(-2).to(torch.uint8)
    code = code.unflatten(-1, (-1, 4, 8)).transpose(-3, -2).flatten(-3)  # chunk c to unit (c % 4) (D / 32) + c / 4
    return code[..., 0::2] | (code[..., 1::2] << 4), b.to(torch.uint8)


def _values(codes, scales, dtype):
    """The values, float32 [..., D], that codes [..., D / 2] and scale bytes [..., D / 32] stand for."""
    hi = BYTES[dtype][1]
    table = torch.tensor(LEVELS + [-v for v in LEVELS], device=codes.device)
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    nib = nib.unflatten(-1, (4, -1, 8)).transpose(-3, -2).flatten(-3).int()
    scale = (scales.int().clamp(max=hi) << 23).view(torch.float32)
    return (table[nib].unflatten(-1, (-1, 32)) * scale.unsqueeze(-1)).flatten(-2)


def _plain_write(s):
    dt, live, page = s["dtype"], s["live"], s["page"]
    slots = s["slots"][live]
    blk, off = slots // page, slots % page
    kv = torch.stack([s["key"][live], s["value"][live]], 1).float()  # [T, 2, H, D]
    codes, scales = _quantise(kv, dt)
    half = torch.arange(2, device=blk.device)
    s["codes"][blk[:, None], half, off[:, None]] = codes
    s["scales"][blk[:, None], half, off[:, None]] = scales


def _plain_read(s):
    slots, page = s["slots"], s["page"]
    at = slots.clamp(min=0)
    blk, off = at // page, at % page
    half = torch.arange(2, device=blk.device)
    v = _values(s["codes"][blk[:, None], half, off[:, None]], s["scales"][blk[:, None], half, off[:, None]], s["dtype"])
    v = (v * (slots >= 0)[:, None, None, None]).to(DTYPES[s["dtype"]])
    return {"key": v[:, 0].contiguous(), "value": v[:, 1].contiguous()}


def _plain_group(s, g):
    """Attention of the requests of one group (the one-token ones, or the others), padded to its longest."""
    n, page, heads, kv_heads = g["keys"], s["page"], s["heads"], s["kv_heads"]
    key = torch.arange(n, device=s["q"].device)
    blk, off = g["table"][:, key // page], key % page
    k = _values(s["codes"][blk, 0, off], s["scales"][blk, 0, off], s["dtype"])  # [R, keys, H, D]
    v = _values(s["codes"][blk, 1, off], s["scales"][blk, 1, off], s["dtype"])
    q = s["q"][g["token"]].float()  # [R, new, Hq, D]
    r, new, _, d = q.shape
    q = q.view(r, new, kv_heads, heads // kv_heads, d).permute(0, 2, 3, 1, 4).reshape(r, kv_heads, -1, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]
    x = x.view(r, heads, new, n)
    if s["softcap"]:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    pos = g["pos"][:, None, :, None]  # [R, 1, new, 1]
    if s["slopes"] is not None:
        x = x + (s["slopes"] * math.log(2.0))[None, :, None, None] * (key - pos)
    seen = key <= pos
    if s["window"]:
        seen = seen & (key > pos - s["window"])
    x = x.masked_fill(~seen, -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    y = torch.matmul(w.view(r, kv_heads, -1, n), v.permute(0, 2, 1, 3))
    y = y.view(r, heads, new, d).transpose(1, 2).to(DTYPES[s["dtype"]])
    s["o"][g["flat"]] = y.flatten(0, 1)[g["pick"]]


def _plain_attn(s):
    if s["write"]:
        _plain_write(s)
    if s["dec"] is not None:
        _plain_group(s, s["dec"])
    if s["pre"] is not None:
        _plain_group(s, s["pre"])
    return s["o"]


# ---------------------------------------------------------------------------
# What a program has in hand before the call.


def _cache(blocks, case, dev):
    """An empty cache: blocks of [2, heads, page] rows, seen as [blocks, 2, page, heads, ...]."""
    h, p, d = case["kv_heads"], case["page"], case["head_dim"]
    codes = torch.zeros(blocks, 2, h, p, d // 2, dtype=torch.uint8, device=dev).transpose(2, 3)
    scales = torch.full((blocks, 2, h, p, d // 32), 127, dtype=torch.uint8, device=dev).transpose(2, 3)
    return codes, scales


def _activations(shape, gen, dev, outliers):
    """Normal rows; a few channels of a head (a key's) are several times larger, as in trained models."""
    x = torch.randn(shape, generator=gen, device=dev)
    if outliers:
        x *= 1.0 + 5.0 * (torch.rand(shape[-2:], generator=gen, device=dev) < 0.03)
    return x


def _fill(codes, scales, case, gen, dev):
    """Every row of the cache, quantised from activations, some blocks at a time."""
    step = max(1, (1 << 26) // (codes[0].numel() * 2))
    for b in range(0, codes.shape[0], step):
        n = min(step, codes.shape[0] - b)
        shape = (n, case["page"], case["kv_heads"], case["head_dim"])
        for half in (0, 1):
            c, s = _quantise(_activations(shape, gen, dev, half == 0), case["dtype"])
            codes[b : b + n, half], scales[b : b + n, half] = c, s


def _slots(tokens, blocks, page, gen, dev):
    """Token by token through scattered pages."""
    pages = torch.randperm(blocks, generator=gen, device=dev)
    t = torch.arange(tokens, device=dev)
    return pages[t // page] * page + t % page


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed * 7919 + 17)
    dt, page, h, d = DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["head_dim"]
    s = {"kind": case["kind"], "dtype": case["dtype"], "page": page, "kv_heads": h}
    if case["kind"] != "attn":
        blocks = -(-case["tokens"] // page) * 5 // 4 + 3
        s["codes"], s["scales"] = _cache(blocks, case, dev)
        s["slots"] = _slots(case["tokens"], blocks, page, gen, dev)
        if case["kind"] == "read":
            _fill(s["codes"], s["scales"], case, gen, dev)
            return s
        live = case["tokens"] - case["padding"]
        s["slots"][live:] = -1
        s["live"] = slice(0, live)
        shape = (case["tokens"], h, d)
        s["key"], s["value"] = (_activations(shape, gen, dev, i == 0).to(dt) for i in (0, 1))
        return s
    dec, pre = _requests(case)
    reqs = dec + pre
    need = [-(-ctx // page) for _, ctx in reqs]
    width = max(need)
    blocks = sum(need) * 9 // 8 + 3
    s["codes"], s["scales"] = _cache(blocks, case, dev)
    _fill(s["codes"], s["scales"], case, gen, dev)
    perm = torch.randperm(blocks, generator=gen, device=dev)
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device=dev)
    col = torch.arange(width, device=dev)
    held = col < torch.tensor(need, device=dev)[:, None]
    table = torch.where(held, perm[(first[:, None] + col).clamp(max=blocks - 1)], 0)
    s["table"] = table.to(torch.int32)
    starts = [0]
    for n, _ in reqs:
        starts.append(starts[-1] + n)
    tokens = starts[-1]
    s["qsl"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    s["lens"] = torch.tensor([c for _, c in reqs], dtype=torch.int32, device=dev)
    s["new"] = max(n for n, _ in reqs)
    s["heads"], s["window"], s["softcap"], s["write"] = case["heads"], case["window"], case["softcap"], case["write"]
    s["scale"] = d ** -0.5
    s["slopes"] = None
    if case["alibi"]:
        hq = case["heads"]
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) / math.log(2.0) for i in range(hq)], device=dev)
    s["q"] = torch.randn((tokens, case["heads"], d), generator=gen, device=dev).to(dt)
    s["o"] = torch.empty_like(s["q"])
    req = torch.repeat_interleave(torch.arange(len(reqs), device=dev), torch.tensor([n for n, _ in reqs], device=dev))
    pos = torch.arange(tokens, device=dev) - s["qsl"][:-1][req] + (s["lens"] - s["qsl"].diff())[req]
    s["slots"] = table[req, pos // page] * page + pos % page
    if case["write"]:
        s["live"] = slice(0, tokens)
        s["key"], s["value"] = (_activations((tokens, h, d), gen, dev, i == 0).to(dt) for i in (0, 1))

    def group(a, b):
        if a == b:
            return None
        new = max(n for n, _ in reqs[a:b])
        at = torch.arange(new, device=dev)
        count = torch.tensor([n for n, _ in reqs[a:b]], device=dev)[:, None]
        start = s["qsl"][a:b, None].long()
        ctx = s["lens"][a:b, None].long()
        inside = at < count
        token = torch.where(inside, start + at, start)
        return {"keys": max(c for _, c in reqs[a:b]), "table": table[a:b], "token": token,
                "pos": torch.where(inside, ctx - count + at, ctx - count), "flat": token[inside],
                "pick": inside.flatten().nonzero().flatten()}

    s["dec"], s["pre"] = group(0, len(dec)), group(len(dec), len(reqs))
    return s


def _ops():
    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "vllm-triton-fixed-point-reductions_amd"))
    import fxpr_vllm  # noqa: F401  (registers torch.ops.fxpr.*)

    sys.path.pop(0)
    return torch.ops.fxpr


def run(s):
    if not own:
        if s["kind"] == "write":
            _plain_write(s)
        return _plain_attn(s) if s["kind"] == "attn" else _plain_read(s)
    ops = torch.ops.fxpr if "fxpr_vllm" in sys.modules else _ops()
    if s["kind"] == "write" or (s["kind"] == "attn" and s["write"]):
        ops.reshape_and_cache_mx4(s["key"], s["value"], s["codes"], s["scales"], s["slots"])
    if s["kind"] == "attn":
        ops.unified_attention_mx4_fxp(s["q"], s["codes"], s["scales"], s["o"], s["qsl"], s["lens"], s["table"], s["new"],
                                      s["slopes"], True, s["scale"], 32, 16, s["softcap"], s["window"], 0)
        return s["o"]
    key, value = ops.gather_cache_mx4(s["codes"], s["scales"], s["slots"], DTYPES[s["dtype"]])
    return {"key": key, "value": value}


# ---------------------------------------------------------------------------
# From the definition, in 64 bits.


def _nearest(x, dtype):
    """What x [..., D] reads back as once written, by comparing with every representable magnitude."""
    lo, hi = BYTES[dtype]
    blocks = x.double().unflatten(-1, (-1, 32))
    blocks = torch.where(blocks.isnan(), torch.zeros_like(blocks), blocks)
    amax = blocks.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(amax.clamp(min=2.0 ** -140, max=2.0 ** 130))  # amax = m 2^e, m in [1/2, 1)
    e = e.double() - 3 + (amax > 7.0 * torch.exp2(e.double() - 3)).double()
    s = torch.exp2(e.clamp(lo - 127, hi - 127))
    y = (blocks.abs() / s).clamp(max=6.0)
    out = torch.zeros_like(y)
    best = y.clone()  # distance to 0
    for i, level in enumerate(LEVELS[1:], 1):
        dist = (y - level).abs()
        take = (dist < best) | ((dist == best) & (i % 2 == 0))
        out, best = torch.where(take, level, out), torch.where(take, dist, best)
    return (out * s * blocks.sign()).flatten(-2)


def _decode(codes, scales, dtype):
    """float64 values of cache rows, element by element of the byte layout."""
    hi = BYTES[dtype][1]
    d = codes.shape[-1] * 2
    e = torch.arange(d, device=codes.device)
    chunk, i = e // 8, e % 8
    byte = 4 * ((chunk % 4) * (d // 32) + chunk // 4) + i // 2
    code = (codes.int()[..., byte] >> (4 * (i % 2)).int()) & 15
    m = code & 7
    mag = torch.where(m < 2, 0.5 * m, (2 + (m & 1)) * torch.exp2((m >> 1).double() - 2))
    power = torch.exp2(scales.double().clamp(max=hi) - 127)
    return torch.where(code > 7, -mag, mag) * power.repeat_interleave(32, -1)


def exact(case, seed):
    s = prepare(case, seed)
    page = s["page"]
    if case["kind"] == "write":
        keep = (s["slots"] >= 0)[:, None, None]
        return {"key": _nearest(s["key"], s["dtype"]) * keep, "value": _nearest(s["value"], s["dtype"]) * keep}
    if case["kind"] == "read":
        blk, off = s["slots"] // page, s["slots"] % page
        return {n: _decode(s["codes"][blk, i, off], s["scales"][blk, i, off], s["dtype"])
                for i, n in enumerate(("key", "value"))}
    dec, pre = _requests(case)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    t = 0
    for r, (n, ctx) in enumerate(dec + pre):
        p = torch.arange(ctx, device=out.device)
        blk, off = s["table"][r].long()[p // page], p % page
        k, v = (_decode(s["codes"][blk, i, off], s["scales"][blk, i, off], s["dtype"]) for i in (0, 1))
        if case["write"]:
            k[ctx - n :] = _nearest(s["key"][t : t + n], s["dtype"])
            v[ctx - n :] = _nearest(s["value"][t : t + n], s["dtype"])
        k, v = (x.permute(1, 0, 2).repeat_interleave(case["heads"] // case["kv_heads"], 0) for x in (k, v))
        for a in range(0, n, 256):  # rows at a time, for their memory
            rows = torch.arange(a, min(n, a + 256), device=out.device)
            x = (s["q"][t + rows].double().permute(1, 0, 2).contiguous() @ k.transpose(1, 2).contiguous()) * s["scale"]
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            dist = p[None, :] - (ctx - n + rows)[:, None]
            if s["slopes"] is not None:
                x = x + s["slopes"].double()[:, None, None] * math.log(2.0) * dist
            gone = dist > 0
            if case["window"]:
                gone = gone | (dist <= -case["window"])
            out[t + rows] = (torch.softmax(x.masked_fill(gone, -math.inf), -1) @ v).permute(1, 0, 2)
        t += n
    return out
