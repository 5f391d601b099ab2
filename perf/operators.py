"""Cases, plain forms and exact results of the quantised KV cache operators.

Four operators share one cache: pages of 8-bit elements (e4m3 or int8) with one
power-of-two scale per (token, KV head), kept as an E8M0 byte (scale =
2^(byte - 127)).

  store    per-head RMSNorm and RoPE of q and k, q returned in bf16, k and v
           rounded to 8 bits into their cache slots
  decode   attention of one new token per sequence over the cache
  read     the cache of a batch read back to bf16
  prefill  causal attention of prompts, or of prompt chunks after a cached
           prefix, over the cache
"""
import math
import random
import sys

import torch

own = False

DEV = "cuda"
D = 128
EPS = 1e-6


def listed():
    return [
        # one decode step of a single request, 16 query / 8 KV heads
        {"name": "store_one_token", "op": "store", "dtype": "e4m3", "tokens": 1, "hq": 16,
         "hkv": 8, "bs": 16, "top": 2000},
        # a mixed step of odd length, 32 query heads, pages of 32 tokens
        {"name": "store_mixed_257", "op": "store", "dtype": "int8", "tokens": 257, "hq": 32,
         "hkv": 8, "bs": 32, "top": 9000},
        # a full token budget of prompts, 64 query heads
        {"name": "store_prompts_16384", "op": "store", "dtype": "e4m3", "tokens": 16384, "hq": 64,
         "hkv": 8, "bs": 16, "top": 16384},
        # the first steps of a single chat request: latency
        {"name": "decode_one_short", "op": "decode", "dtype": "e4m3", "batch": 1, "lo": 17,
         "hi": 17, "lens_seed": 1, "hq": 16, "hkv": 8, "bs": 16},
        # one request with a long document: the context is split over the GPU
        {"name": "decode_one_long", "op": "decode", "dtype": "int8", "batch": 1, "lo": 30001,
         "hi": 30001, "lens_seed": 1, "hq": 32, "hkv": 8, "bs": 16},
        # one rank's heads of an 8-way tensor parallel model, an odd batch
        {"name": "decode_shard_33", "op": "decode", "dtype": "int8", "batch": 33, "lo": 100,
         "hi": 2000, "lens_seed": 3, "hq": 4, "hkv": 1, "bs": 16},
        # a batch whose lengths differ by four orders of magnitude, 8 query heads a KV head
        {"name": "decode_ragged_64", "op": "decode", "dtype": "e4m3", "batch": 64, "lo": 1,
         "hi": 8192, "lens_seed": 4, "hq": 64, "hkv": 8, "bs": 32},
        # the steady state of a loaded server
        {"name": "decode_batch_256", "op": "decode", "dtype": "e4m3", "batch": 256, "lo": 512,
         "hi": 8192, "lens_seed": 5, "hq": 32, "hkv": 8, "bs": 16},
        # three short contexts read back
        {"name": "read_short_3", "op": "read", "dtype": "int8", "batch": 3, "lo": 1, "hi": 200,
         "lens_seed": 6, "hkv": 8, "bs": 16},
        # long cached prefixes of a chunked step read back
        {"name": "read_long_16", "op": "read", "dtype": "e4m3", "batch": 16, "lo": 1024,
         "hi": 8192, "lens_seed": 7, "hkv": 8, "bs": 16},
        # a few short prompts without a prefix
        {"name": "prefill_prompts_4", "op": "prefill", "dtype": "int8", "batch": 4, "lo": 17,
         "hi": 300, "lens_seed": 8, "prefix": 0, "hq": 16, "hkv": 8, "bs": 16},
        # two prompt chunks of a token-budget step after a cached prefix
        {"name": "prefill_chunks_2", "op": "prefill", "dtype": "e4m3", "batch": 2, "lo": 2048,
         "hi": 2048, "lens_seed": 9, "prefix": 4096, "hq": 32, "hkv": 8, "bs": 16},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "decode", "decode", "read", "prefill"])
    hkv = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 4, 8])
    bs = rng.choice([16, 32, 64])
    seed = rng.randrange(1 << 30)
    if op == "store":
        return {"op": op, "dtype": rng.choice(["e4m3", "int8"]), "tokens": _log(rng, 1, 16384),
                "hq": g * hkv, "hkv": hkv, "bs": bs, "top": _log(rng, 2000, 32000)}
    case = {"op": op, "dtype": rng.choice(["e4m3", "int8"]), "lens_seed": seed, "hkv": hkv,
            "bs": bs}
    if op == "prefill":
        hi = _log(rng, 1, 2048)
        return {**case, "batch": rng.randint(1, 2), "lo": max(1, hi // rng.randint(1, 8)),
                "hi": hi, "prefix": rng.choice([0, _log(rng, 1, 4096)]),
                "hq": min(g * hkv, 32)}
    batch = _log(rng, 1, 256 if op == "decode" else 16)
    hi = _log(rng, 1, 32768 if batch <= 8 and op == "decode" else 8192)
    case.update(batch=batch, lo=max(1, hi // rng.choice([1, 4, 100, 10000])), hi=hi)
    if op == "decode":
        case["hq"] = g * hkv
    return case


def _lens(case):
    """Tokens per sequence (prefill: new tokens), log-uniform; a batch of 8 or
    more has one empty sequence, as a padded decode batch has."""
    r = random.Random(case["lens_seed"])
    lens = [_log(r, case["lo"], case["hi"]) for _ in range(case["batch"])]
    if case["op"] != "prefill" and case["batch"] >= 8:
        lens[case["batch"] // 2] = 0
    return lens


def _prefixes(case):
    r = random.Random(case["lens_seed"] + 1)
    p = case["prefix"]
    return [_log(r, max(1, p // 4), p) if p else 0 for _ in range(case["batch"])]


def _ctx(case):
    lens = _lens(case)
    return [a + b for a, b in zip(lens, _prefixes(case))] if case["op"] == "prefill" else lens


def _up(x, m):
    return -(-x // m) * m


def _pool(case, ctx, gen):
    """A pool of pages in a shuffled order, as a server's block manager leaves
    it, and the batch's block tables (unused entries -1)."""
    bs, hkv, B = case["bs"], case["hkv"], case["batch"]
    need = [-(-n // bs) for n in ctx]
    nb = sum(need) + 3
    width = max(max(need), 1)
    perm = torch.randperm(nb, generator=gen, device=DEV).to(torch.int32)
    tables = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = perm[at:at + n]
        at += n
    x = torch.randn((2, nb, bs, hkv, D), generator=gen, device=DEV, dtype=torch.bfloat16)
    if case["dtype"] == "e4m3":
        data = x.mul_(130.0).clamp_(-448, 448).to(torch.float8_e4m3fn)
    else:
        data = x.mul_(36.0).round_().clamp_(-127, 127).to(torch.int8)
    # the scales of rows whose amplitude varies by a factor of about four
    base = 120 if case["dtype"] == "e4m3" else 122
    scales = torch.randint(base - 2, base + 1, (2, nb, hkv, bs), generator=gen, device=DEV,
                           dtype=torch.uint8)
    return data, scales, tables


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    ints = dict(dtype=torch.int32, device=DEV)
    if case["op"] == "store":
        T, hq, hkv, bs = case["tokens"], case["hq"], case["hkv"], case["bs"]
        # q, k, v are column slices of one projection's output
        qkv = torch.randn((T, hq + 2 * hkv, D), generator=gen, device=DEV)
        qkv[:, hq + hkv:] *= 0.5 * torch.exp(
            0.5 * torch.randn((T, hkv, 1), generator=gen, device=DEV))
        qkv = qkv.to(torch.bfloat16)
        nb = -(-T // bs) + 2
        slots = torch.randperm(nb * bs, generator=gen, device=DEV)[:T].to(torch.int32)
        # one RoPE row per position: 64 words of (cos, sin) bf16 pairs
        pos = torch.arange(case["top"], device=DEV, dtype=torch.float64)
        freq = 1e6 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        ang = pos[:, None] * freq
        table = torch.stack([ang.cos(), ang.sin()], -1).to(torch.bfloat16)
        table = table.view(torch.int32).reshape(-1)
        if case["dtype"] == "e4m3":
            data = torch.zeros((2, nb, bs, hkv, D), dtype=torch.float8_e4m3fn, device=DEV)
        else:
            data = torch.zeros((2, nb, bs, hkv, D), dtype=torch.int8, device=DEV)
        return {"case": case, "q": qkv[:, :hq], "k": qkv[:, hq:hq + hkv], "v": qkv[:, hq + hkv:],
                "slots": slots, "table": table, "data": data,
                "scales": torch.full((2, nb, hkv, bs), 127, dtype=torch.uint8, device=DEV),
                "positions": torch.randint(0, case["top"], (T,), generator=gen, **ints),
                "qw": (1 + 0.2 * torch.randn(D, generator=gen, device=DEV)).to(torch.bfloat16),
                "kw": (1 + 0.2 * torch.randn(D, generator=gen, device=DEV)).to(torch.bfloat16)}
    ctx = _ctx(case)
    data, scales, tables = _pool(case, ctx, gen)
    s = {"case": case, "data": data, "scales": scales, "tables": tables,
         "ctx": torch.tensor(ctx, **ints), "max_ctx": max(max(ctx), 1)}
    if case["op"] == "decode":
        s["q"] = torch.randn((case["batch"], case["hq"], D), generator=gen, device=DEV,
                             dtype=torch.bfloat16)
    if case["op"] == "prefill":
        new = _lens(case)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, **ints)
        s["max_new"] = max(new)
        s["q"] = torch.randn((cu[-1], case["hq"], D), generator=gen, device=DEV,
                             dtype=torch.bfloat16)
    return s


# ----------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------
def _norm_rope(x, w, words, eps):
    """RMSNorm over the head, then rotation of the pairs (2i, 2i+1), in x's type."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.to(x.dtype)
    cs = words.to(x.dtype)[:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]],
                       -1).flatten(-2)


def _quantise(x, dtype):
    """Rows of x (64 bits: the rounded values lie next to borders) -> 8-bit
    values and E8M0 bytes: the smallest power of two that fits the row."""
    amax = x.abs().amax(-1)
    m, ex = torch.frexp(amax)
    if dtype == "e4m3":      # 448 = 1.75 * 2^8
        e = ex - 9 + (m > 0.875).to(ex.dtype)
    else:                    # 127 = (127 / 64) * 2^6
        e = ex - 7 + (m > 127 / 128).to(ex.dtype)
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(-126, 127)
    y = torch.ldexp(x, -e[..., None])
    if dtype == "e4m3":
        step = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp(min=-5) - 4)
        y = (torch.round(y / step) * step).float().to(torch.float8_e4m3fn)
    else:
        y = torch.round(y).to(torch.int8)
    return y, (e + 127).to(torch.uint8)


def _plain_store(s):
    c = s["case"]
    bs = c["bs"]
    words = s["table"].view(torch.bfloat16).view(-1, D // 2, 2)[s["positions"].long()]
    q = _norm_rope(s["q"].float(), s["qw"], words, EPS).to(torch.bfloat16)
    k = _norm_rope(s["k"].double(), s["kw"], words, EPS)
    slot = s["slots"].long()
    blk, off = slot // bs, slot % bs
    for i, x in enumerate((k, s["v"].double())):
        y, e = _quantise(x, c["dtype"])
        s["data"][i].view(torch.uint8)[blk, off] = y.view(torch.uint8)
        s["scales"][i][blk, :, off] = e
    return q


def _gathered(s):
    """The batch's K and V in 32 bits, [2, B, width * bs, Hkv, D]."""
    t = s["tables"].clamp(min=0).long()
    x = s["data"].view(torch.uint8)[:, t].view(s["data"].dtype).float()
    x = x * torch.exp2(s["scales"][:, t].float() - 127).transpose(-1, -2)[..., None]
    return x.flatten(2, 3)


def _attend(q, k, v, seen):
    """q [B, n, Hq, D], k/v [B, L, Hkv, D], seen [B, n, L] -> [B, n, Hq, D]; rows that see
    nothing come out 0."""
    B, n, hq, _ = q.shape
    hkv = k.shape[2]
    q = q.float().view(B, n, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4)
    w = torch.matmul(q, k.permute(0, 2, 3, 1)[:, :, None]) * (1 / math.sqrt(D))
    w = w.masked_fill_(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w, v.permute(0, 2, 1, 3)[:, :, None])
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, hq, D)


def _plain_decode(s):
    k, v = _gathered(s)
    seen = torch.arange(k.shape[1], device=DEV)[None] < s["ctx"][:, None]
    return _attend(s["q"][:, None], k, v, seen[:, None])[:, 0].to(torch.bfloat16)


def _plain_read(s):
    x = _gathered(s)[:, :, :s["max_ctx"]]
    seen = torch.arange(s["max_ctx"], device=DEV)[None] < s["ctx"][:, None]
    return torch.where(seen[None, :, :, None, None], x, torch.zeros_like(x)).to(torch.bfloat16)


def _plain_prefill(s):
    k, v = _gathered(s)
    cu, n = s["cu"].long(), s["max_new"]
    T = s["q"].shape[0]
    new = cu[1:] - cu[:-1]
    i = torch.arange(n, device=DEV)
    rows = (cu[:-1, None] + i).clamp(max=T - 1)
    pos = (s["ctx"] - new)[:, None] + i
    seen = torch.arange(k.shape[1], device=DEV) <= pos[:, :, None]
    o = _attend(s["q"][rows], k, v, seen)
    tok = torch.arange(T, device=DEV)
    seq = torch.searchsorted(cu, tok, right=True) - 1
    return o[seq, tok - cu[seq]].to(torch.bfloat16)


# ----------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        if "vllm-jax_b200" not in sys.path:
            sys.path.insert(0, "vllm-jax_b200")
        from vllm_b200.kernels import quantized_cache as qc
        cache = qc.QuantizedKVCache(s["data"], s["scales"])
        if c["op"] == "store":
            q = qc.kv_store_quantized(s["q"], s["k"], s["v"], cache, s["slots"], s["positions"],
                                      s["qw"], s["kw"], eps=EPS, table=s["table"])
        elif c["op"] == "decode":
            return qc.paged_decode_quantized(s["q"], cache, s["tables"], s["ctx"])
        elif c["op"] == "read":
            return qc.read_kv_cache(cache, s["tables"], s["ctx"], s["max_ctx"])
        else:
            return qc.paged_prefill_quantized(s["q"], cache, s["tables"], s["cu"], s["ctx"],
                                              max_seqlen_q=s["max_new"],
                                              max_context_len=s["max_ctx"])
    elif c["op"] == "store":
        q = _plain_store(s)
    else:
        return {"decode": _plain_decode, "read": _plain_read,
                "prefill": _plain_prefill}[c["op"]](s)
    # the cache's own values: elements, and scales as the powers of two they stand for
    return {"q": q, "data": s["data"], "scales": s["scales"].view(torch.float8_e8m0fnu)}


# ----------------------------------------------------------------------------
def work(case):
    hkv, ctx = case["hkv"], None
    if case["op"] == "store":
        T, hq = case["tokens"], case["hq"]
        return {"bytes": T * ((2 * hq + 2 * hkv) * D * 2 + 2 * hkv * (D + 1) + 8)
                + min(T, case["top"]) * D * 2,
                "flops": T * (hq + hkv) * D * 8}
    ctx = _ctx(case)
    cached = sum(ctx) * hkv * 2 * (D + 1) + sum(-(-n // case["bs"]) for n in ctx) * 4
    if case["op"] == "read":
        return {"bytes": cached + 2 * case["batch"] * max(max(ctx), 1) * hkv * D * 2,
                "flops": sum(ctx) * hkv * 2 * D}
    hq = case["hq"]
    if case["op"] == "decode":
        return {"bytes": cached + 2 * case["batch"] * hq * D * 2, "flops": sum(ctx) * hq * 4 * D}
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(_lens(case), _prefixes(case)))
    return {"bytes": cached + 2 * sum(_lens(case)) * hq * D * 2, "flops": pairs * hq * 4 * D}


# ----------------------------------------------------------------------------
def _exact_rows(x, dtype):
    """Nearest 8-bit value by search in the sorted list of all of them (ties to
    the even code), with the smallest sufficient power-of-two scale."""
    top = 448.0 if dtype == "e4m3" else 127.0
    amax = x.abs().amax(-1)
    e = torch.full_like(amax, -126)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):     # largest e whose predecessor is too small
        e = torch.where(amax > top * torch.exp2(e + step - 1), e + step, e)
    e = torch.where(amax > 0, e, torch.zeros_like(e))
    if dtype == "e4m3":
        vals = torch.arange(0, 127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    else:
        vals = torch.arange(0, 128, device=DEV)
    vals = vals.double()
    mids = (vals[1:] + vals[:-1]) / 2
    y = x * torch.exp2(-e)[..., None]
    lo = torch.searchsorted(mids, y.abs().contiguous(), right=False)
    hi = torch.searchsorted(mids, y.abs().contiguous(), right=True)
    code = torch.where(lo % 2 == 0, lo, hi)       # equal unless the value is a midpoint
    return torch.copysign(vals[code], y), torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        table = s["table"].view(torch.bfloat16).double().view(-1, D)

        def turned(x, w):
            x = x.double()
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS) * w.double()
            z = torch.view_as_complex(x.unflatten(-1, (D // 2, 2)).contiguous())
            r = torch.view_as_complex(table[s["positions"].long()].unflatten(-1, (D // 2, 2)))
            return torch.view_as_real(z * r[:, None]).flatten(-2)

        data, scales = s["data"].double(), torch.ones_like(s["scales"], dtype=torch.float64)
        slot, bs = s["slots"].long(), case["bs"]
        for i, x in enumerate((turned(s["k"], s["kw"]), s["v"].double())):
            y, e = _exact_rows(x, case["dtype"])
            data[i].view(-1, case["hkv"], D)[slot] = y
            scales[i].transpose(1, 2)[slot // bs, slot % bs] = e
        return {"q": turned(s["q"], s["qw"]), "data": data, "scales": scales}
    ctx, bs, hkv = _ctx(case), case["bs"], case["hkv"]
    if case["op"] == "read":
        out = torch.zeros((2, case["batch"], s["max_ctx"], hkv, D), dtype=torch.float64,
                          device=DEV)
    else:
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    first = 0
    for b, n in enumerate(ctx):
        if n == 0:
            continue
        pages = s["tables"][b, :-(-n // bs)].long()
        kv = []
        for i in range(2):
            x = s["data"][i].view(torch.uint8)[pages].view(s["data"].dtype).double()
            f = torch.pow(2.0, s["scales"][i][pages].double() - 127)
            kv.append((x * f.permute(0, 2, 1)[..., None]).reshape(-1, hkv, D)[:n])
        if case["op"] == "read":
            out[0, b, :n], out[1, b, :n] = kv
            continue
        g = case["hq"] // hkv
        new = _lens(case)[b] if case["op"] == "prefill" else 1
        rows = s["q"][first:first + new].double() if case["op"] == "prefill" else \
            s["q"][b:b + 1].double()
        late = torch.arange(n, device=DEV)[None] > torch.arange(n - new, n, device=DEV)[:, None]
        for h in range(case["hq"]):
            w = rows[:, h] @ kv[0][:, h // g].T / math.sqrt(D)
            w = torch.softmax(w.masked_fill(late, -math.inf), -1)
            at = slice(first, first + new) if case["op"] == "prefill" else slice(b, b + 1)
            out[at, h] = w @ kv[1][:, h // g]
        first += new
    return out
