"""The quantised KV cache on the GPU against 64-bit NumPy (oracle/quantized.py).

Tolerances. The cache itself is exact: a stored row is the correctly rounded
one and reading back rounds nothing, so both are compared bit for bit. A bf16
result r is rounded by at most half a step, 2^-8 |r|. In decode attention the
weights enter the product rounded to f16 (half a step: 2^-11 of each, so 2^-11
sum p|v|); the scores' fp32 sums of 128 products are off by at most
128 * 2^-24 * sum|q_i k_i| * scale, below 2^-13 here (sum|q_i k_i| * scale <
16), which moves a weight by that much relatively, and the fp32 sum of up to
2^14 weighted values by at most 2^14 / 16 additions of 2^-24, 2^-14: together
below (2^-11 + 2^-12) sum p|v|. Prefill rounds its weights to bf16: 2^-8
instead of 2^-11.
"""
import math

import numpy as np
import pytest
import torch

from oracle import quantized as oq
from oracle.bf16 import bf16

pytestmark = pytest.mark.gpu

D = 128
TORCH = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def _t(x, dtype=torch.bfloat16):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def _i(x):
    return torch.tensor(np.asarray(x, np.int32), device="cuda")


def _cache(codes, scales, dtype):
    """codes (2, nb, bs, H, D) uint8, scales (2, nb, H, bs) uint8 -> QuantizedKVCache."""
    from vllm_b200.kernels.quantized_cache import QuantizedKVCache
    return QuantizedKVCache(_t(codes, torch.uint8).view(TORCH[dtype]), _t(scales, torch.uint8))


def _random_pool(rng, nb, bs, H, dtype, spread=2):
    codes = rng.integers(0, 256, (2, nb, bs, H, D)).astype(np.uint8)
    if dtype == "e4m3":
        codes = np.where((codes & 127) == 127, 0, codes)      # no NaN codes
        # e4m3 codes drawn evenly are mostly tiny: use rounded normal numbers
        codes[:], _ = oq.quantise_rows(rng.standard_normal(codes.shape), dtype)
    scales = rng.integers(120 - spread, 121 + spread, (2, nb, H, bs)).astype(np.uint8)
    return codes.astype(np.uint8), scales


def _tables(rng, lens, nb, bs, width):
    perm, at = rng.permutation(nb), 0
    bt = np.full((len(lens), width), -1, np.int32)
    for b, n in enumerate(lens):
        m = min(-(-n // bs), width)
        bt[b, :m] = perm[at:at + m]
        at += m
    assert at <= nb
    return bt


def _values(codes, scales, dtype):
    return [oq.dequantise(codes[i], scales[i], dtype) for i in range(2)]


def _check(got, ref, mag, weight):
    got = got.double().cpu().numpy()
    err = np.abs(got - ref)
    tol = 2.0 ** -8 * np.abs(ref) + weight * mag + 1e-30
    assert np.isfinite(got).all() and (err <= tol).all(), \
        f"worst {np.max(err / tol):.3f} of the tolerance"


DECODE = 2.0 ** -11 + 2.0 ** -12
PREFILL = 2.0 ** -8 + 2.0 ** -11


# ----------------------------------------------------------------------------- store
def _store_case(T, Hq, Hkv, bs, dtype, seed, norm=True, rope=True, edit=None, top=5000,
                table_len=4096):
    from vllm_b200.kernels.kv_store import rope_table
    from vllm_b200.kernels.quantized_cache import kv_store_quantized
    rng = np.random.default_rng(seed)
    nb = -(-T // bs) + 3
    qkv = bf16(rng.standard_normal((T, Hq + 2 * Hkv, D)) * np.exp(
        rng.uniform(-2, 2, (T, Hq + 2 * Hkv, 1))))
    if edit:
        edit(qkv)
    qw, kw = (bf16(1 + 0.3 * rng.standard_normal(D)) for _ in range(2))
    pos = rng.integers(0, top, T).astype(np.int32)
    slots = rng.permutation(nb * bs)[:T].astype(np.int32)
    if T > 4:
        slots[[1, 3]] = -1, nb * bs              # dropped
    old_codes, old_scales = _random_pool(rng, nb, bs, Hkv, dtype)
    cache = _cache(old_codes, old_scales, dtype)
    d = _t(qkv)
    # built by the table kernel: its words are the reference for positions past a short table
    full = rope_table(torch.device("cuda", 0), 1e6, max(top, 8192))
    table = full[:table_len * 64]
    q = kv_store_quantized(d[:, :Hq], d[:, Hq:Hq + Hkv], d[:, Hq + Hkv:], cache, _i(slots),
                           _i(pos) if rope else None, _t(qw) if norm else None,
                           _t(kw) if norm else None, norm=norm, rope=rope, table=table)
    torch.cuda.synchronize()
    words = full.view(torch.bfloat16).double().cpu().numpy().reshape(-1, D // 2, 2)
    cs = words[pos] if rope else None
    x = qkv.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        yq = oq.norm_rope(x[:, :Hq], qw.astype(np.float64) if norm else None, cs, 1e-6)
        yk = oq.norm_rope(x[:, Hq:Hq + Hkv], kw.astype(np.float64) if norm else None, cs, 1e-6)
        new = [oq.quantise_rows(y, dtype) for y in (yk, x[:, Hq + Hkv:])]
    codes, scales = old_codes.copy(), old_scales.copy()
    for t, s in enumerate(slots):
        if 0 <= s < nb * bs:
            for i in range(2):
                codes[i, s // bs, s % bs] = new[i][0][t]
                scales[i, s // bs, :, s % bs] = new[i][1][t]
    np.testing.assert_array_equal(cache.data.view(torch.uint8).cpu().numpy(), codes)
    np.testing.assert_array_equal(cache.scales.cpu().numpy(), scales)
    got = q.double().cpu().numpy()
    ok = np.isfinite(yq).all(-1)
    # bf16 rounding, and fp32 arithmetic on values of the row's size
    tol = 2.0 ** -8 * np.abs(yq) + 2.0 ** -20 * np.abs(yq).max(-1, keepdims=True) + 1e-38
    assert (np.abs(got - yq)[ok] <= tol[ok]).all()
    assert not np.isfinite(got[~ok]).all(-1).any()
    return cache


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("T,Hq,Hkv,bs", [(1, 16, 8, 16), (2, 1, 1, 16), (7, 5, 3, 32),
                                         (257, 32, 8, 16), (100, 64, 8, 64), (33, 4, 1, 48)])
def test_store_matches_oracle(T, Hq, Hkv, bs, dtype):
    _store_case(T, Hq, Hkv, bs, dtype, seed=T)


@pytest.mark.parametrize("norm,rope", [(False, False), (True, False), (False, True)])
def test_store_without_norm_or_rope(norm, rope):
    _store_case(50, 8, 2, 16, "int8", 3, norm, rope)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_store_of_unusual_rows(dtype):
    """Zero rows, infinities and NaN, the largest and smallest magnitudes; positions past
    the table (computed in the kernel)."""
    def edit(x):
        x[0] = 0
        x[5, :, 3] = np.inf
        x[6, :, 100] = np.nan
        x[7] = bf16(x[7] * 1e-38)
        x[8] = bf16(x[8] * 1e36)
        x[9] = 0
        x[9, :, 64] = bf16(np.float32(1e-40))
        x[10, :, :] = 1.0
    _store_case(40, 6, 2, 16, dtype, 4, norm=False, rope=False, edit=edit)
    _store_case(40, 6, 2, 16, dtype, 5, norm=True, rope=True, top=8000, table_len=64)


def test_store_kv_only_and_in_place_q():
    from vllm_b200.kernels.quantized_cache import QuantizedKVCache, kv_store_quantized
    rng = np.random.default_rng(0)
    a, b = (QuantizedKVCache.zeros(4, 16, 2, dtype="e4m3", device="cuda") for _ in range(2))
    qkv = _t(bf16(rng.standard_normal((20, 8, D))))
    w, pos, slots = _t(np.ones(D)), _i(np.arange(20)), _i(np.arange(20) + 7)
    assert kv_store_quantized(None, qkv[:, 4:6], qkv[:, 6:], a, slots, pos, None, w) is None
    mine = qkv.clone()
    q = kv_store_quantized(mine[:, :4], qkv[:, 4:6], qkv[:, 6:], b, slots, pos, w, w,
                           q_out=mine[:, :4])
    ref = kv_store_quantized(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], b, slots, pos, w, w)
    assert q.data_ptr() == mine.data_ptr()
    assert torch.equal(q, ref) and torch.equal(mine[:, 4:], qkv[:, 4:])
    assert torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8))
    assert torch.equal(a.scales, b.scales)


# ----------------------------------------------------------------------------- read
@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("H,bs,lens,L", [(8, 16, [1, 0, 33, 200], 0), (1, 32, [64, 5], 70),
                                         (3, 48, [100], 17), (2, 64, [0, 0], 1)])
def test_read_back_is_exact(H, bs, lens, L, dtype):
    from vllm_b200.kernels.quantized_cache import read_kv_cache
    rng = np.random.default_rng(len(lens))
    nb = sum(-(-n // bs) for n in lens) + 2
    width = max(-(-n // bs) for n in lens) + 1
    codes, scales = _random_pool(rng, nb, bs, H, dtype, spread=100)
    bt = _tables(rng, lens, nb, bs, width)
    rows = L or width * bs
    out = torch.full((2, len(lens), rows, H, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    got = read_kv_cache(_cache(codes, scales, dtype), _i(bt), _i(lens), L, out=out)
    vals = _values(codes, scales, dtype)
    ref = np.zeros((2, len(lens), rows, H, D))
    for b, n in enumerate(lens):
        for i in range(2):
            g = oq.gather(vals[i], bt[b], n)[:rows]
            ref[i, b, :len(g)] = g
    np.testing.assert_array_equal(got.double().cpu().numpy(), ref)


def test_read_back_of_every_code_and_scale():
    from vllm_b200.kernels.quantized_cache import read_kv_cache
    for dtype in ("e4m3", "int8"):
        codes = np.zeros((2, 8, 32, 1, D), np.uint8)
        codes[:] = np.arange(D)
        codes[1] += 128
        scales = np.arange(256, dtype=np.uint8).reshape(1, 8, 1, 32).repeat(2, 0)
        # byte 255 stands with zero elements
        codes[:, 7, 31] = 0
        got = read_kv_cache(_cache(codes, scales, dtype), _i([np.arange(8)]), _i([256]))
        ref = np.stack([oq.dequantise(codes[i], scales[i], dtype) for i in range(2)])
        ref = torch.from_numpy(ref.reshape(2, 1, 256, 1, D)).to(torch.bfloat16)
        # past bf16's range the product is infinite or subnormal: the same rounding
        assert torch.equal(got.cpu().nan_to_num(7.0, 1e38, -1e38),
                           ref.nan_to_num(7.0, 1e38, -1e38))


# ----------------------------------------------------------------------------- decode
def _decode_case(B, Hq, Hkv, bs, lens, dtype, seed, spread=2, scale=None, width=None, q_scale=1.0):
    from vllm_b200.kernels.quantized_cache import paged_decode_quantized
    rng = np.random.default_rng(seed)
    width = width or max(max(-(-n // bs) for n in lens) + 2, 1)
    nb = sum(min(-(-n // bs), width) for n in lens) + 3
    codes, scales = _random_pool(rng, nb, bs, Hkv, dtype, spread)
    bt = _tables(rng, lens, nb, bs, width)
    # what no sequence covers holds NaN codes and NaN scales
    live = np.zeros((nb, bs), bool)
    for b, n in enumerate(lens):
        for t in range(min(n, width * bs)):
            live[bt[b, t // bs], t % bs] = True
    if dtype == "e4m3":
        codes[:, ~live] = 0x7f
    scales.transpose(0, 1, 3, 2)[:, ~live] = 255
    q = bf16(rng.standard_normal((B, Hq, D)) * q_scale)
    out = torch.full((B, Hq, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    got = paged_decode_quantized(_t(q), _cache(codes, scales, dtype), _i(bt), _i(lens), scale,
                                 out=out)
    torch.cuda.synchronize()
    vals = _values(np.where(live[None, :, :, None, None], codes, 0).astype(np.uint8),
                   np.where(live[None, :, None, :], scales, 127), dtype)
    ref, mag = np.zeros((B, Hq, D)), np.zeros((B, Hq, D))
    for b, n in enumerate(lens):
        n = min(n, width * bs)
        if n:
            k, v = (oq.gather(vals[i], bt[b], n) for i in range(2))
            o, m = oq.attend(q[b:b + 1].astype(np.float64), k, v, n - 1,
                             scale if scale is not None else 1 / math.sqrt(D))
            ref[b], mag[b] = o[0], m[0]
    _check(got, ref, mag, DECODE)
    return got


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("B,Hq,Hkv,bs,lens", [
    (1, 16, 8, 16, [1]),
    (1, 1, 1, 16, [16]),
    (5, 32, 8, 16, [0, 15, 16, 17, 1000]),
    (3, 64, 8, 16, [4000, 33, 2048]),
    (6, 4, 1, 16, [700, 1, 2, 3000, 48, 129]),
    (4, 6, 3, 48, [31, 96, 33, 2500]),
    (2, 16, 1, 64, [64, 5000]),
    (2, 48, 4, 32, [100, 999]),
    (3, 5, 5, 16, [70, 0, 300]),
    (3, 18, 2, 16, [70, 0, 300]),
    (1, 32, 8, 16, [12345]),
])
def test_decode_matches_oracle(B, Hq, Hkv, bs, lens, dtype):
    _decode_case(B, Hq, Hkv, bs, lens, dtype, seed=B * 100 + Hq)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_decode_many_sequences(dtype):
    rng = np.random.default_rng(8)
    lens = np.round(np.exp(rng.uniform(0, np.log(600), 300))).astype(int)
    lens[[0, 7, 8, 9, 120, 299]] = 0
    lens[200:260] = 0                      # a run of empty rows
    _decode_case(300, 8, 2, 16, lens.tolist(), dtype, 9)


def test_decode_batch_larger_than_a_block_of_threads():
    lens = [(i * 7) % 40 for i in range(2500)]
    _decode_case(2500, 2, 1, 16, lens, "int8", 10)


@pytest.mark.parametrize("Hq,Hkv,dtype", [(74, 37, "e4m3"), (8 * 37, 37, "int8"),
                                          (370, 37, "e4m3"), (64, 64, "int8"),
                                          (128, 64, "e4m3"), (74, 37, "int8")])
def test_decode_of_so_many_pages_that_a_part_is_dealt(Hq, Hkv, dtype):
    """Enough work (32 pages a warp and KV head) that a fifth of it is dealt in pieces:
    against 64 bits, the same bits every time, and on two streams at once."""
    from vllm_b200.kernels.quantized_cache import (QuantizedKVCache,
                                                   decode_quantized_workspace_bytes,
                                                   paged_decode_quantized)
    lens = [9001, 17, 0, 1, 12000, 3, 333, 300, 16, 11000, 8000, 700, 90, 32]
    bs, B = 32, len(lens)
    gen = torch.Generator(device="cuda").manual_seed(Hq)
    need = [-(-n // bs) for n in lens]
    nb, width = sum(need) + 1, max(need)
    x = torch.randn((2, nb, bs, Hkv, D), generator=gen, device="cuda")
    data = ((x * 100).clamp(-448, 448).to(torch.float8_e4m3fn) if dtype == "e4m3"
            else (x * 36).round().clamp(-127, 127).to(torch.int8))
    scales = torch.randint(119, 122, (2, nb, Hkv, bs), generator=gen, device="cuda",
                           dtype=torch.uint8)
    del x
    perm = torch.randperm(nb, generator=gen, device="cuda").to(torch.int32)
    bt = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[at:at + n]
        at += n
    q = torch.randn((B, Hq, D), generator=gen, device="cuda", dtype=torch.bfloat16)
    cache, ln = QuantizedKVCache(data, scales), _i(lens)
    out = paged_decode_quantized(q, cache, bt, ln)
    ref, mag = torch.zeros((2, B, Hq, D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n:
            t = bt[b, :need[b]].long()
            k, v = (data[i].view(torch.uint8)[t].view(data.dtype).double()
                    * torch.exp2(scales[i][t].double() - 127).transpose(1, 2)[..., None]
                    for i in range(2))
            k, v = (y.flatten(0, 1)[:n].permute(1, 0, 2) for y in (k, v))     # [Hkv, n, D]
            p = torch.softmax(q[b].double().view(Hkv, -1, D) @ k.transpose(1, 2) / math.sqrt(D), -1)
            ref[b], mag[b] = (p @ v).view(Hq, D), (p @ v.abs()).view(Hq, D)
    _check(out, ref.cpu().numpy(), mag.cpu().numpy(), DECODE)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    again = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                again.append(paged_decode_quantized(q, cache, bt, ln))
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for o in again)
    # whatever the scratch holds before the call (counts of pieces among it)
    ws = torch.empty(decode_quantized_workspace_bytes(B, Hq, Hkv, width, bs) // 4,
                     dtype=torch.int32, device="cuda")
    # (and often: a stage refilled before its page is read shows in one call of ten)
    for word in (0, 1, 2, 3, -1, 0x7fc00000) * 10:
        ws.fill_(word)
        assert torch.equal(paged_decode_quantized(q, cache, bt, ln, workspace=ws.view(torch.uint8)),
                           out)


def test_decode_context_longer_than_the_table_is_cut():
    _decode_case(2, 8, 2, 16, [400, 37], "e4m3", 11, width=5)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_decode_scales_of_very_different_rows(dtype):
    """Row scales from 2^-20 to 2^20 within a sequence: scores saturate the softmax
    and values of small weight are large, or the other way round."""
    _decode_case(3, 8, 2, 16, [200, 1000, 31], dtype, 12, spread=20, scale=1e-7)
    _decode_case(3, 16, 1, 16, [200, 1000, 31], dtype, 13, spread=30, scale=1e-10)


def test_decode_large_and_small_queries():
    _decode_case(2, 8, 2, 16, [100, 333], "e4m3", 14, q_scale=1e30, scale=1e-31)
    _decode_case(2, 8, 2, 16, [100, 333], "int8", 15, q_scale=1e-30, scale=1e29)
    _decode_case(2, 8, 2, 16, [100, 333], "int8", 16, scale=0.0)


def test_decode_zero_value_rows_keep_their_weight():
    """A zero row of V counts in the softmax's sum, whatever its neighbours' scales."""
    from vllm_b200.kernels.quantized_cache import paged_decode_quantized
    for tiny in (120, 60, 2):
        codes = np.zeros((2, 2, 16, 1, D), np.uint8)
        codes[1] = 1                                    # int8 ones
        scales = np.full((2, 2, 1, 16), tiny, np.uint8)
        zero, byte = oq.quantise_rows(np.zeros(D), "int8")
        codes[1, 0, 3], scales[1, 0, 0, 3] = zero, byte
        out = paged_decode_quantized(_t(np.ones((1, 4, D))), _cache(codes, scales, "int8"),
                                     _i([[0, 1]]), _i([20]))
        ref = 19 / 20 * 2.0 ** (tiny - 127)
        np.testing.assert_allclose(out.double().cpu().numpy(), ref, rtol=2.0 ** -8 + 2.0 ** -10)


def test_decode_nan_row_reaches_its_sequence_only():
    from vllm_b200.kernels.quantized_cache import paged_decode_quantized
    rng = np.random.default_rng(17)
    for which in (0, 1):
        codes, scales = _random_pool(rng, 8, 16, 2, "e4m3")
        codes[which, 1, 3, 1], scales[which, 1, 1, 3] = 0, 255
        bt = np.arange(8).reshape(2, 4)
        out = paged_decode_quantized(_t(rng.standard_normal((2, 4, D))),
                                     _cache(codes, scales, "e4m3"), _i(bt), _i([40, 64]))
        bad = torch.isnan(out).all(-1).cpu().numpy()
        np.testing.assert_array_equal(bad, [[False, False, True, True], [False] * 4])
        assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, :2]).all()


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_layouts_and_strides(dtype):
    """Head-major pages, a pool that is a slice of a larger one, and block tables that
    are columns of a wider table give the packed layout's bits."""
    from vllm_b200.kernels.quantized_cache import (QuantizedKVCache, paged_decode_quantized,
                                                   paged_prefill_quantized, read_kv_cache)
    rng = np.random.default_rng(18)
    nb, bs, H, lens = 24, 16, 4, [100, 33, 200]
    codes, scales = _random_pool(rng, nb, bs, H, dtype)
    bt = _tables(rng, lens, nb, bs, 13)
    a = _cache(codes, scales, dtype)
    raw = a.data.view(torch.uint8)
    head_major = raw.permute(0, 3, 1, 2, 4).contiguous().permute(0, 2, 3, 1, 4).view(TORCH[dtype])
    wide = torch.zeros((2, nb, bs, H + 2, D), dtype=torch.uint8, device="cuda")
    wide[:, :, :, 1:H + 1] = raw
    wide_s = torch.zeros((2, nb, H + 3, bs), dtype=torch.uint8, device="cuda")
    wide_s[:, :, 2:H + 2] = a.scales
    tables = torch.full((3, 40), 9999, dtype=torch.int32, device="cuda")
    tables[:, 5:18] = _i(bt)
    q = _t(bf16(rng.standard_normal((3, 8, D))))
    qp = _t(bf16(rng.standard_normal((30, 8, D))))
    cu, ln = _i([0, 10, 20, 30]), _i(lens)
    ref = (paged_decode_quantized(q, a, _i(bt), ln), read_kv_cache(a, _i(bt), ln),
           paged_prefill_quantized(qp, a, _i(bt), cu, ln, 10))
    for c in (QuantizedKVCache(head_major, a.scales),
              QuantizedKVCache(wide[:, :, :, 1:H + 1].view(TORCH[dtype]), wide_s[:, :, 2:H + 2])):
        t = tables[:, 5:18]
        got = (paged_decode_quantized(q, c, t, ln), read_kv_cache(c, t, ln),
               paged_prefill_quantized(qp, c, t, cu, ln, 10))
        for x, y in zip(got, ref):
            assert torch.equal(x, y)


def test_decode_pool_beyond_32_bit_offsets():
    """Blocks whose element offsets pass 2^32, and scale offsets that pass 2^25."""
    from vllm_b200.kernels.quantized_cache import (QuantizedKVCache, kv_store_quantized,
                                                   paged_decode_quantized, read_kv_cache)
    nb, bs, H = 300_000, 16, 8
    cache = QuantizedKVCache.zeros(nb, bs, H, dtype="int8", device="cuda")
    assert nb * bs * H * D > 2 ** 32
    rng = np.random.default_rng(19)
    T = 50
    blocks = [nb - 1, 3, nb - 7, nb // 2]
    slots = np.concatenate([np.arange(16) + b * bs for b in blocks])[:T]
    k, v = (bf16(rng.standard_normal((T, H, D))) for _ in range(2))
    kv_store_quantized(None, _t(k), _t(v), cache, _i(slots), norm=False, rope=False)
    bt = _i([blocks])
    got = read_kv_cache(cache, bt, _i([T]), T)
    vals = []
    for i, x in enumerate((k, v)):
        codes, b = oq.quantise_rows(x.astype(np.float64), "int8")
        vals.append(oq.element_values(codes, "int8") * np.exp2(b.astype(float) - 127)[..., None])
        np.testing.assert_array_equal(got[i, 0].double().cpu().numpy(), vals[i])
    q = bf16(rng.standard_normal((1, 16, D)))
    out = paged_decode_quantized(_t(q), cache, bt, _i([T]))
    _check(out, *oq.attend(q.astype(np.float64), *vals, T - 1, 1 / math.sqrt(D)), DECODE)


# ----------------------------------------------------------------------------- prefill
@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("Hq,Hkv,bs,new,prefix", [
    (16, 8, 16, [17, 64, 1], [0, 0, 0]),
    (8, 2, 32, [130, 5, 0, 1], [0, 200, 16, 300]),
    (4, 1, 16, [300], [129]),
    (16, 1, 64, [33, 40], [7, 600]),
    (32, 8, 16, [100, 90, 1, 100, 77, 100, 99, 3], [0, 5, 0, 20, 16, 0, 17, 100]),   # read back first
])
def test_prefill_matches_oracle(Hq, Hkv, bs, new, prefix, dtype, monkeypatch):
    from vllm_b200.kernels import quantized_cache as qc
    rng = np.random.default_rng(sum(new))
    ctx = [a + b for a, b in zip(new, prefix)]
    nb, width = sum(-(-n // bs) for n in ctx) + 2, max(-(-n // bs) for n in ctx) + 1
    codes, scales = _random_pool(rng, nb, bs, Hkv, dtype)
    bt = _tables(rng, ctx, nb, bs, width)
    cu = np.concatenate([[0], np.cumsum(new)])
    T = int(cu[-1])
    q = bf16(rng.standard_normal((T + 5, Hq, D)))          # five padding rows
    cache = _cache(codes, scales, dtype)
    got = qc.paged_prefill_quantized(_t(q), cache, _i(bt), _i(cu), _i(ctx), max(new))
    vals = _values(codes, scales, dtype)
    ref, mag = np.zeros(q.shape), np.zeros(q.shape)
    for s, (n, p) in enumerate(zip(new, prefix)):
        if n:
            k, v = (oq.gather(vals[i], bt[s], n + p) for i in range(2))
            rows = slice(cu[s], cu[s + 1])
            ref[rows], mag[rows] = oq.attend(q[rows].astype(np.float64), k, v, p, 1 / math.sqrt(D))
    _check(got, ref, mag, PREFILL)
    # in groups of one sequence, with an exact bound on the contexts: the same bits
    monkeypatch.setattr(qc, "PREFILL_SCRATCH_ROWS", 1)
    again = qc.paged_prefill_quantized(_t(q), cache, _i(bt), _i(cu), _i(ctx), max(new),
                                       max_context_len=max(ctx))
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_prefill_of_every_code_and_scale(dtype):
    """One token that sees itself alone: its result is its V row, whatever element and
    scale, and NaN for byte 255. Where the row's value leaves bf16's range or its normal
    numbers, it is what reading back gives."""
    from vllm_b200.kernels.quantized_cache import paged_prefill_quantized, read_kv_cache
    S = 512
    codes = np.zeros((2, S, 16, 1, D), np.uint8)
    codes[1, :, 0, 0] = np.arange(2 * D).reshape(2, D)[np.arange(S) % 2]
    if dtype == "e4m3":
        codes = np.where((codes & 127) == 127, 0, codes)      # no NaN codes
    scales = np.full((2, S, 1, 16), 127, np.uint8)
    scales[1, :, 0, 0] = np.arange(S) // 2
    codes[1, 510:, 0] = 0
    cache, bt = _cache(codes, scales, dtype), _i(np.arange(S)[:, None])
    one, cu = _i(np.ones(S)), _i(np.arange(S + 1))
    q = _t(bf16(np.random.default_rng(24).standard_normal((S, 2, D))))
    out = paged_prefill_quantized(q, cache, bt, cu, one, 1)
    ref = read_kv_cache(cache, bt, one, 1)[1, :, 0]           # [S, 1, D]
    assert torch.equal(out.nan_to_num(7.0, 1e38, -1e38),
                       ref.expand(S, 2, D).nan_to_num(7.0, 1e38, -1e38))
    assert torch.isnan(out[510:]).all() and torch.isfinite(out[:480]).all()


@pytest.mark.parametrize("lens", [(70, 1, 129), (900, 1, 1029)])
def test_prefill_scratch_garbage_does_not_matter(lens):
    """The scratch comes uninitialised: memory full of NaN gives the same bits."""
    from vllm_b200.kernels import quantized_cache as qc
    rng = np.random.default_rng(20)
    need = sum(-(-n // 16) for n in lens)
    codes, scales = _random_pool(rng, need, 16, 2, "e4m3")
    bt = _tables(rng, lens, need, 16, -(-max(lens) // 16))
    q = _t(bf16(rng.standard_normal((sum(lens), 16, D))))
    args = (q, _cache(codes, scales, "e4m3"), _i(bt), _i(np.cumsum((0,) + lens)), _i(lens),
            max(lens))
    a = qc.paged_prefill_quantized(*args)
    junk = [torch.full((1 << 22,), float("nan"), device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    del junk
    assert torch.equal(a, qc.paged_prefill_quantized(*args)) and torch.isfinite(a).all()


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("Hq,Hkv,bs,new,prefix", [
    (8, 2, 16, [1], [2000]),
    (4, 1, 16, [3, 0, 2], [1500, 700, 4000]),
    (16, 8, 32, [40], [1030]),
    (32, 4, 16, [2, 17, 5], [5000, 3, 0]),      # more parts than key tiles
    (8, 1, 16, [300], [1400]),                  # parts that early rows see nothing of
    (16, 1, 48, [700], [2500]),
    (12, 3, 16, [1, 1, 1, 1], [3000, 1023, 1024, 1025]),
    (32, 8, 16, [256], [2500]),                 # these two are read back first
    (8, 1, 32, [900, 40], [1400, 9]),
])
def test_prefill_split_over_keys_matches_oracle(Hq, Hkv, bs, new, prefix, dtype):
    """Few new tokens after long prefixes; scratch full of NaN; the same bits again."""
    from vllm_b200 import _native
    from vllm_b200.kernels import quantized_cache as qc
    rng = np.random.default_rng(sum(prefix))
    ctx = [a + b for a, b in zip(new, prefix)]
    nb, width = sum(-(-n // bs) for n in ctx) + 2, max(-(-n // bs) for n in ctx) + 1
    codes, scales = _random_pool(rng, nb, bs, Hkv, dtype)
    bt = _tables(rng, ctx, nb, bs, width)
    cu = np.concatenate([[0], np.cumsum(new)])
    T = int(cu[-1])
    q = bf16(rng.standard_normal((T + 5, Hq, D)))          # five padding rows
    args = (_t(q), _cache(codes, scales, dtype), _i(bt), _i(cu), _i(ctx), max(new))
    sizes = (T + 5, len(new), Hq, Hkv, D, max(new), max(ctx))
    assert _native.load().vj_paged_prefill_split_workspace_size(*sizes) > 0
    assert _native.load().vj_paged_prefill_quantized_workspace_size(*sizes) > 0 or max(new) > 500
    junk = [torch.full((1 << 22,), float("nan"), device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    del junk
    got = qc.paged_prefill_quantized(*args, max_context_len=max(ctx))
    vals = _values(codes, scales, dtype)
    ref, mag = np.zeros(q.shape), np.zeros(q.shape)
    for s, (n, p) in enumerate(zip(new, prefix)):
        if n:
            k, v = (oq.gather(vals[i], bt[s], n + p) for i in range(2))
            rows = slice(cu[s], cu[s + 1])
            ref[rows], mag[rows] = oq.attend(q[rows].astype(np.float64), k, v, p, 1 / math.sqrt(D))
    _check(got, ref, mag, PREFILL)
    for _ in range(3):
        assert torch.equal(got, qc.paged_prefill_quantized(*args, max_context_len=max(ctx)))


@pytest.mark.parametrize("longest", [2, 0, 800])
@pytest.mark.parametrize("S,new", [(0, 0), (3, 0), (1, 2)])
def test_prefill_rows_behind_the_last_sequence_are_zeroed(S, new, longest):
    """Also where there is no sequence, or none has new tokens; for every way there is
    (the bound on the new tokens chooses)."""
    from vllm_b200.kernels.quantized_cache import QuantizedKVCache, paged_prefill_quantized
    cache = QuantizedKVCache.zeros(8, 16, 2, device="cuda")
    cache.data.view(torch.uint8).fill_(0x38)                   # ones
    q = torch.ones((1000, 16, D), dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, float("nan"))
    paged_prefill_quantized(q, cache, _i(np.zeros((S, 2))), _i(np.arange(S + 1) * new),
                            _i(np.full(S, new)), longest, out=out,
                            max_context_len=16 if longest == 2 else 0)
    assert (out[:S * new] == 1).all() and not out[S * new:].any()


@pytest.mark.parametrize("prefix,new", [(0, (5, 7)), (2000, (5, 7)), (2000, (300, 310)),
                                        (0, (1300, 1240))])
def test_prefill_nan_row_stays_in_its_sequence(prefix, new):
    """A NaN row in the first page of the first sequence, whose block every unused table
    entry stands for."""
    from vllm_b200.kernels.quantized_cache import paged_prefill_quantized
    rng = np.random.default_rng(23)
    ctx = [prefix + n for n in new]
    need = [-(-n // 16) for n in ctx]
    codes, scales = _random_pool(rng, sum(need), 16, 2, "e4m3")
    codes[:, 0, 0], scales[:, 0, :, 0] = 0, 255
    bt = np.full((2, max(need) + 3), -1, np.int32)
    bt[0, :need[0]] = np.arange(need[0])
    bt[1, :need[1]] = need[0] + np.arange(need[1])
    a, T = new[0], sum(new)
    q = _t(bf16(rng.standard_normal((T, 16, D))))
    out = paged_prefill_quantized(q, _cache(codes, scales, "e4m3"), _i(bt), _i([0, a, T]),
                                  _i(ctx), max(new))
    assert torch.isnan(out[:a]).all() and torch.isfinite(out[a:]).all()


# ----------------------------------------------------------------------------- streams, graphs
def test_decode_is_deterministic_on_two_streams_at_once_and_in_graphs():
    from vllm_b200.kernels.quantized_cache import paged_decode_quantized
    rng = np.random.default_rng(21)
    cases = []
    for i, lens in enumerate(([3000, 17, 900], [40, 5000, 1, 0, 260])):
        codes, scales = _random_pool(rng, 340, 16, 4, "int8")
        bt = _tables(rng, lens, 340, 16, 320)
        q = _t(bf16(rng.standard_normal((len(lens), 16, D))))
        cases.append((q, _cache(codes, scales, "int8"), _i(bt), _i(lens)))
    ref = [paged_decode_quantized(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    for _ in range(20):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                outs[i].append(paged_decode_quantized(*c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, ref[i]) for o in outs[i])
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = paged_decode_quantized(*c)
        graphs.append((g, o))
    for _ in range(5):
        for (g, o), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                o.fill_(float("nan"))
                g.replay()
    torch.cuda.synchronize()
    for (_, o), r in zip(graphs, ref):
        assert torch.equal(o, r)


@pytest.mark.parametrize("new,prefix,Hq,Hkv", [
    ((1, 3), (1500, 40), 8, 2),                # direct, split
    ((20, 60, 0), (0, 30, 50), 8, 2),          # direct, one launch
    ((260, 30), (2400, 1000), 32, 8),          # read back, split
    ((900, 1000), (0, 100), 32, 8),            # read back, one launch
])
def test_prefill_in_graphs_and_on_two_streams_at_once(new, prefix, Hq, Hkv):
    """Captured, replayed with other inputs in the same places, and next to itself on
    another stream: the eager call's bits."""
    from vllm_b200.kernels.quantized_cache import QuantizedKVCache, paged_prefill_quantized
    rng = np.random.default_rng(25)
    ctx = [a + b for a, b in zip(new, prefix)]
    need = sum(-(-n // 16) for n in ctx)
    width = -(-max(ctx) // 16)
    T, cu = sum(new), np.concatenate([[0], np.cumsum(new)])

    def inputs(lens):
        codes, scales = _random_pool(rng, need, 16, Hkv, "e4m3")
        return (_t(bf16(rng.standard_normal((T, Hq, D)))), *_cache(codes, scales, "e4m3"),
                _i(_tables(rng, lens, need, 16, width)), _i(lens))

    def call(x, out=None):
        return paged_prefill_quantized(x[0], QuantizedKVCache(x[1], x[2]), x[3], _i(cu) if out is None
                                       else d_cu, x[4], max(new), max_context_len=max(ctx), out=out)

    d_cu = _i(cu)
    sets = [inputs(ctx), inputs([max(n - 7 * i, new[i]) for i, n in enumerate(ctx)])]
    ref = [call(x) for x in sets]
    live = [t.clone() for t in sets[0]]
    out = torch.empty_like(ref[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(live, out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in (1, 0, 1):
        for a, b in zip(live, sets[i]):
            a.copy_(b)
        torch.cuda.synchronize()
        beside = []
        for _ in range(4):
            for k, s in enumerate(streams):
                with torch.cuda.stream(s):
                    beside.append((k, torch.empty_like(out)))
                    call(sets[k], beside[-1][1])
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref[i])
        assert all(torch.equal(o, ref[k]) for k, o in beside)


@pytest.mark.parametrize("op", ["decode", "prefill"])
@pytest.mark.parametrize("lens,Hq,Hkv", [((2900, 17, 600, 0, 1500, 44), 8, 2), ((5000,), 16, 4)])
def test_calls_back_to_back_on_other_inputs(op, lens, Hq, Hkv):
    """Three inputs in turn, eager and from one graph: each call launches before the last
    one is done, and its scratch often is the last one's memory."""
    from vllm_b200.kernels.quantized_cache import (QuantizedKVCache, paged_decode_quantized,
                                                   paged_prefill_quantized)
    rng = np.random.default_rng(26)
    B, need = len(lens), sum(-(-n // 16) for n in lens)
    cu = _i(np.arange(B + 1))
    sets = []
    for _ in range(3):
        codes, scales = _random_pool(rng, need, 16, Hkv, "int8")
        sets.append((_t(bf16(rng.standard_normal((B, Hq, D)))), _cache(codes, scales, "int8"),
                     _i(_tables(rng, lens, need, 16, -(-max(lens) // 16))),
                     _i([max(n, op == "prefill") for n in lens])))

    def call(k):
        q, cache, bt, ln = sets[k]
        if op == "decode":
            return paged_decode_quantized(q, cache, bt, ln)
        return paged_prefill_quantized(q, cache, bt, cu, ln, 1, max_context_len=max(lens))

    ref = []
    for k in range(3):
        ref.append(call(k))
        torch.cuda.synchronize()
    got = [(i % 3, call(i % 3)) for i in range(60)]
    graph, held = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        for i in range(9):
            held.append((i % 3, call(i % 3)))
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref[k]) for k, o in got + held)


def test_a_step_as_it_is_used():
    """Prompts stored, attended to, extended token by token and read back: every step
    against the oracle on the cache's own values, replayed from one captured graph."""
    from vllm_b200.kernels import quantized_cache as qc
    from vllm_b200.kernels.kv_store import rope_table
    rng = np.random.default_rng(22)
    Hq, Hkv, bs, lens, dtype = 8, 2, 16, [30, 16, 5], "e4m3"
    cache = qc.QuantizedKVCache.zeros(16, bs, Hkv, dtype=dtype, device="cuda")
    bt = np.arange(15).reshape(3, 5)[:, ::-1].copy()
    w = _t(np.ones(D))
    table = rope_table(torch.device("cuda", 0))
    cu = np.concatenate([[0], np.cumsum(lens)])
    pos = np.concatenate([np.arange(n) for n in lens])
    seq = np.repeat(np.arange(3), lens)
    x = _t(bf16(rng.standard_normal((cu[-1], Hq + 2 * Hkv, D))))
    slots = bt[seq, pos // bs] * bs + pos % bs
    q = qc.kv_store_quantized(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], cache, _i(slots),
                              _i(pos), w, w, table=table)
    out = qc.paged_prefill_quantized(q, cache, _i(bt), _i(cu), _i(lens), max(lens))

    def reference(q, lens, n):
        vals = _values(cache.data.view(torch.uint8).cpu().numpy(), cache.scales.cpu().numpy(),
                       dtype)
        parts = [oq.attend(q[r], *(oq.gather(vals[i], bt[s], lens[s]) for i in range(2)),
                           lens[s] - (r.stop - r.start), 1 / math.sqrt(D))
                 for s, r in enumerate(n)]
        return [np.concatenate(p) for p in zip(*parts)]

    _check(out, *reference(q.double().cpu().numpy(), lens,
                           [slice(cu[s], cu[s + 1]) for s in range(3)]), PREFILL)
    x1 = torch.empty((3, Hq + 2 * Hkv, D), dtype=torch.bfloat16, device="cuda")
    d_slots, d_pos, d_len = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(3))
    d_bt = _i(bt)
    x1.zero_(), d_slots.fill_(-1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q1 = qc.kv_store_quantized(x1[:, :Hq], x1[:, Hq:Hq + Hkv], x1[:, Hq + Hkv:], cache,
                                   d_slots, d_pos, w, w, table=table)
        o1 = qc.paged_decode_quantized(q1, cache, d_bt, d_len)
        r1 = qc.read_kv_cache(cache, d_bt, d_len)
    for _ in range(4):
        x1.copy_(_t(bf16(rng.standard_normal(x1.shape))))
        d_slots.copy_(_i([bt[s, n // bs] * bs + n % bs for s, n in enumerate(lens)]))
        d_pos.copy_(_i(lens))
        lens = [n + 1 for n in lens]
        d_len.copy_(_i(lens))
        g.replay()
        torch.cuda.synchronize()
        _check(o1, *reference(q1.double().cpu().numpy(), lens, [slice(s, s + 1) for s in range(3)]),
               DECODE)
        vals = _values(cache.data.view(torch.uint8).cpu().numpy(), cache.scales.cpu().numpy(),
                       dtype)
        for s, n in enumerate(lens):
            for i in range(2):
                got = r1[i, s].double().cpu().numpy()
                np.testing.assert_array_equal(got[:n], oq.gather(vals[i], bt[s], n))
                assert not got[n:].any()


def test_calls_keep_nothing_and_count_their_launches():
    """Refused and accepted calls leave no references and no memory behind."""
    import sys

    from vllm_b200 import _native
    from vllm_b200.kernels import quantized_cache as qc
    c = qc.QuantizedKVCache.zeros(4, 16, 2, device="cuda")
    q = torch.ones((3, 4, D), dtype=torch.bfloat16, device="cuda")
    kv = torch.ones((3, 2, D), dtype=torch.bfloat16, device="cuda")
    bt, idx = _i(np.arange(3)[:, None]), _i([0, 17, 34])
    ln, cu, w = _i([1, 2, 3]), _i([0, 1, 2, 3]), _t(np.ones(D))
    out = torch.empty_like(q)

    def calls():
        qc.kv_store_quantized(q, kv, kv, c, idx, ln, w, w)
        qc.paged_decode_quantized(q, c, bt, ln)
        assert qc.paged_decode_quantized(q, c, bt, ln, out=out) is out
        qc.read_kv_cache(c, bt, ln)
        qc.paged_prefill_quantized(q, c, bt, cu)
        for bad in (lambda: qc.paged_decode_quantized(q, c, bt, ln, out=q),
                    lambda: qc.paged_decode_quantized(q[:2], c, bt, ln),
                    lambda: qc.kv_store_quantized(q, kv, kv, c, idx, ln, w)):
            with pytest.raises(ValueError):
                bad()

    calls()                          # tables, identity pages, error word
    torch.cuda.synchronize()
    things = (q, kv, *c, bt, idx, ln, cu, w, out, _native, torch.device("cuda", 0))
    refs, mem = [sys.getrefcount(x) for x in things], torch.cuda.memory_allocated()
    before = _native.launch_count
    for _ in range(20):
        calls()
    torch.cuda.synchronize()
    assert _native.launch_count - before == 20 * (1 + 2 + 2 + 1 + 1)
    assert torch.cuda.memory_allocated() == mem
    assert [sys.getrefcount(x) for x in things] == refs


# ----------------------------------------------------------------------------- refusals
def test_wrapper_refusals():
    from vllm_b200.kernels import quantized_cache as qc
    c = qc.QuantizedKVCache.zeros(4, 16, 2, device="cuda")
    q = torch.zeros((3, 4, D), dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros((3, 2, D), dtype=torch.bfloat16, device="cuda")
    bt, ln, w = _i(np.zeros((3, 4))), _i([1, 1, 1]), _t(np.ones(D))
    bad = [
        (lambda: qc.paged_decode_quantized(q.float(), c, bt, ln), "dtype of `q`"),
        (lambda: qc.paged_decode_quantized(q[:, :3], c, bt, ln), "contiguous"),
        (lambda: qc.paged_decode_quantized(q[:, :3].contiguous(), c, bt, ln), "do not match"),
        (lambda: qc.paged_decode_quantized(q, c, bt[:2], ln), "one row per sequence"),
        (lambda: qc.paged_decode_quantized(q, c, bt, ln[:2]), "context_lens"),
        (lambda: qc.paged_decode_quantized(q, c, bt.long(), ln), "block_tables"),
        (lambda: qc.paged_decode_quantized(q, c, bt.t().contiguous().t(), ln), "contiguous"),
        (lambda: qc.paged_decode_quantized(q, c, bt[:1].expand(3, 4), ln), "overlap"),
        (lambda: qc.paged_decode_quantized(q, c, bt, ln, out=q.float()), "out"),
        (lambda: qc.paged_decode_quantized(q, c, bt, ln, out=q), "overlap"),
        (lambda: qc.paged_decode_quantized(q, c, bt, ln, workspace=torch.zeros(
            1, dtype=torch.uint8, device="cuda")), "workspace"),
        (lambda: qc.paged_decode_quantized(q, qc.QuantizedKVCache(c.data, c.scales[:, :3]), bt,
                                           ln), "scales"),
        (lambda: qc.paged_decode_quantized(q, qc.QuantizedKVCache(c.data.to(torch.bfloat16),
                                                                  c.scales), bt, ln), "float8"),
        (lambda: qc.paged_decode_quantized(q, c, bt.cpu(), ln), "CUDA"),
        (lambda: qc.read_kv_cache(c, bt, ln, -1), "negative"),
        (lambda: qc.read_kv_cache(c, bt, ln, 8, out=q), "out"),
        (lambda: qc.kv_store_quantized(q, kv, kv[:2], c, ln, ln, w, w), "same shape"),
        (lambda: qc.kv_store_quantized(q, kv, kv, c, ln, None, w, w), "positions"),
        (lambda: qc.kv_store_quantized(q, kv, kv, c, ln, ln), "norm"),
        (lambda: qc.kv_store_quantized(q, kv, kv, c, ln[:2], ln, w, w), "slot_mapping"),
        (lambda: qc.kv_store_quantized(q, kv, kv, c, ln, ln, w.float(), w), "q_norm_weight"),
        (lambda: qc.kv_store_quantized(q, kv[:, :1], kv[:, :1], c, ln, ln, w, w), "do not match"),
        (lambda: qc.kv_store_quantized(q, kv, kv, c, ln, ln, w, w, q_out=q[:, :2]), "q_out"),
        (lambda: qc.kv_store_quantized(q, kv[:1].expand(3, 2, D), kv, c, ln, ln, w, w), "overlap"),
        (lambda: qc.kv_store_quantized(q, kv, kv[:1].expand(3, 2, D), c, ln, ln, w, w), "overlap"),
        (lambda: qc.kv_store_quantized(q[:1].expand(3, 4, D), kv, kv, c, ln, ln, w, w), "overlap"),
        (lambda: qc.paged_decode_quantized(q[:, :0].contiguous(), c, bt, ln), "size"),
        (lambda: qc.paged_prefill_quantized(q[:, :0].contiguous(), c, bt, _i([0, 1, 2, 3]), ln), "size"),
        (lambda: qc.paged_prefill_quantized(q, c, bt, ln, ln), "one row per sequence"),
        (lambda: qc.paged_prefill_quantized(q, c, bt[:2], ln, ln[:2], scale=0.0), "positive"),
        (lambda: qc.paged_prefill_quantized(q, c, bt[:2], ln, ln[:2], max_context_len=-4),
         "negative"),
    ]
    for i, (call, msg) in enumerate(bad):
        with pytest.raises(ValueError, match=msg):
            call()
            pytest.fail(f"refusal {i} did not happen")
