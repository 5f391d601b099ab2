"""Calls of the quantised KV cache at the edges of what they accept, on the GPU
against 64-bit NumPy (oracle/quantized.py). Tolerances as derived in
test_quantized_cache_gpu.py: a bf16 result is off by half a step, 2^-8 |r|, the
weights of decode by 2^-11 + 2^-12 and of prefill by 2^-8 + 2^-11 of each."""
import math

import numpy as np
import pytest
import torch

from oracle import quantized as oq
from oracle.bf16 import bf16

pytestmark = pytest.mark.gpu

D = 128
TORCH = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
DECODE = 2.0 ** -11 + 2.0 ** -12
PREFILL = 2.0 ** -8 + 2.0 ** -11


def _t(x, dtype=torch.bfloat16):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def _i(x):
    return torch.tensor(np.asarray(x, np.int32), device="cuda")


def _check(got, ref, mag, weight):
    got = got.double().cpu().numpy()
    err = np.abs(got - ref)
    tol = 2.0 ** -8 * np.abs(ref) + weight * mag + 1e-30
    assert np.isfinite(got).all() and (err <= tol).all(), \
        f"worst {np.max(err / tol):.3f} of the tolerance"


class _Prompts:
    """A batch of new tokens after cached prefixes, with five padding rows of q."""

    def __init__(self, Hq, Hkv, new, prefix, dtype="e4m3", bs=16, seed=0):
        from vllm_b200.kernels.quantized_cache import QuantizedKVCache
        rng = np.random.default_rng(seed)
        self.new, self.prefix = new, prefix
        self.ctx = [a + b for a, b in zip(new, prefix)]
        need = [-(-n // bs) for n in self.ctx]
        nb = sum(need) + 2
        self.codes, _ = oq.quantise_rows(rng.standard_normal((2, nb, bs, Hkv, D)), dtype)
        self.scales = rng.integers(118, 123, (2, nb, Hkv, bs)).astype(np.uint8)
        perm, at = rng.permutation(nb), 0
        self.bt = np.full((len(new), max(need) + 1), -1, np.int32)
        for s, n in enumerate(need):
            self.bt[s, :n] = perm[at:at + n]
            at += n
        self.cu = np.concatenate([[0], np.cumsum(new)])
        self.q_np = bf16(rng.standard_normal((int(self.cu[-1]) + 5, Hq, D)))
        self.dtype = dtype
        self.q = _t(self.q_np)
        self.args = (QuantizedKVCache(_t(self.codes, torch.uint8).view(TORCH[dtype]),
                                      _t(self.scales, torch.uint8)),
                     _i(self.bt), _i(self.cu), _i(self.ctx), max(new))

    def call(self, q=None, out=None, **kw):
        from vllm_b200.kernels.quantized_cache import paged_prefill_quantized
        kw.setdefault("max_context_len", max(self.ctx))
        return paged_prefill_quantized(self.q if q is None else q, *self.args, out=out, **kw)

    def reference(self):
        vals = [oq.dequantise(self.codes[i], self.scales[i], self.dtype) for i in range(2)]
        ref, mag = np.zeros(self.q_np.shape), np.zeros(self.q_np.shape)
        for s, (n, p) in enumerate(zip(self.new, self.prefix)):
            if n:
                k, v = (oq.gather(vals[i], self.bt[s], n + p) for i in range(2))
                rows = slice(self.cu[s], self.cu[s + 1])
                ref[rows], mag[rows] = oq.attend(self.q_np[rows].astype(np.float64), k, v, p,
                                                 1 / math.sqrt(D))
        return ref, mag


@pytest.mark.parametrize("Hq,Hkv,new,prefix,groups,launches", [
    (8, 2, (20, 60, 0), (0, 30, 50), 1, 1),              # from the pages
    (8, 2, (1, 3), (1500, 40), 1, 2),                    # and their keys split
    (32, 8, (900, 1000), (0, 100), 1, 2),                # read back first
    (32, 8, (256,), (2500,), 1, 3),                      # and their keys split
    (32, 8, (900, 1000, 700), (0, 100, 5), 3, 6),        # read back in groups
    (32, 8, (300, 0, 280), (1400, 30, 1100), 3, 9),      # and their keys split
])
def test_prefill_in_the_queries_place(Hq, Hkv, new, prefix, groups, launches, monkeypatch):
    """out may be q itself, however the call is carried out."""
    from vllm_b200 import _native
    from vllm_b200.kernels import quantized_cache as qc
    if groups > 1:
        monkeypatch.setattr(qc, "PREFILL_SCRATCH_ROWS", 1)
    case = _Prompts(Hq, Hkv, new, prefix)
    before = _native.launch_count
    ref = case.call()
    assert _native.launch_count - before == launches
    q = case.q.clone()
    assert case.call(q, out=q) is q
    assert torch.equal(q, ref)
    _check(q, *case.reference(), PREFILL)



def test_prefill_groups_in_the_queries_place_in_a_graph(monkeypatch):
    """Captured with groups of one sequence, replayed on other queries next to eager calls on
    another stream."""
    from vllm_b200.kernels import quantized_cache as qc
    monkeypatch.setattr(qc, "PREFILL_SCRATCH_ROWS", 1)
    case = _Prompts(32, 8, (300, 0, 280), (1400, 30, 1100))
    queries = [case.q, _t(bf16(np.random.default_rng(3).standard_normal(case.q_np.shape)))]
    refs = [case.call(q) for q in queries]
    live, graph, side = queries[0].clone(), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        case.call(live, out=live)
    for i in (1, 0, 1):
        live.copy_(queries[i])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = case.call(queries[1 - i])
        torch.cuda.synchronize()
        assert torch.equal(live, refs[i]) and torch.equal(beside, refs[1 - i])


@pytest.mark.parametrize("Hq,Hkv,new,prefix", [(8, 2, (20, 60), (0, 30)),
                                               (32, 8, (900, 1000), (0, 100))])
def test_prefill_refuses_an_output_that_lies_across_the_queries(Hq, Hkv, new, prefix):
    case = _Prompts(Hq, Hkv, new, prefix)
    T = case.q.shape[0]
    both = torch.cat([case.q, case.q[:1]])
    kept = both.clone()
    for q, out in ((both[:T], both[1:]), (both[1:], both[:T])):
        with pytest.raises(ValueError, match="overlap"):
            case.call(q, out=out)
    torch.cuda.synchronize()
    assert torch.equal(both, kept)


@pytest.mark.parametrize("most,sizes", [(4, (3, 4)), (4, (3, 3)), (2, (1, 2, 2, 2)), (1, (1,) * 6)])
def test_prefill_in_uneven_groups_with_split_keys(most, sizes, monkeypatch):
    """Groups of sequences read back one after another, where some are split further over
    their keys than others: a group's parts begin at its own first token."""
    from vllm_b200 import _native
    from vllm_b200.kernels import quantized_cache as qc
    new = (130, 0, 140, 129, 1, 140, 133)[:sum(sizes)]
    prefix = (2200, 30, 1100, 2000, 1500, 1024, 2290)[:sum(sizes)]
    case = _Prompts(32, 8, new, prefix, "int8", 32, seed=1)
    padded = -(-max(case.ctx) // 128) * 128                  # rows that a sequence takes
    monkeypatch.setattr(qc, "PREFILL_SCRATCH_ROWS", most * padded * 8)
    before = _native.launch_count
    out = torch.full_like(case.q, float("nan"))
    case.call(out=out)
    parts = [_native.load().vj_paged_prefill_split_workspace_size(
        case.q.shape[0], n, 32, 8, D, max(new), max(case.ctx)) > 0 for n in sizes]
    assert _native.launch_count - before == sum(2 + p for p in parts) and any(parts)
    _check(out, *case.reference(), PREFILL)


def test_prefill_scratch_of_many_small_groups_is_bounded(monkeypatch):
    """A group's share of the scratch does not grow with the batch: 40 sequences of 64 new
    tokens one after another, contexts of up to 8192."""
    from vllm_b200.kernels import quantized_cache as qc
    S, n, bound = 40, 64, 8192
    cache = qc.QuantizedKVCache.zeros(S * 4, 16, 8, device="cuda")
    cache.data.view(torch.uint8).fill_(0x38)                   # ones
    q = torch.randn((S * n, 64, D), device="cuda").to(torch.bfloat16)
    bt = torch.zeros((S, bound // 16), dtype=torch.int32, device="cuda")
    out, cu, ln = torch.empty_like(q), _i(np.arange(S + 1) * n), _i(np.full(S, n))
    monkeypatch.setattr(qc, "PREFILL_SCRATCH_ROWS", 1)
    qc.paged_prefill_quantized(q, cache, bt, cu, ln, n, out=out, max_context_len=bound)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    qc.paged_prefill_quantized(q, cache, bt, cu, ln, n, out=out, max_context_len=bound)
    torch.cuda.synchronize()
    took = torch.cuda.max_memory_allocated() - held
    # K and V of one sequence, and the parts' rows of one (148 CTAs of 256, 130 words each)
    assert took <= 2 * bound * 8 * D * 2 + 148 * 256 * 130 * 4 + (2 << 20)
    scale = cache.scales[0, 0, 0, 0].float()                  # every row of V is this one
    assert torch.equal(out, torch.full_like(out, float(torch.exp2(scale - 127))))


# ----------------------------------------------------------------------------- store
@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("eps", [1e-6, 0.0, 1e-38, 1e-12, 1e30, -1e-8])
def test_stored_k_rows_of_every_magnitude_are_correctly_rounded(dtype, eps):
    """Normalised and turned rows from 2^-130 to 2^125, whose squares leave the range of
    32 bits at both ends, and rows of zeros, infinities and NaN."""
    from vllm_b200.kernels.kv_store import rope_table
    from vllm_b200.kernels.quantized_cache import QuantizedKVCache, kv_store_quantized
    rng = np.random.default_rng(31)
    T, Hkv, bs = 256, 3, 16
    with np.errstate(over="ignore"):
        kv = bf16(rng.standard_normal((T, 2 * Hkv, D)) * np.exp2(np.arange(T) - 130.0)[:, None, None])
    kv[5] = 0
    kv[200, :, 3] = np.inf
    kv[201, :, 100] = np.nan
    kv[202, 0] = 0
    kv[202, 0, 64] = bf16(np.float32(1e-40))
    kv[203] = 0
    kv[203, :, 7] = bf16(np.float32(3e38))
    w = bf16(1 + 0.3 * rng.standard_normal(D))
    pos = rng.integers(0, 4096, T)
    slots = rng.permutation(T)
    table = rope_table(torch.device("cuda", 0), 1e6, 4096)
    cache = QuantizedKVCache.zeros(T // bs, bs, Hkv, dtype=dtype, device="cuda")
    d = _t(kv)
    kv_store_quantized(None, d[:, :Hkv], d[:, Hkv:], cache, _i(slots), _i(pos), None, _t(w), eps=eps,
                       table=table)
    cs = table.view(torch.bfloat16).double().cpu().numpy().reshape(-1, D // 2, 2)[pos]
    x = kv.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        rows = oq.norm_rope(x[:, :Hkv], w.astype(np.float64), cs, eps), x[:, Hkv:]
        new = [oq.quantise_rows(y, dtype) for y in rows]
    data, scales = cache.data.view(torch.uint8).cpu().numpy(), cache.scales.cpu().numpy()
    for i in range(2):
        got = data[i].reshape(T, Hkv, D)[slots], scales[i].transpose(0, 2, 1).reshape(T, Hkv)[slots]
        np.testing.assert_array_equal(got[1], new[i][1], err_msg="scales of " + "kv"[i])
        np.testing.assert_array_equal(got[0], new[i][0], err_msg="elements of " + "kv"[i])


@pytest.mark.parametrize("T", [1, 33])
def test_store_in_place_and_next_to_its_inputs(T):
    """q_out as q's own columns of one projection's output, and as columns of the same rows
    that nothing else takes."""
    from vllm_b200.kernels.quantized_cache import QuantizedKVCache, kv_store_quantized
    rng = np.random.default_rng(33)
    x = _t(bf16(rng.standard_normal((T, 4 + 2 + 2 + 4, D))))
    w, pos, slots = _t(np.ones(D)), _i(np.arange(T)), _i(np.arange(T) + 5)

    def call(y, out):
        cache = QuantizedKVCache.zeros(4, 16, 2, device="cuda")
        q = kv_store_quantized(y[:, :4], y[:, 4:6], y[:, 6:8], cache, slots, pos, w, w, q_out=out)
        return q, cache.data.view(torch.uint8), cache.scales

    ref = call(x, None)
    for columns in (slice(0, 4), slice(8, 12)):
        y = x.clone()
        for a, b in zip(call(y, y[:, columns]), ref):
            assert torch.equal(a, b)
        keep = [i for i in range(12) if i not in range(*columns.indices(12))]
        assert torch.equal(y[:, keep], x[:, keep])
    if T > 1:
        y = x.clone()
        for columns in (slice(1, 5), slice(3, 7), slice(5, 9)):
            with pytest.raises(ValueError, match="overlap"):
                call(y, y[:, columns])
        torch.cuda.synchronize()
        assert torch.equal(y, x)


# ----------------------------------------------------------------------------- decode
@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("n,Hq", [(40, 8), (40, 32), (3000, 2), (3000, 32)])
def test_rows_that_nothing_stored_count_as_zeros(n, Hq, dtype):
    """Rows of a fresh pool inside a context, next to values of 1e-6: their scales must not
    outweigh the others'. Whole pages of them too, and a row of NaN in another sequence."""
    from vllm_b200.kernels.quantized_cache import (QuantizedKVCache, kv_store_quantized,
                                                   paged_decode_quantized)
    rng = np.random.default_rng(32)
    nb = -(-n // 16) + 1
    cache = QuantizedKVCache.zeros(nb + 1, 16, 2, dtype=dtype, device="cuda")
    cache.scales[:, nb] = 255
    slots = np.arange(n)
    missing = [3, 20, n - 1] + list(range(0 if n < 99 else 700, 0 if n < 99 else 760))
    slots[missing] = -1
    k, v = bf16(rng.standard_normal((n, 2, D))), bf16(1e-6 * rng.standard_normal((n, 2, D)))
    kv_store_quantized(None, _t(k), _t(v), cache, _i(slots), norm=False, rope=False)
    q = bf16(rng.standard_normal((1, Hq, D)))
    bt = np.full((2, nb), nb)
    bt[0] = np.arange(nb)
    out = paged_decode_quantized(_t(np.concatenate([q, q])), cache, _i(bt), _i([n, 5]))
    assert torch.isnan(out[1]).all()
    out = out[:1]
    codes, scales = cache.data.view(torch.uint8).cpu().numpy(), cache.scales.cpu().numpy()
    vals = [oq.gather(oq.dequantise(codes[i], scales[i], dtype), np.arange(nb), n) for i in range(2)]
    assert not vals[1][missing].any() and vals[1][4].any()
    _check(out, *oq.attend(q.astype(np.float64), *vals, n - 1, 1 / math.sqrt(D)), DECODE)
