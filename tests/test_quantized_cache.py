"""The quantised KV cache without a GPU: the oracle's number formats, and what
the C entries refuse before they touch a device."""
import numpy as np
import pytest
import torch

from oracle import quantized as oq


def test_e4m3_values_are_torchs():
    codes = np.arange(256, dtype=np.uint8)
    ref = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(oq.element_values(codes, "e4m3"), ref)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_quantise_rows_properties(dtype):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 128)) * np.exp(rng.uniform(-60, 60, (200, 1)))
    x[0] = 0
    x[1, 5] = np.inf
    x[2, 7] = np.nan
    x[3] = 0
    x[3, 0] = oq.LARGEST[dtype]              # exactly the largest element: scale 1
    x[4] = 0
    x[4, 0] = np.nextafter(oq.LARGEST[dtype], 1e9)
    codes, b = oq.quantise_rows(x, dtype)
    assert b[0] == 1 and b[1] == b[2] == 255 and b[3] == 127 and b[4] == 128
    assert not codes[:3].any()
    y = oq.element_values(codes, dtype) * np.exp2(b.astype(float) - 127)[:, None]
    ok = np.isfinite(x).all(-1)
    # half a step: relative 2^-4 for e4m3 (absolute 2^-10 of the scale below its normal
    # numbers), half a unit of the scale for int8
    unit = np.exp2(b.astype(float) - 127)[:, None]
    tol = np.maximum(np.abs(x) * 2.0 ** -4, unit * 2.0 ** -10) if dtype == "e4m3" else unit / 2
    assert (np.abs(y - x)[ok] <= tol[ok]).all()
    # the scale is the smallest: half of it would not hold the row
    big = np.abs(x[ok]).max(-1)
    big, bb = big[big > 0], b[ok][np.abs(x[ok]).max(-1) > 0].astype(float)
    assert (big <= oq.LARGEST[dtype] * np.exp2(bb - 127)).all()
    assert ((big > oq.LARGEST[dtype] * np.exp2(bb - 128)) | (bb == 1)).all()


def test_products_are_bf16_numbers():
    for dtype in ("e4m3", "int8"):
        v = oq.element_values(np.arange(256, dtype=np.uint8), dtype)
        v = v[np.isfinite(v)]
        for e in (-100, -8, 0, 100):
            x = torch.from_numpy(v * 2.0 ** e)
            assert torch.equal(x.to(torch.bfloat16).double(), x)


def _store(lib, **kw):
    a = dict(q=16, k=16, v=16, qw=16, kw=16, pos=16, slots=16, qo=16, kc=16, vc=16, ks=16, vs=16,
             dt=1, T=4, Hq=8, Hkv=2, D=128, nb=4, bs=16, sb=4096, st=256, sh=128, cb=32, ch=16,
             qrs=0, krs=0, vrs=0, qors=0, tab=None, tl=0, eps=1e-6, th=1e6, fl=3, err=None, stream=None)
    a.update(kw)
    return lib.vj_kv_store_quantized(*a.values())


def _decode(lib, **kw):
    a = dict(q=16, kc=16, vc=16, ks=16, vs=16, dt=1, bt=16, lens=16, out=16, B=2, Hq=8, Hkv=2,
             D=128, nb=4, bs=16, w=4, bts=4, sb=4096, st=256, sh=128, cb=32, ch=16, scale=0.1,
             ws=256, wsb=1 << 30, err=None, stream=None)
    a.update(kw)
    return lib.vj_paged_decode_quantized(*a.values())


def _read(lib, **kw):
    a = dict(kc=16, vc=16, ks=16, vs=16, dt=1, bt=16, lens=16, ko=16, vo=16, B=2, L=32, z=0,
             Hkv=2, D=128, nb=4, bs=16, w=4, bts=4, sb=4096, st=256, sh=128, cb=32, ch=16,
             stream=None)
    a.update(kw)
    return lib.vj_kv_read_quantized(*a.values())


def _split(lib, **kw):
    a = dict(q=16, k=16, v=16, bt=16, cu=16, ctx=16, out=16, T=4, S=1, Hq=8, Hkv=2, D=128, nb=200,
             bs=16, w=200, bts=200, sb=4096, st=256, sh=128, mq=4, mc=3200, scale=0.1, ws=None,
             wsb=0, err=16, stream=None)
    a.update(kw)
    return lib.vj_paged_prefill_split(*a.values())


def _prefill(lib, **kw):
    a = dict(q=16, kc=16, vc=16, ks=16, vs=16, dt=1, bt=16, cu=16, ctx=16, out=16, T=4, S=1, Hq=8,
             Hkv=2, D=128, nb=200, bs=16, w=200, bts=200, sb=4096, st=256, sh=128, cb=32, ch=16,
             mq=4, mc=3200, scale=0.1, ws=None, wsb=0, err=None, stream=None)
    a.update(kw)
    return lib.vj_paged_prefill_quantized(*a.values())


COMMON = [
    (dict(D=64), "UNSUPPORTED", b"head_dim"),
    (dict(dt=0), "INVALID_ARGUMENT", b"cache_dtype"),
    (dict(dt=3), "INVALID_ARGUMENT", b"cache_dtype"),
    (dict(bs=8), "UNSUPPORTED", b"multiple of 16"),
    (dict(bs=0), "INVALID_ARGUMENT", b"size"),
    (dict(nb=0), "INVALID_ARGUMENT", b"size"),
    (dict(Hkv=0), "INVALID_ARGUMENT", b"size"),
    (dict(nb=1 << 27), "UNSUPPORTED", b"2^31"),
    (dict(kc=None), "INVALID_ARGUMENT", b"null"),
    (dict(vs=None), "INVALID_ARGUMENT", b"null"),
    (dict(kc=24), "INVALID_ARGUMENT", b"multiples of 16"),
    (dict(ks=8), "INVALID_ARGUMENT", b"multiples of 16"),
    (dict(sh=120), "INVALID_ARGUMENT", b"multiples of 16"),
    (dict(ch=8), "INVALID_ARGUMENT", b"multiples of 16"),
]


@pytest.mark.parametrize("entry", [_store, _decode, _read, _prefill])
@pytest.mark.parametrize("kw,status,msg", COMMON)
def test_refusals_of_every_entry(entry, kw, status, msg):
    from vllm_b200 import _native
    lib = _native.load()
    assert entry(lib, **kw) == getattr(_native, "VJ_ERR_" + status)
    assert msg in lib.vj_get_last_error()


@pytest.mark.parametrize("entry,kw,status,msg", [
    (_store, dict(T=-1), "INVALID_ARGUMENT", b"negative"),
    (_store, dict(Hq=-1), "INVALID_ARGUMENT", b"negative"),
    (_store, dict(Hq=5000), "UNSUPPORTED", b"4096"),
    (_store, dict(fl=4), "INVALID_ARGUMENT", b"flags"),
    (_store, dict(fl=8 | 3), "INVALID_ARGUMENT", b"flags"),
    (_store, dict(slots=None), "INVALID_ARGUMENT", b"null"),
    (_store, dict(q=None), "INVALID_ARGUMENT", b"null"),
    (_store, dict(qo=None), "INVALID_ARGUMENT", b"null"),
    (_store, dict(qw=None), "INVALID_ARGUMENT", b"weights"),
    (_store, dict(kw=None), "INVALID_ARGUMENT", b"weights"),
    (_store, dict(pos=None), "INVALID_ARGUMENT", b"positions"),
    (_store, dict(tab=8, tl=4), "INVALID_ARGUMENT", b"rope_table"),
    (_store, dict(tab=None, tl=4), "INVALID_ARGUMENT", b"rope_table"),
    (_store, dict(tl=-1), "INVALID_ARGUMENT", b"negative"),
    (_store, dict(k=24), "INVALID_ARGUMENT", b"16-byte"),
    (_store, dict(krs=260), "INVALID_ARGUMENT", b"16-byte"),
    (_decode, dict(Hq=7), "INVALID_ARGUMENT", b"divisible"),
    (_decode, dict(Hq=0), "INVALID_ARGUMENT", b"size"),
    (_decode, dict(Hq=34), "UNSUPPORTED", b"16 query heads"),
    (_decode, dict(B=-1), "INVALID_ARGUMENT", b"size"),
    (_decode, dict(bts=3), "INVALID_ARGUMENT", b"size"),
    (_decode, dict(Hkv=2048, Hq=2048, st=128 * 2048, sb=16 * 128 * 2048), "UNSUPPORTED",
     b"KV heads"),
    (_decode, dict(sb=8192), "UNSUPPORTED", b"evenly"),
    (_decode, dict(q=None), "INVALID_ARGUMENT", b"null"),
    (_decode, dict(bt=None), "INVALID_ARGUMENT", b"null"),
    (_decode, dict(q=8), "INVALID_ARGUMENT", b"aligned"),
    (_decode, dict(ws=None), "WORKSPACE", b"workspace"),
    (_decode, dict(ws=8), "WORKSPACE", b"workspace"),
    (_decode, dict(wsb=16), "WORKSPACE", b"workspace"),
    (_decode, dict(), "INVALID_ARGUMENT", b"same memory"),
    (_decode, dict(vc=32, vs=16), "INVALID_ARGUMENT", b"same memory"),
    (_decode, dict(vc=16 + (1 << 40), vs=32), "UNSUPPORTED", b"2^40"),
    (_decode, dict(vc=32, vs=32), "INVALID_ARGUMENT", b"overlap"),
    (_decode, dict(vc=32, vs=32, q=16 + 2 * 8 * 128 * 2 - 16), "INVALID_ARGUMENT", b"overlap"),
    (_decode, dict(vc=32, vs=32, out=16 + 2 * 8 * 128 * 2 - 16), "INVALID_ARGUMENT", b"overlap"),
    (_read, dict(B=-1), "INVALID_ARGUMENT", b"size"),
    (_read, dict(L=-1), "INVALID_ARGUMENT", b"size"),
    (_read, dict(z=-1), "INVALID_ARGUMENT", b"size"),
    (_read, dict(B=70000), "UNSUPPORTED", b"65535"),
    (_read, dict(Hkv=5000, st=128 * 5000, sb=16 * 128 * 5000), "UNSUPPORTED", b"4096"),
    (_read, dict(ko=None), "INVALID_ARGUMENT", b"null"),
    (_read, dict(vo=8), "INVALID_ARGUMENT", b"aligned"),
    (_prefill, dict(scale=0.0), "INVALID_ARGUMENT", b"positive"),
    (_prefill, dict(scale=-1.0), "INVALID_ARGUMENT", b"positive"),
    (_prefill, dict(scale=float("nan")), "INVALID_ARGUMENT", b"positive"),
    (_prefill, dict(mc=-1), "INVALID_ARGUMENT", b"size"),
    (_prefill, dict(S=-1), "INVALID_ARGUMENT", b"size"),
    (_prefill, dict(bts=3), "INVALID_ARGUMENT", b"size"),
    (_prefill, dict(Hq=7), "INVALID_ARGUMENT", b"divisible"),
    (_prefill, dict(Hq=12), "UNSUPPORTED", b"divide 128"),
    (_prefill, dict(q=None), "INVALID_ARGUMENT", b"null"),
    (_prefill, dict(bt=None), "INVALID_ARGUMENT", b"null"),
    (_prefill, dict(ctx=None), "INVALID_ARGUMENT", b"null"),
    (_prefill, dict(q=8), "INVALID_ARGUMENT", b"aligned"),
    (_prefill, dict(), "WORKSPACE", b"workspace"),
    (_prefill, dict(ws=8, wsb=1 << 30), "WORKSPACE", b"workspace"),
    (_prefill, dict(S=70000), "UNSUPPORTED", b"grid"),
    (_split, dict(scale=0.0), "INVALID_ARGUMENT", b"positive"),
    (_split, dict(scale=-1.0), "INVALID_ARGUMENT", b"positive"),
    (_split, dict(scale=float("nan")), "INVALID_ARGUMENT", b"positive"),
    (_split, dict(scale=float("inf")), "INVALID_ARGUMENT", b"positive"),
    (_split, dict(mc=-1), "INVALID_ARGUMENT", b"size"),
    (_split, dict(Hq=7), "INVALID_ARGUMENT", b"divisible"),
    (_split, dict(Hq=12), "UNSUPPORTED", b"divide 128"),
    (_split, dict(D=64), "UNSUPPORTED", b"head_dim"),
    (_split, dict(q=None), "INVALID_ARGUMENT", b"null"),
    (_split, dict(bt=None, S=1 << 16, bts=1 << 16), "UNSUPPORTED", b"2^31"),
    (_split, dict(), "WORKSPACE", b"workspace"),
    (_split, dict(ws=8, wsb=1 << 30), "WORKSPACE", b"workspace"),
])
def test_refusals_of_one_entry(entry, kw, status, msg):
    from vllm_b200 import _native
    lib = _native.load()
    assert entry(lib, **kw) == getattr(_native, "VJ_ERR_" + status)
    assert msg in lib.vj_get_last_error()


def test_empty_calls_need_no_memory():
    from vllm_b200 import _native
    lib = _native.load()
    none = dict(kc=None, vc=None, ks=None, vs=None)
    assert _store(lib, T=0, **none) == 0
    assert _decode(lib, B=0, **none) == 0
    assert _read(lib, B=0, **none) == 0
    assert _prefill(lib, T=0, **none) == 0
    size = lib.vj_paged_decode_quantized_workspace_size
    assert size(4, 8, 2, 64, 4, 16) == size(4, 8, 2, 128, 4, 0) == size(4, 0, 2, 128, 4, 16) == 0
    assert 16 <= size(4, 8, 2, 128, 4, 16) <= size(400, 8, 2, 128, 4000, 16)


def test_wrapper_refuses_cpu_tensors_and_unknown_types():
    from vllm_b200.kernels import quantized_cache as qc
    with pytest.raises(ValueError, match="e4m3"):
        qc.QuantizedKVCache.zeros(4, 16, 2, dtype="fp4")
    cache = qc.QuantizedKVCache.zeros(4, 16, 2, dtype="int8")
    assert cache.data.shape == (2, 4, 16, 2, 128) and cache.scales.shape == (2, 4, 2, 16)
    with pytest.raises(ValueError, match="CUDA"):
        qc.paged_decode_quantized(torch.zeros(1, 4, 128, dtype=torch.bfloat16), cache,
                                  torch.zeros(1, 4, dtype=torch.int32),
                                  torch.ones(1, dtype=torch.int32))


def test_arguments_of_other_types():
    from vllm_b200.kernels import quantized_cache as qc
    q, bt = torch.zeros(1, 4, 128, dtype=torch.bfloat16), torch.zeros(1, 4, dtype=torch.int32)
    cache = qc.QuantizedKVCache.zeros(4, 16, 2)
    for call, msg in ((lambda: qc.paged_decode_quantized(q, cache, bt, [1]), "context_lens"),
                      (lambda: qc.paged_decode_quantized(q, cache.data, bt, bt[0]), "cache"),
                      (lambda: qc.paged_decode_quantized(q, (None, None), bt, bt[0]), "cache.data"),
                      (lambda: qc.paged_decode_quantized(None, cache, bt, bt[0]), "`q`"),
                      (lambda: qc.paged_decode_quantized(q, cache, bt, bt[0], out=1), "out"),
                      (lambda: qc.kv_store_quantized(None, None, q, cache, bt[0]), "`k`"),
                      (lambda: qc.read_kv_cache(cache, None, bt[0]), "block_tables"),
                      (lambda: qc.paged_prefill_quantized(q, cache, bt, "x"), "cu_seqlens_q")):
        with pytest.raises(TypeError, match=msg):
            call()


def test_config_refusals():
    from vllm_b200 import Config
    from vllm_b200.src.model_runner import check_kv_cache_dtype
    base = dict(model="tiny", max_num_batched_tokens=64, max_num_seqs=2, num_blocks=8)
    check_kv_cache_dtype(Config(**base, block_size=8))
    check_kv_cache_dtype(Config(**base, block_size=16, compat=False, kv_cache_dtype="int8"))
    for kw, msg in ((dict(block_size=16, compat=False, kv_cache_dtype="fp4"), "kv_cache_dtype"),
                    (dict(block_size=16, kv_cache_dtype="e4m3"), "compat"),
                    (dict(block_size=8, compat=False, kv_cache_dtype="e4m3"), "multiple of 16")):
        with pytest.raises(ValueError, match=msg):
            check_kv_cache_dtype(Config(**base, **kw))
