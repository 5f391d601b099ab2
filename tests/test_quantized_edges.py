"""What the quantised cache's calls refuse or work out on the host, without a GPU."""
import pytest


def _prefill(lib, **kw):
    a = dict(q=16, kc=16, vc=16, ks=16, vs=16, dt=1, bt=16, cu=16, ctx=16, out=16, T=4, S=1, Hq=8,
             Hkv=2, D=128, nb=200, bs=16, w=200, bts=200, sb=4096, st=256, sh=128, cb=32, ch=16,
             mq=4, mc=3200, scale=0.1, ws=None, wsb=0, err=None, stream=None)
    return lib.vj_paged_prefill_quantized(*{**a, **kw}.values())


def _split(entry):
    def call(lib, **kw):
        a = dict(q=16, k=16, v=16, bt=16, cu=16, ctx=16, out=16, T=4, S=1, Hq=8, Hkv=2, D=128,
                 nb=200, bs=16, w=200, bts=200, sb=4096, st=256, sh=128, mq=4, mc=3200, scale=0.1,
                 ws=None, wsb=0, err=16, stream=None)
        return getattr(lib, entry)(*{**a, **kw}.values())
    return call


PREFILLS = [_prefill, _split("vj_paged_prefill_split"), _split("vj_paged_prefill_split_part")]
ROWS = 4 * 8 * 128 * 2        # bytes of q, and of out


def _bf16_prefill(lib, **kw):
    a = dict(q=16, k=16, v=16, bt=16, cu=16, ctx=16, out=16, T=4, S=1, Hq=8, Hkv=2, D=128, nb=200,
             bs=16, w=200, bts=200, sb=4096, st=256, sh=128, mq=4, scale=0.1, err=16, stream=None)
    return lib.vj_paged_prefill(*{**a, **kw}.values())


def _mixed(lib, **kw):
    a = dict(q=16, k=16, v=16, bt=16, cu=16, ctx=16, out=16, T=4, S=2, nd=1, Hq=8, Hkv=2, D=128,
             nb=200, bs=16, w=200, bts=200, sb=4096, st=256, sh=128, mq=4, scale=0.1, mc=0, plan=1,
             ws=None, wsb=0, err=16, stream=None)
    return lib.vj_paged_attention_mixed(*{**a, **kw}.values())


@pytest.mark.parametrize("entry", PREFILLS + [_bf16_prefill, _mixed])
@pytest.mark.parametrize("kw", [dict(out=16 + 8), dict(out=1 << 20 | 2), dict(q=1 << 20 | 8)])
def test_prefill_refuses_rows_off_16_byte_boundaries(entry, kw):
    """Rows are written 16 bytes at a time: elsewhere that is a fault on the GPU."""
    from vllm_b200 import _native
    lib = _native.load()
    assert entry(lib, **kw) == _native.VJ_ERR_INVALID_ARGUMENT
    assert b"aligned" in lib.vj_get_last_error()


@pytest.mark.parametrize("entry", PREFILLS)
@pytest.mark.parametrize("kw,overlaps", [
    (dict(out=32), True), (dict(q=32), True), (dict(out=16 + ROWS - 16), True),
    (dict(q=16 + ROWS - 16), True), (dict(out=16 + ROWS), False), (dict(q=16 + ROWS), False),
    (dict(), False),
])
def test_prefill_refuses_an_output_that_lies_across_the_queries(entry, kw, overlaps):
    """out may be q, or elsewhere: the call then goes on to ask for its workspace."""
    from vllm_b200 import _native
    lib = _native.load()
    status = entry(lib, **kw)
    if overlaps:
        assert status == _native.VJ_ERR_INVALID_ARGUMENT and b"overlap" in lib.vj_get_last_error()
    else:
        assert status == _native.VJ_ERR_WORKSPACE


@pytest.mark.parametrize("size", ["vj_paged_prefill_split_workspace_size",
                                  "vj_paged_prefill_quantized_workspace_size"])
@pytest.mark.parametrize("Hq,Hkv", [(64, 8), (8, 8), (16, 1)])
@pytest.mark.parametrize("new", [1, 64, 300, 2048])
def test_prefill_workspace_is_bounded_however_large_the_batch(size, Hq, Hkv, new):
    """Room for the rows of the sequences asked for, split over as many CTAs as the GPU
    holds (148 of 256 rows, and a part's row is 130 32-bit words), not for the whole
    batch's rows."""
    from vllm_b200 import _native
    f = getattr(_native.load(), size)
    most = 148 * 256 * 130 * 4
    assert f(1, 1, Hq, Hkv, 128, 1, 1 << 16) > 0
    for seqs in (1, 2, 9):
        for batch in (9, 257):
            need = f(batch * new, seqs, Hq, Hkv, 128, new, 1 << 16)
            assert need == f(seqs * new, seqs, Hq, Hkv, 128, new, 1 << 16) <= most


def test_calls_of_another_torch_are_neither_loaded_nor_kept(monkeypatch):
    """The compiled calls hold what they were built for: another torch or Python refuses
    them, and the build makes them again."""
    from vllm_b200 import _native, build
    assert _native.load_calls().target == _native.calls_target()
    assert _native.calls_match()
    monkeypatch.setattr(_native, "calls_target", lambda: "vllm_b200 calls for torch 9.9, cpython-399;")
    assert build._calls_stale()
    with pytest.raises(RuntimeError, match="torch 9.9"):
        _native.load_calls()


@pytest.mark.parametrize("seqs,hkv,ctx", [(1, 8, 100), (256, 8, 16384), (4, 1, 300), (2, 8, 300_000)])
def test_pool_leaves_room_for_the_prefill_scratch(seqs, hkv, ctx):
    """A gpu_memory_utilization that leaves a bf16 engine enough leaves a quantised one as
    much beside its prefill's scratch, which is what the wrapper and the C entries ask for."""
    from vllm_b200 import Config, _native
    from vllm_b200.kernels.quantized_cache import PREFILL_SCRATCH_ROWS, prefill_scratch_bytes
    from vllm_b200.model.qwen3 import Qwen3Config
    from vllm_b200.src import model_runner as mr
    mcfg = Qwen3Config(num_attention_heads=4 * hkv, num_key_value_heads=hkv)
    base = dict(model="tiny", max_num_batched_tokens=8192, max_num_seqs=seqs, num_blocks=0,
                block_size=16, max_model_len=ctx, compat=False, gpu_memory_utilization=0.9)
    free = 150 << 30
    bf16, e4m3 = Config(**base), Config(**base, kv_cache_dtype="e4m3")
    assert mr.kv_cache_num_blocks(free, bf16, mcfg, 1) == \
        int(free * 0.9) // mr.kv_cache_bytes_per_block(mcfg, 16, 1)
    n = mr.kv_cache_num_blocks(free, e4m3, mcfg, 1)
    taken = n * mr.kv_cache_bytes_per_block(mcfg, 16, 1, "e4m3")
    held = -(-ctx // 16) * 16                       # what a sequence's block table holds
    padded = -(-held // 128) * 128
    groups = -(-seqs // min(seqs, max(1, PREFILL_SCRATCH_ROWS // (padded * hkv))))
    group = -(-seqs // groups)
    needs = 2 * group * padded * hkv * 128 * 2 + max(
        _native.load().vj_paged_prefill_split_workspace_size(8192, s, 4 * hkv, hkv, 128, new, padded)
        for s in (group, max(group - 1, 1)) for new in (1, 33, 64, 100, 300))
    assert needs <= prefill_scratch_bytes(seqs, hkv, held)
    assert taken + prefill_scratch_bytes(seqs, hkv, held) <= int(free * 0.9)
    assert mr.kv_cache_num_blocks(1 << 20, e4m3, mcfg, 1) == 0


def test_bf16_calls_name_the_quantised_ones():
    import torch
    from vllm_b200.kernels.decode_paged_attention import decode_paged_attention
    from vllm_b200.kernels.prefill_paged_attention import prefill_paged_attention
    q, pages = torch.zeros(2, 4, 128), torch.zeros(2, 3, 16, 128)
    bt, n = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    cu, scales = torch.tensor([0, 1, 2], dtype=torch.int32), torch.zeros(2, 3, 16)
    for kw in (dict(k_scales_pages=scales), dict(v_scales_pages=scales)):
        with pytest.raises(NotImplementedError, match="paged_decode_quantized"):
            decode_paged_attention(q, pages, pages, bt, n, **kw)
        with pytest.raises(NotImplementedError, match="paged_prefill_quantized"):
            prefill_paged_attention(q, pages, pages, bt, cu, n, n, max_seqlen_bucket=1, **kw)
    with pytest.raises(NotImplementedError, match="soft-cap"):
        decode_paged_attention(q, pages, pages, bt, n, attn_logits_soft_cap=30.0)
    with pytest.raises(NotImplementedError, match="soft-cap"):
        prefill_paged_attention(q, pages, pages, bt, cu, n, n, max_seqlen_bucket=1,
                                attn_logits_soft_cap=30.0)


def _store(lib, **kw):
    """Five tokens of 4/2 heads, q, k and v side by side in rows of 8 heads from 1 << 20 on."""
    at = 1 << 20
    a = dict(q=at, k=at + 4 * 256, v=at + 6 * 256, qw=16, kw=16, pos=16, slots=16, qo=1 << 24, kc=16,
             vc=16, ks=16, vs=16, dt=1, T=5, Hq=4, Hkv=2, D=128, nb=4, bs=16, sb=4096, st=256, sh=128,
             cb=32, ch=16, qrs=1024, krs=1024, vrs=1024, qors=1024, tab=None, tl=0, eps=1e-6, th=1e6,
             fl=3, err=None, stream=None)
    return lib.vj_kv_store_quantized(*{**a, **kw}.values())


@pytest.mark.parametrize("kw", [
    dict(qo=1 << 20, qors=512),                            # packed, over rows that are not
    dict(qo=(1 << 20) + 256),                              # a head further on, into k
    dict(qo=(1 << 20) - 256),                              # a head back, into v of the row before
    dict(qo=(1 << 20) + 1024),                             # k's and v's place
    dict(qo=(1 << 20) + 2048 * 2 + 512),                   # two rows on
    dict(qo=(1 << 20) + 256, T=1, qrs=0, krs=0, vrs=0),
    dict(k=1 << 24),
    dict(v=(1 << 24) + 2048 * 4),
])
def test_store_refuses_an_output_that_lies_across_its_inputs(kw):
    from vllm_b200 import _native
    lib = _native.load()
    assert _store(lib, **kw) == _native.VJ_ERR_INVALID_ARGUMENT
    assert b"overlap" in lib.vj_get_last_error()
