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
