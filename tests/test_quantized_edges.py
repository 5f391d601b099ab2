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
