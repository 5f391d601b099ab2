"""The engine with a quantised KV cache (Config.kv_cache_dtype).

Greedy tokens are checked against the oracle replaying the engine's recorded
schedule on a cache that holds what the quantised one stands for: the first
token that differs must be a near tie, as in the bf16 engine's tests (4 bf16
units in the last place of the top logit). A q that the engine rounds once and
the oracle after every step, and the rare k element on the other side of a
rounding border, are of the size of the bf16 roundings that bound already
covers."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cfg():
    from vllm_b200.model.qwen3 import Qwen3Config
    return Qwen3Config(vocab_size=4096, hidden_size=512, intermediate_size=1024,
                       num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=4)


def _engine(w, cfg, **kw):
    from vllm_b200 import Config
    from vllm_b200.src.engine import Engine
    from vllm_b200.src.request import Request
    Request.reset_ids()
    graphs = kw.pop("use_cuda_graphs", True)
    base = dict(model="tiny", max_num_batched_tokens=48, max_num_seqs=4, num_blocks=96,
                block_size=16, max_model_len=256, compat=False)
    return Engine(Config(**{**base, **kw}), torch.device("cuda", 0), model_config=cfg, weights=w,
                  max_slots=16, use_cuda_graphs=graphs)


def _weights(cfg, seed):
    from vllm_b200.model.qwen3 import Qwen3Weights
    return Qwen3Weights(cfg, torch.device("cuda", 0), seed=seed, gen_device="cpu")


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("prefix_caching", [False, True])
def test_chunked_engine_greedy_vs_oracle(dtype, prefix_caching):
    from oracle.quantized import quantised_qwen3
    from oracle.qwen3 import greedy_replay_chunked
    from vllm_b200 import SamplingParams
    cfg = _cfg()
    w = _weights(cfg, 7)
    eng = _engine(w, cfg, kv_cache_dtype=dtype, enable_chunked_prefill=True,
                  enable_prefix_caching=prefix_caching)
    eng.trace = []
    rng = np.random.default_rng(8)
    stem = rng.integers(0, cfg.vocab_size, 60).tolist()
    prompts = [stem + rng.integers(0, cfg.vocab_size, n).tolist() for n in (40, 3, 17)]
    prompts += [rng.integers(0, cfg.vocab_size, n).tolist() for n in (9, 130)]
    new = 12
    outs = eng.generate(prompts, SamplingParams(temperature=0, max_new_tokens=new,
                                                ignore_eos=True))
    assert [len(o) for o in outs] == [new] * len(prompts)
    steps = [st["batch"] for st in eng.trace]
    assert any(any(n == 1 for *_, n in s) and any(n > 1 for *_, n in s) for s in steps)
    if prefix_caching:
        assert eng.scheduler.prefix_hit_tokens > 0
    model = quantised_qwen3(cfg, w.full_numpy(), 96, 16, dtype)
    tokens, gaps = greedy_replay_chunked(model, eng.trace, prompts)
    n_match, first = 0, None
    for r, p in enumerate(prompts):
        for i, (a, b) in enumerate(zip(outs[r], tokens[r][len(p):])):
            if a != b:
                first = (r, i) if first is None or i < first[1] else first
                break
            n_match += 1
    if first is not None:
        r, i = first
        k = -1
        for g in gaps:
            if r in g:
                k += 1
                if k == i:
                    _, top, gap = g[r]
                    break
        ulp = 2.0 ** (math.floor(math.log2(max(abs(top), 2.0 ** -10))) - 7)
        assert gap <= 4 * ulp + 1e-9, f"request {r} diverged at token {i}, oracle gap {gap}"
    assert n_match >= new * len(prompts) // 2


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_graphs_fused_projections_and_lookahead_give_the_same_tokens(dtype):
    """Prefill and decode batches: captured decode steps equal eager ones, token for token;
    the lookahead loop and the fused projections run (their GEMMs sum in another order)."""
    from vllm_b200 import SamplingParams
    cfg = _cfg()
    w = _weights(cfg, 9)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, cfg.vocab_size, n).tolist() for n in (20, 33, 7, 16, 40)]
    sp = SamplingParams(temperature=0, max_new_tokens=10, ignore_eos=True)
    runs = []
    for kw in (dict(), dict(use_cuda_graphs=False), dict(async_scheduling=False)):
        eng = _engine(w, cfg, kv_cache_dtype=dtype, max_num_batched_tokens=128, **kw)
        runs.append(eng.generate(prompts, sp))
        eng.close()
    assert runs[0] == runs[1] == runs[2]
    assert [len(o) for o in runs[0]] == [10] * len(prompts)
    eng = _engine(w, cfg, kv_cache_dtype=dtype, max_num_batched_tokens=128, fused_gemm_max_rows=16)
    assert [len(o) for o in eng.generate(prompts, sp)] == [10] * len(prompts)


def test_pool_is_sized_by_the_row_bytes():
    from vllm_b200.src.model_runner import kv_cache_bytes_per_block
    cfg = _cfg()
    eng = _engine(_weights(cfg, 1), cfg, kv_cache_dtype="int8")
    cache = eng.runner.kv_caches[0]
    per = kv_cache_bytes_per_block(cfg, 16, 1, "int8")
    assert (cache.data.numel() + cache.scales.numel()) * cfg.num_hidden_layers == per * 96
    assert kv_cache_bytes_per_block(cfg, 16, 1) * 129 == per * 256
