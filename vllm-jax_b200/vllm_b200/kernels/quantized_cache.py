"""The quantised KV cache and the operators on it, torch-facing.

A cached row (one token, one KV head, K or V) is head_dim 8-bit elements, e4m3
or int8, and one power-of-two scale, so a cache takes 129 bytes a row instead
of 256. The calls mirror the bf16 ones:

  kv_store_quantized        kv_store_qknorm_rope with k and v rounded to 8 bits
  paged_decode_quantized    paged_decode
  paged_prefill_quantized   paged_prefill
  read_kv_cache             a batch's K and V back as bf16

vllm-jax names quantised pages in its attention signatures (k_scales_pages,
v_scales_pages, vllm/kernels/decode_paged_attention.py:300-341) but has no
cache that holds them; the format here (vj_kv_store_quantized in
include/vjattn.h) has no counterpart there.
"""
from __future__ import annotations

import threading
from typing import NamedTuple

import torch

from .. import _native
from .kv_store import rope_table
from .prefill_paged_attention import _err_flag

CACHE_DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class QuantizedKVCache(NamedTuple):
    """A layer's pool: `data` (2, num_blocks, block_size, Hkv, head_dim)
    float8_e4m3fn or int8, and `scales` (2, num_blocks, Hkv, block_size) uint8,
    the E8M0 byte of each row: a row stands for data * 2^(scales - 127). Any
    strides that are multiples of 16 do, as long as data's last dim and scales'
    last dim are contiguous and a block's tokens are evenly strided on to the
    next block's."""
    data: torch.Tensor
    scales: torch.Tensor

    @staticmethod
    def zeros(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int = 128,
              dtype: str = "e4m3", device=None) -> "QuantizedKVCache":
        """A pool whose every row reads as zeros. dtype: "e4m3" or "int8"."""
        if dtype not in CACHE_DTYPES:
            raise ValueError(f"cache dtype must be one of {sorted(CACHE_DTYPES)}; got {dtype!r}")
        return QuantizedKVCache(
            torch.zeros((2, num_blocks, block_size, num_kv_heads, head_dim),
                        dtype=CACHE_DTYPES[dtype], device=device),
            torch.full((2, num_blocks, num_kv_heads, block_size), 127, dtype=torch.uint8,
                       device=device))


_lock = threading.Lock()
_calls = None


def _bound():
    """The compiled calls, which check the arguments, allocate and launch."""
    global _calls
    with _lock:
        if _calls is None:
            calls = _native.load_calls()
            calls.bind(*(_native.address(name) for name in
                         ("vj_kv_store_quantized", "vj_paged_decode_quantized",
                          "vj_paged_decode_quantized_workspace_size", "vj_kv_read_quantized",
                          "vj_paged_prefill_split", "vj_paged_prefill_split_part",
                          "vj_paged_prefill_split_workspace_size",
                          "vj_paged_prefill_quantized",
                          "vj_paged_prefill_quantized_workspace_size")),
                       _native, _error_address, rope_table)
            _calls = calls
    return _calls


def _error_address(index: int) -> int:
    return _err_flag(torch.device("cuda", index)).data_ptr()


def kv_store_quantized(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                       cache: QuantizedKVCache, slot_mapping: torch.Tensor,
                       positions: torch.Tensor | None = None,
                       q_norm_weight: torch.Tensor | None = None,
                       k_norm_weight: torch.Tensor | None = None, *, eps: float = 1e-6,
                       rope_theta: float = 1e6, norm: bool = True, rope: bool = True,
                       q_out: torch.Tensor | None = None,
                       table: torch.Tensor | None = None) -> torch.Tensor | None:
    """One launch: q_out = rope(norm(q)), cache[slot] = 8 bits of (rope(norm(k)), v).

    The arguments are kv_store_qknorm_rope's. q is rounded to bf16 once, k and
    v to 8 bits once (kv_store_qknorm_rope rounds after every step, as the
    reference does). Slots outside the pool store nothing (there is no wrap of
    negative ones); the others must differ from each other within a call. q_out may
    be q, or must not overlap q, k and v."""
    return (_calls or _bound()).kv_store(q, k, v, cache, slot_mapping, positions, q_norm_weight,
                                         k_norm_weight, eps, rope_theta, norm, rope, q_out, table)


def paged_decode_quantized(q: torch.Tensor, cache: QuantizedKVCache, block_tables: torch.Tensor,
                           context_lens: torch.Tensor, scale: float | None = None,
                           out: torch.Tensor | None = None,
                           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode over a quantised cache: q [B, Hq, D] bf16, at most 16 query
    heads per KV head; rows with no context come out 0. Cached rows past a
    sequence's context are not used, whatever they hold. `workspace` (uint8,
    decode_quantized_workspace_bytes(...) long): the split's scratch; by
    default a fresh allocation of the call's own."""
    return (_calls or _bound()).paged_decode(q, cache, block_tables, context_lens, scale, out,
                                             workspace)


def decode_quantized_workspace_bytes(batch: int, num_q_heads: int, num_kv_heads: int,
                                     table_width: int, block_size: int,
                                     head_dim: int = 128) -> int:
    """Scratch of one paged_decode_quantized call, on the current device, with
    block tables of table_width entries."""
    return int(_native.load().vj_paged_decode_quantized_workspace_size(
        batch, num_q_heads, num_kv_heads, head_dim, table_width, block_size))


def read_kv_cache(cache: QuantizedKVCache, block_tables: torch.Tensor,
                  context_lens: torch.Tensor, max_context_len: int = 0,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The K and V of a batch as bf16, (2, B, max_context_len, Hkv, D): row t of
    sequence b is its cached position t, exactly (a scale is a power of two),
    and zeros from context_lens[b] on. max_context_len: rows per sequence
    (default: what a block table row holds); longer contexts are cut there."""
    return (_calls or _bound()).read_kv_cache(cache, block_tables, context_lens,
                                              int(max_context_len), out)


# bf16 rows (token x KV head) of one read-back inside paged_prefill_quantized:
# 1 GiB of K and V. Batches that need more run in groups of sequences.
PREFILL_SCRATCH_ROWS = 1 << 21


def prefill_scratch_bytes(num_seqs: int, num_kv_heads: int, max_context_len: int,
                          head_dim: int = 128) -> int:
    """A bound on the memory that a paged_prefill_quantized call of up to num_seqs
    sequences allocates beside its output: the contexts read back (whole key tiles of
    128), and the parts of split keys (256 rows a CTA at most, one CTA an SM of 148)."""
    rows = -(-max_context_len // 128) * 128 * num_kv_heads
    rows = min(num_seqs * rows, max(PREFILL_SCRATCH_ROWS, rows))
    return rows * 2 * head_dim * 2 + 148 * 256 * (head_dim + 2) * 4


def paged_prefill_quantized(q: torch.Tensor, cache: QuantizedKVCache, block_tables: torch.Tensor,
                            cu_seqlens_q: torch.Tensor, context_lens: torch.Tensor | None = None,
                            max_seqlen_q: int = 0, scale: float | None = None,
                            out: torch.Tensor | None = None,
                            max_context_len: int = 0) -> torch.Tensor:
    """paged_prefill over a quantised cache: causal attention of the new tokens
    (rows [cu_seqlens_q[s], cu_seqlens_q[s+1]) of q) of each sequence over its
    cached context, theirs included (context_lens is no less than the new tokens).
    Few new tokens take the quantised pages in directly; for many, whose attention
    does far more work per key, the contexts are read back to bf16 first, which is
    exact, once instead of once per query tile. max_seqlen_q and max_context_len:
    bounds on the new tokens and on context_lens (default: all tokens, and what a
    block table row holds); they size the grid and the scratch, and decide how the
    keys are split. scale: positive. Rows behind cu_seqlens_q[-1] come out 0. `out` may be
    q, or must not overlap it."""
    return (_calls or _bound()).paged_prefill(q, cache, block_tables, cu_seqlens_q, context_lens,
                                              int(max_seqlen_q), scale, out, int(max_context_len),
                                              PREFILL_SCRATCH_ROWS)
