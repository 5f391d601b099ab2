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

import functools
import math
from typing import NamedTuple

import torch

from .. import _native
from ._util import require_cuda, require_dtype
from .kv_store import rope_table
from .prefill_paged_attention import _err_flag, _err_flags

CACHE_DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_CODES = {torch.float8_e4m3fn: _native.VJ_CACHE_E4M3, torch.int8: _native.VJ_CACHE_INT8}


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


def _pool(cache: QuantizedKVCache):
    """(pointers, element type, Hkv, D, num_blocks, block_size, strides) of a cache."""
    data, scales = cache.data, cache.scales
    shape = data.shape
    if len(shape) != 5 or shape[0] != 2:
        raise ValueError("cache.data must have shape (2, num_blocks, block_size, Hkv, D); "
                         f"got {tuple(shape)}")
    _, nb, bs, hkv, D = shape
    code = _CODES.get(data.dtype)
    if code is None:
        raise ValueError(f"The dtype of `cache.data` must be float8_e4m3fn or int8. Got {data.dtype}")
    if scales.dtype is not torch.uint8:
        require_dtype(scales, torch.uint8, "cache.scales")
    if scales.shape != (2, nb, hkv, bs):
        raise ValueError(f"cache.scales must have shape (2, num_blocks, Hkv, block_size) = "
                         f"{(2, nb, hkv, bs)}; got {tuple(scales.shape)}")
    s2, sb, st, sh, s1 = data.stride()
    c2, cb, ch, c1 = scales.stride()
    if s1 != 1 or c1 != 1:
        raise ValueError("cache.data's head_dim and cache.scales' block_size must be contiguous")
    d, s = data.data_ptr(), scales.data_ptr()
    return (d, d + s2, s, s + c2), code, hkv, D, nb, bs, (sb, st, sh, cb, ch)


def _index(*tensors: torch.Tensor | None) -> int:
    """The CUDA device all tensors are on."""
    index = -1
    for t in tensors:
        if t is not None:
            i = t.get_device()
            if i != index or i < 0:
                if index >= 0 or i < 0:
                    require_cuda(*tensors)       # raises
                index = i
    return index


def _call(index: int, name: str, *args) -> None:
    """A C entry on the tensors' device (it launches on the current one)."""
    if index == torch._C._cuda_getDevice():
        _native.call(name, *args)
    else:
        with torch.cuda.device(index):
            _native.call(name, *args)


def _error(index: int) -> int:
    t = _err_flags.get(index)
    return (_err_flag(torch.device("cuda", index)) if t is None else t).data_ptr()


def _stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _rows(t: torch.Tensor, name: str, T: int, D: int) -> tuple[int, int]:
    """(heads, row stride) of a [T, H, D] tensor with packed heads."""
    shape = t.shape
    if len(shape) == 3 and t.dtype is torch.bfloat16:
        rs, hs, es = t.stride()
        if shape[0] == T and shape[2] == D and es == 1 and (hs == D or shape[1] == 1):
            return shape[1], rs
    require_dtype(t, torch.bfloat16, name)
    raise ValueError(f"`{name}` must be a [num_tokens, H, head_dim] tensor with packed heads")


def _indices(t: torch.Tensor, name: str, T: int) -> None:
    if t.dtype is not torch.int32:
        require_dtype(t, torch.int32, name)
    if t.shape != (T,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{T}] tensor; got shape {tuple(t.shape)}")


def _weight(w: torch.Tensor, name: str, D: int) -> int:
    require_dtype(w, torch.bfloat16, name)
    if w.shape != (D,) or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [head_dim] tensor")
    return w.data_ptr()


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
    negative ones); the others must differ from each other within a call."""
    dev = _index(k, v, cache.data, cache.scales, slot_mapping, q, positions, q_norm_weight,
                 k_norm_weight, q_out, table)
    ptrs, code, Hkv, D, nb, bs, strides = _pool(cache)
    T = k.shape[0]
    if v.shape != k.shape:
        raise ValueError(f"k and v must have the same shape. Got {tuple(k.shape)} and {tuple(v.shape)}")
    heads, k_stride = _rows(k, "k", T, D)
    _, v_stride = _rows(v, "v", T, D)
    if heads != Hkv:
        raise ValueError("cache heads/head_dim do not match k")
    _indices(slot_mapping, "slot_mapping", T)
    Hq = q_stride = out_stride = 0
    q_ptr = out_ptr = qw_ptr = kw_ptr = pos_ptr = table_ptr = None
    if q is not None:
        Hq, q_stride = _rows(q, "q", T, D)
        if q_out is None:
            q_out = k.new_empty((T, Hq, D))
            out_stride = Hq * D
        else:
            out_heads, out_stride = _rows(q_out, "q_out", T, D)
            if out_heads != Hq:
                raise ValueError("q_out must have q's shape")
        q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out needs q")
    flags = 0
    if norm:
        flags = _native.VJ_KV_NORM
        if k_norm_weight is None or (q is not None and q_norm_weight is None):
            raise ValueError("norm=True needs q_norm_weight and k_norm_weight")
        kw_ptr = _weight(k_norm_weight, "k_norm_weight", D)
        if q is not None:
            qw_ptr = _weight(q_norm_weight, "q_norm_weight", D)
    tab_len = 0
    if rope:
        flags |= _native.VJ_KV_ROPE
        if positions is None:
            raise ValueError("rope=True needs positions")
        _indices(positions, "positions", T)
        pos_ptr = positions.data_ptr()
        if table is None:
            table = rope_table(k.device, rope_theta)
        require_dtype(table, torch.int32, "table")
        if not table.is_contiguous():
            raise ValueError("table must be contiguous")
        tab_len = table.numel() // 64
        if tab_len:
            table_ptr = table.data_ptr()
    _call(dev, "vj_kv_store_quantized", q_ptr, k.data_ptr(), v.data_ptr(), qw_ptr, kw_ptr,
          pos_ptr, slot_mapping.data_ptr(), out_ptr, *ptrs, code, T, Hq, Hkv, D, nb, bs, *strides,
          q_stride, k_stride, v_stride, out_stride, table_ptr, tab_len, eps, rope_theta, flags,
          _error(dev), _stream(dev))
    return q_out


def _tables(block_tables: torch.Tensor, context_lens: torch.Tensor, B: int) -> tuple[int, int]:
    """(width, row stride) of the block tables."""
    if block_tables.dtype is not torch.int32:
        require_dtype(block_tables, torch.int32, "block_tables")
    shape = block_tables.shape
    if len(shape) != 2 or shape[0] != B:
        raise ValueError("`block_tables` must have one row per sequence")
    width = shape[1]
    stride, s1 = block_tables.stride()
    if s1 != 1 and width > 1:
        raise ValueError("block_tables rows must be contiguous")
    if stride < width:
        if B > 1:
            raise ValueError("block_tables rows must not overlap")
        stride = width
    _indices(context_lens, "context_lens", B)
    return width, stride


def paged_decode_quantized(q: torch.Tensor, cache: QuantizedKVCache, block_tables: torch.Tensor,
                           context_lens: torch.Tensor, scale: float | None = None,
                           out: torch.Tensor | None = None,
                           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode over a quantised cache: q [B, Hq, D] bf16, at most 16 query
    heads per KV head; rows with no context come out 0. Cached rows past a
    sequence's context are not used, whatever they hold. `workspace` (uint8,
    decode_quantized_workspace_bytes(...) long): the split's scratch; by
    default a fresh allocation of the call's own."""
    dev = _index(q, cache.data, cache.scales, block_tables, context_lens, out, workspace)
    ptrs, code, Hkv, D, nb, bs, strides = _pool(cache)
    require_dtype(q, torch.bfloat16, "q")
    if q.dim() != 3 or not q.is_contiguous():
        raise ValueError("q must be a contiguous [batch, Hq, head_dim] tensor")
    B, Hq, Dq = q.shape
    if Dq != D or Hq % Hkv:
        raise ValueError("q heads/head_dim do not match the cache")
    width, stride = _tables(block_tables, context_lens, B)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous bf16 tensor of q's shape")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    need = _decode_workspace_bytes(dev, B, Hq, Hkv, D, width, bs)
    if workspace is None:
        workspace = q.new_empty(need, dtype=torch.uint8)
    elif workspace.dtype != torch.uint8 or workspace.numel() < need \
            or not workspace.is_contiguous():
        raise ValueError(f"decode workspace must be contiguous uint8 with >= {need} bytes")
    _call(dev, "vj_paged_decode_quantized", q.data_ptr(), *ptrs, code, block_tables.data_ptr(),
          context_lens.data_ptr(), out.data_ptr(), B, Hq, Hkv, D, nb, bs, width, stride, *strides,
          scale, workspace.data_ptr(), workspace.numel(), _error(dev), _stream(dev))
    return out


@functools.lru_cache(maxsize=1024)
def _decode_workspace_bytes(index: int, *sizes: int) -> int:
    with torch.cuda.device(index):       # the split goes by the device's SMs
        return int(_native.load().vj_paged_decode_quantized_workspace_size(*sizes))


def decode_quantized_workspace_bytes(batch: int, num_q_heads: int, num_kv_heads: int,
                                     table_width: int, block_size: int,
                                     head_dim: int = 128) -> int:
    """Scratch of one paged_decode_quantized call, on the current device, with
    block tables of table_width entries."""
    return _decode_workspace_bytes(torch.cuda.current_device(), batch, num_q_heads, num_kv_heads,
                                   head_dim, table_width, block_size)


def _read(index: int, pool, tables: int, width: int, stride: int, lens: int, out: int, B: int,
          max_len: int, zero_to: int) -> None:
    """vj_kv_read_quantized into packed K, then V, at address `out`."""
    ptrs, code, Hkv, D, nb, bs, strides = pool
    _call(index, "vj_kv_read_quantized", *ptrs, code, tables, lens, out,
          out + B * max_len * Hkv * D * 2, B, max_len, zero_to, Hkv, D, nb, bs, width, stride,
          *strides, _stream(index))


def read_kv_cache(cache: QuantizedKVCache, block_tables: torch.Tensor,
                  context_lens: torch.Tensor, max_context_len: int = 0,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The K and V of a batch as bf16, (2, B, max_context_len, Hkv, D): row t of
    sequence b is its cached position t, exactly (a scale is a power of two),
    and zeros from context_lens[b] on. max_context_len: rows per sequence
    (default: what a block table row holds); longer contexts are cut there."""
    dev = _index(cache.data, cache.scales, block_tables, context_lens, out)
    pool = _pool(cache)
    _, _, Hkv, D, _, bs, _ = pool
    B = block_tables.shape[0]
    width, stride = _tables(block_tables, context_lens, B)
    if max_context_len < 0:
        raise ValueError("max_context_len must not be negative")
    L = int(max_context_len) or width * bs
    shape = (2, B, L, Hkv, D)
    if out is None:
        out = cache.data.new_empty(shape, dtype=torch.bfloat16)
    elif out.shape != shape or out.dtype != torch.bfloat16 or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous bf16 tensor of shape {shape}")
    _read(dev, pool, block_tables.data_ptr(), width, stride, context_lens.data_ptr(),
          out.data_ptr(), B, L, 0)
    return out


_identity: dict[int, torch.Tensor] = {}
_retired_identity: list[torch.Tensor] = []


def _identity_pages(dev: torch.device, n: int) -> torch.Tensor:
    """0, 1, .., the block tables of a scratch whose pages lie in order, kept per
    device and only grown. An outgrown tensor is kept too: a captured graph may
    read it. What a capture makes is the graph's own."""
    if torch.cuda.is_current_stream_capturing():
        t = _identity.get(dev.index)
        return t[:n] if t is not None and t.numel() >= n else \
            torch.arange(n, dtype=torch.int32, device=dev)
    t = _identity.get(dev.index)
    if t is None or t.numel() < n:
        if t is not None:
            _retired_identity.append(t)
        # a blocking copy: complete for every stream when it returns
        t = torch.arange(max(n, 1 << 16), dtype=torch.int32).to(dev)
        _identity[dev.index] = t
    return t[:n]


# bf16 rows (token x KV head) of one read-back inside paged_prefill_quantized:
# 1 GiB of K and V. Batches that need more run in groups of sequences.
PREFILL_SCRATCH_ROWS = 1 << 21
_KEY_TILE = 128      # keys a prefill tile reads at once


def paged_prefill_quantized(q: torch.Tensor, cache: QuantizedKVCache, block_tables: torch.Tensor,
                            cu_seqlens_q: torch.Tensor, context_lens: torch.Tensor | None = None,
                            max_seqlen_q: int = 0, scale: float | None = None,
                            out: torch.Tensor | None = None,
                            max_context_len: int = 0) -> torch.Tensor:
    """paged_prefill over a quantised cache: causal attention of the new tokens
    (rows [cu_seqlens_q[s], cu_seqlens_q[s+1]) of q) of each sequence over its
    cached context, theirs included. The contexts are read back to bf16, which
    is exact, and attended to from there: a prompt's attention does far more
    work per key than reading it back, and the conversion is done once instead
    of once per query tile. max_context_len: a bound on context_lens (default:
    what a block table row holds); it sizes the scratch, as max_seqlen_q sizes
    the grid."""
    dev = _index(q, cache.data, cache.scales, block_tables, cu_seqlens_q, context_lens, out)
    pool = _pool(cache)
    _, _, Hkv, D, _, bs, _ = pool
    require_dtype(q, torch.bfloat16, "q")
    require_dtype(cu_seqlens_q, torch.int32, "cu_seqlens_q")
    if q.dim() != 3 or not q.is_contiguous():
        raise ValueError("q must be a contiguous [num_tokens, Hq, head_dim] tensor")
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] < 1 or not cu_seqlens_q.is_contiguous():
        raise ValueError("cu_seqlens_q must be a contiguous [num_seqs + 1] tensor")
    if q.shape[2] != D or q.shape[1] % Hkv:
        raise ValueError("q heads/head_dim do not match the cache")
    S = cu_seqlens_q.shape[0] - 1
    if context_lens is None:
        context_lens = cu_seqlens_q[1:] - cu_seqlens_q[:-1]
    width, stride = _tables(block_tables, context_lens, S)
    if max_context_len < 0:
        raise ValueError("max_context_len must not be negative")
    capacity = width * bs
    L = min(int(max_context_len) or capacity, capacity)
    L = max(-(-L // 16) * 16, 16)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous bf16 tensor of q's shape")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    group = max(1, min(S, PREFILL_SCRATCH_ROWS // (L * Hkv)))
    T, Hq, _ = q.shape
    per_seq = L // 16                  # page p of the group's sequence b: block b * per_seq + p
    half = group * L * Hkv * D         # elements of the scratch's K, and of its V
    pages = _identity_pages(q.device, group * per_seq).data_ptr()
    scratch = q.new_empty(2 * half)
    k_ptr = scratch.data_ptr()
    tables, lens = block_tables.data_ptr(), context_lens.data_ptr()
    for s in range(0, max(S, 1), group):
        n = min(group, S - s)
        _read(dev, pool, tables + 4 * s * stride, width, stride, lens + 4 * s, k_ptr, n, L,
              _KEY_TILE)
        _call(dev, "vj_paged_prefill", q.data_ptr(), k_ptr, k_ptr + n * L * Hkv * D * 2, pages,
              cu_seqlens_q.data_ptr() + 4 * s, lens + 4 * s, out.data_ptr(), T, n, Hq, Hkv, D,
              max(n, 1) * per_seq, 16, per_seq, per_seq, 16 * Hkv * D, Hkv * D, D,
              int(max_seqlen_q), scale, _error(dev), _stream(dev))
    return out
