"""The quantised KV cache in NumPy, 64 bits throughout.

A row of 128 is 8-bit elements and one E8M0 byte; quantise_rows searches the
nearest element among all of them (ties to the even code) under the smallest
power-of-two scale that fits the row, dequantise is the product.
No counterpart in vllm-jax, which caches bf16 only.
"""
from __future__ import annotations

import numpy as np


def _e4m3_values() -> np.ndarray:
    """Value of each e4m3 code 0..126 (127 is NaN); codes 128.. are their negatives."""
    c = np.arange(127)
    e, m = c >> 3, c & 7
    return np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))


POSITIVE = {"e4m3": _e4m3_values(), "int8": np.arange(128, dtype=np.float64)}
LARGEST = {"e4m3": 448.0, "int8": 127.0}


def quantise_rows(x: np.ndarray, dtype: str) -> tuple[np.ndarray, np.ndarray]:
    """x [..., D] float64 -> (codes uint8 [..., D], scale bytes uint8 [...])."""
    pos = POSITIVE[dtype]
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], 0.0, x)
    amax = np.abs(x).max(-1)
    e = np.full(amax.shape, -126)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):
        e = np.where(amax > LARGEST[dtype] * np.exp2(e + step - 1.0), e + step, e)
    y = x * np.exp2(-e.astype(np.float64))[..., None]
    mids = (pos[1:] + pos[:-1]) / 2
    lo, hi = np.searchsorted(mids, np.abs(y), "left"), np.searchsorted(mids, np.abs(y), "right")
    code = np.where(lo % 2 == 0, lo, hi)      # equal unless y is a midpoint
    if dtype == "e4m3":
        code = code | np.where(np.signbit(y), 128, 0)
    else:
        code = np.where(y < 0, -code, code)
    return code.astype(np.int64).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def element_values(codes: np.ndarray, dtype: str) -> np.ndarray:
    codes = codes.astype(np.uint8)
    if dtype == "int8":
        return codes.view(np.int8).astype(np.float64)
    v = np.append(POSITIVE["e4m3"], np.nan)[codes & 127]
    return np.where(codes & 128, -v, v)


def scale_values(b: np.ndarray) -> np.ndarray:
    return np.where(b == 255, np.nan, np.exp2(b.astype(np.float64) - 127))


def dequantise(codes: np.ndarray, scales: np.ndarray, dtype: str) -> np.ndarray:
    """codes [nb, bs, H, D], scales [nb, H, bs] -> float64 [nb, bs, H, D]."""
    return element_values(codes, dtype) * scale_values(scales).transpose(0, 2, 1)[..., None]


def norm_rope(x: np.ndarray, w: np.ndarray | None, cos_sin: np.ndarray | None,
              eps: float) -> np.ndarray:
    """x [T, H, D] float64: RMSNorm with weight w, then the pairs (2i, 2i+1)
    turned by cos_sin [T, D/2, 2]."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    if cos_sin is not None:
        z = (x[..., 0::2] + 1j * x[..., 1::2]) * (cos_sin[..., 0] + 1j * cos_sin[..., 1])[:, None]
        x = np.stack([z.real, z.imag], -1).reshape(x.shape)
    return x


def gather(values: np.ndarray, table: np.ndarray, n: int) -> np.ndarray:
    """First n positions of a sequence: values [nb, bs, H, D] through a block
    table row (entries outside the pool read block 0)."""
    nb, bs = values.shape[:2]
    t = table[:-(-n // bs)]
    t = np.where((t < 0) | (t >= nb), 0, t)
    return values[t].reshape(-1, *values.shape[2:])[:n]


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, first: int, scale: float):
    """Rows q [n, Hq, D] at positions first.. over k, v [L, Hkv, D], causal.
    Returns (out, sum of p |v|), both [n, Hq, D]; the second bounds what a
    relative error of the weights can do to the first."""
    n, hq, D = q.shape
    g = hq // k.shape[1]
    out, mag = np.zeros((n, hq, D)), np.zeros((n, hq, D))
    for h in range(hq):
        s = scale * (q[:, h] @ k[:, h // g].T)
        s = np.where(np.arange(k.shape[0])[None] <= first + np.arange(n)[:, None], s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[:, h], mag[:, h] = p @ v[:, h // g], p @ np.abs(v[:, h // g])
    return out, mag


def quantised_qwen3(cfg, W, num_blocks: int, block_size: int, dtype: str):
    """An OracleQwen3 whose cache holds what a quantised one stands for."""
    from .qwen3 import OracleQwen3

    class Model(OracleQwen3):
        def _layer(self, l, x, positions, slots, attn):
            def rounded(l, q):
                for cache in (self.kc[l], self.vc[l]):
                    flat = cache.reshape(-1, *cache.shape[2:])
                    at = np.asarray([s for s in slots if 0 <= s < flat.shape[0]], np.int64)
                    codes, b = quantise_rows(flat[at].astype(np.float64), dtype)
                    flat[at] = element_values(codes, dtype) * scale_values(b)[..., None]
                return attn(l, q)
            return super()._layer(l, x, positions, slots, rounded)

    return Model(cfg, W, num_blocks, block_size)
