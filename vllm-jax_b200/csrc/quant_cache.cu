// Quantised KV cache: the store (q/k RMSNorm + RoPE + rounding of k and v to 8
// bits, in one launch) and the read-back to bf16.
//
// Store, per token and head row x of 128:
//   y = rope(x * w / sqrt(mean(x^2) + eps))        (q and k; v: y = x)
//   q_out = bf16(y)
//   e = smallest integer with max|y| <= qmax * 2^e;  cached = RN8(y * 2^-e), byte e + 127
// K rows are computed in 64 bits and rounded once, to 24 bits with a sticky
// last bit and from there to 8 bits: the cached row is the correctly rounded
// one, whatever order a sum was taken in, so two programs (or two ranks, or a
// recomputed prefix) that cache the same token hold the same bytes.
#include "kv_row.cuh"
#include "quant.cuh"

#include <algorithm>

namespace vj {
namespace {
using namespace qn;

struct StoreArgs {
  const __nv_bfloat16 *q, *k, *v, *qw, *kw;
  const int32_t *positions, *slots;
  __nv_bfloat16 *q_out;
  const uint4 *table;
  Pool pool;
  int64_t t_begin;        // first token of this launch
  uint32_t num_rows;      // rows of this launch
  uint32_t heads;         // Hq + 2 Hkv
  int Hq, Hkv, table_len;
  int64_t qrs, krs, vrs, qors;
  double eps;
  bool norm, rope;
  RopeTable freq;
};

// 24 bits of y, truncated, with the last bit set if anything was cut off:
// rounding that to 8 bits equals rounding y itself.
VJ_DEV float round_to_odd(double y) {
  float f = __double2float_rz(y);
  if (static_cast<double>(f) != y) f = __uint_as_float(__float_as_uint(f) | 1u);
  return f;
}

VJ_DEV uint32_t group_max(unsigned mask, uint32_t v) {
#pragma unroll
  for (int o = 4; o >= 1; o >>= 1) v = max(v, __shfl_xor_sync(mask, v, o));
  return v;
}

constexpr int kStoreThreads = 256;

// 8 lanes own a row; lane l8 holds dims [8*l8, +8) and [64 + 8*l8, +8).
template <bool kInt8>
__global__ void __launch_bounds__(kStoreThreads) kv_store_quantized_kernel(const StoreArgs a) {
  const int l8 = threadIdx.x & 7;
  const unsigned mask = 0xffu << (threadIdx.x & 24);
  const uint32_t step = gridDim.x * (kStoreThreads / 8);
  for (uint32_t r = blockIdx.x * (kStoreThreads / 8) + (threadIdx.x >> 3); r < a.num_rows;
       r += step) {
    const uint32_t tl = r / a.heads;
    const int h = static_cast<int>(r - tl * a.heads);
    const int64_t t = a.t_begin + tl;
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    int64_t slot = 0;
    if (!is_q) {
      slot = __ldg(a.slots + t);
      if (slot < 0 || slot >= a.pool.num_blocks * a.pool.block_size) continue;
    }
    const __nv_bfloat16 *src = is_q   ? a.q + t * a.qrs + h * kD
                               : is_v ? a.v + t * a.vrs + (h - a.Hq - a.Hkv) * kD
                                      : a.k + t * a.krs + (h - a.Hq) * kD;
    const RowSlice x = ldg_slice(src, l8);
    RowSlice w, cs;
    if (!is_v) {
      if (a.norm) w = ldg_nc_slice(is_q ? a.qw : a.kw, l8);
      if (a.rope) {
        const int pos = __ldg(a.positions + t);
        cs = pos >= 0 && pos < a.table_len
                 ? ldg_nc_slice(reinterpret_cast<const __nv_bfloat16 *>(
                                    a.table + static_cast<int64_t>(pos) * 16), l8)
                 : rope_slice(pos, a.freq, l8);
      }
    }
    if (is_q) {
      float y[16];
#pragma unroll
      for (int j = 0; j < 8; ++j) { y[2 * j] = bf16_lo(x.w[j]); y[2 * j + 1] = bf16_hi(x.w[j]); }
      if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) ss = fmaf(y[j], y[j], ss);
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float inv = 1.0f / sqrtf(ss * (1.0f / kD) + static_cast<float>(a.eps));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          y[2 * j] *= inv * bf16_lo(w.w[j]);
          y[2 * j + 1] *= inv * bf16_hi(w.w[j]);
        }
      }
      RowSlice o;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float u = y[2 * j], z = y[2 * j + 1];
        if (a.rope) {
          const float c = bf16_lo(cs.w[j]), s = bf16_hi(cs.w[j]);
          const float u2 = u * c - z * s;
          z = u * s + z * c;
          u = u2;
        }
        o.w[j] = cvt_bf16x2(u, z);
      }
      stg_slice(a.q_out + t * a.qors + h * kD, l8, o, true);
      continue;
    }
    float y[16];
    if (is_v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) { y[2 * j] = bf16_lo(x.w[j]); y[2 * j + 1] = bf16_hi(x.w[j]); }
    } else {
      double inv = 1.0;
      if (a.norm) {
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const double u = bf16_lo(x.w[j]), z = bf16_hi(x.w[j]);
          ss = fma(u, u, fma(z, z, ss));
        }
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        inv = 1.0 / sqrt(ss * (1.0 / kD) + a.eps);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        double u = bf16_lo(x.w[j]), z = bf16_hi(x.w[j]);
        if (a.norm) {
          u *= inv * bf16_lo(w.w[j]);
          z *= inv * bf16_hi(w.w[j]);
        }
        if (a.rope) {
          const double c = bf16_lo(cs.w[j]), s = bf16_hi(cs.w[j]);
          const double u2 = u * c - z * s;
          z = u * s + z * c;
          u = u2;
        }
        y[2 * j] = round_to_odd(u);
        y[2 * j + 1] = round_to_odd(z);
      }
    }
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = max(amax, __float_as_uint(y[j]) & 0x7fffffffu);
    amax = group_max(mask, amax);
    const bool bad = amax >= 0x7f800000u;              // an infinity or NaN in the row
    const int e = bad ? 0 : scale_exponent<kInt8>(amax);
    const float f = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);   // 2^-e
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = quantise2<kInt8>(y[4 * j] * f, y[4 * j + 1] * f);
      const uint32_t hi = quantise2<kInt8>(y[4 * j + 2] * f, y[4 * j + 3] * f);
      o[j] = bad ? 0u : lo | (hi << 16);
    }
    const int hk = is_v ? h - a.Hq - a.Hkv : h - a.Hq;
    const int64_t blk = slot / a.pool.block_size, off = slot % a.pool.block_size;
    uint8_t *row = (is_v ? a.pool.v : a.pool.k) + blk * a.pool.sb + off * a.pool.st +
                   hk * a.pool.sh + l8 * 8;
    *reinterpret_cast<uint2 *>(row) = make_uint2(o[0], o[1]);
    *reinterpret_cast<uint2 *>(row + 64) = make_uint2(o[2], o[3]);
    if (l8 == 0) {
      uint8_t *s = (is_v ? a.pool.vs : a.pool.ks) + blk * a.pool.ssb + hk * a.pool.ssh + off;
      *s = bad ? 255 : static_cast<uint8_t>(e + 127);
    }
  }
}

// ---------------------------------------------------------------------------
// Read-back. 16 lanes own a row (8 elements each): one 128-byte load and one
// 256-byte store per row, both coalesced.
// ---------------------------------------------------------------------------
struct ReadArgs {
  Pool pool;
  const int32_t *bt, *lens;
  __nv_bfloat16 *k_out, *v_out;
  int max_len, zero_to, Hkv, bt_stride, max_tokens;   // max_tokens = bt_width * block_size
};

constexpr int kReadThreads = 256;
constexpr int kReadTok = 16;   // tokens of one CTA (within one block)

template <bool kInt8>
__global__ void __launch_bounds__(kReadThreads) kv_read_quantized_kernel(const ReadArgs a) {
  const int b = blockIdx.y;
  const int t0 = blockIdx.x * kReadTok;
  const int len = min(min(__ldg(a.lens + b), a.max_tokens), a.max_len);
  int end = a.max_len;          // rows [len, end) are zeroed
  if (a.zero_to > 0) {
    const int64_t up = (static_cast<int64_t>(max(len, 1)) + a.zero_to - 1) / a.zero_to * a.zero_to;
    if (up < end) end = static_cast<int>(up);
  }
  const int nt = min(kReadTok, end - t0);
  if (nt <= 0) return;
  int64_t blk = 0;
  if (t0 < len) {
    blk = __ldg(a.bt + static_cast<int64_t>(b) * a.bt_stride + t0 / a.pool.block_size);
    if (blk < 0 || blk >= a.pool.num_blocks) blk = 0;
  }
  const int off0 = t0 % a.pool.block_size;
  const int l16 = threadIdx.x & 15;
  const int rows = nt * a.Hkv;
  for (int r = threadIdx.x >> 4; r < 2 * rows; r += kReadThreads / 16) {
    const bool is_v = r >= rows;
    const int i = is_v ? r - rows : r;
    const int tt = i / a.Hkv, h = i % a.Hkv;
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (t0 + tt < len) {
      const int64_t off = off0 + tt;
      const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(
          (is_v ? a.pool.v : a.pool.k) + blk * a.pool.sb + off * a.pool.st + h * a.pool.sh +
          l16 * 8));
      const float s = scale_of(__ldg((is_v ? a.pool.vs : a.pool.ks) + blk * a.pool.ssb +
                                     h * a.pool.ssh + off));
      const float2 f0 = f16x2_to_f32(dequant_f16x2<kInt8, false>(w.x));
      const float2 f1 = f16x2_to_f32(dequant_f16x2<kInt8, true>(w.x));
      const float2 f2 = f16x2_to_f32(dequant_f16x2<kInt8, false>(w.y));
      const float2 f3 = f16x2_to_f32(dequant_f16x2<kInt8, true>(w.y));
      o = make_uint4(cvt_bf16x2(f0.x * s, f0.y * s), cvt_bf16x2(f1.x * s, f1.y * s),
                     cvt_bf16x2(f2.x * s, f2.y * s), cvt_bf16x2(f3.x * s, f3.y * s));
    }
    __nv_bfloat16 *dst = (is_v ? a.v_out : a.k_out) +
                         ((static_cast<int64_t>(b) * a.max_len + t0 + tt) * a.Hkv + h) * kD;
    *reinterpret_cast<uint4 *>(dst + l16 * 8) = o;
  }
}

}  // namespace
}  // namespace vj

extern "C" vj_status vj_kv_store_quantized(
    const void *q_in, const void *k_in, const void *v_in, const void *q_norm_w,
    const void *k_norm_w, const int32_t *positions, const int32_t *slot_mapping, void *q_out,
    void *k_cache, void *v_cache, void *k_scales, void *v_scales, int32_t cache_dtype,
    int64_t num_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int64_t num_blocks, int32_t block_size, int64_t stride_block, int64_t stride_token,
    int64_t stride_head, int64_t scale_stride_block, int64_t scale_stride_head,
    int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride, int64_t q_out_row_stride,
    const void *rope_table, int32_t rope_table_len, double eps, float rope_theta, int32_t flags,
    cudaStream_t stream) {
  using namespace vj;
  const char *what = "vj_kv_store_quantized";
  StoreArgs a;
  a.pool = {static_cast<uint8_t *>(k_cache), static_cast<uint8_t *>(v_cache),
            static_cast<uint8_t *>(k_scales), static_cast<uint8_t *>(v_scales),
            stride_block, stride_token, stride_head, scale_stride_block, scale_stride_head,
            num_blocks, block_size};
  int rc = check_pool(what, a.pool, cache_dtype, num_kv_heads, head_dim);
  if (rc) return rc;
  if (num_tokens < 0 || num_q_heads < 0 || rope_table_len < 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, std::string(what) + ": negative size");
  }
  const int64_t heads = static_cast<int64_t>(num_q_heads) + 2ll * num_kv_heads;
  if (heads > 4096) {
    return set_error(VJ_ERR_UNSUPPORTED, std::string(what) + ": more than 4096 head rows");
  }
  if (flags & ~(VJ_KV_NORM | VJ_KV_ROPE)) {
    return set_error(VJ_ERR_INVALID_ARGUMENT,
                     std::string(what) + ": flags other than VJ_KV_NORM and VJ_KV_ROPE");
  }
  if (num_tokens == 0) return VJ_OK;
  rc = check_pool_memory(what, a.pool);
  if (rc) return rc;
  if (!k_in || !v_in || !slot_mapping || (num_q_heads > 0 && (!q_in || !q_out))) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, std::string(what) + ": null pointer");
  }
  a.norm = (flags & VJ_KV_NORM) != 0;
  a.rope = (flags & VJ_KV_ROPE) != 0;
  if (a.norm && ((num_q_heads > 0 && !q_norm_w) || !k_norm_w)) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, std::string(what) + ": VJ_KV_NORM needs norm weights");
  }
  if (a.rope && !positions) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, std::string(what) + ": VJ_KV_ROPE needs positions");
  }
  if (rope_table_len > 0 &&
      (rope_table == nullptr || reinterpret_cast<uintptr_t>(rope_table) % 16 != 0)) {
    return set_error(VJ_ERR_INVALID_ARGUMENT,
                     std::string(what) + ": rope_table must be 16-byte aligned");
  }
  a.qrs = q_row_stride ? q_row_stride : static_cast<int64_t>(num_q_heads) * kD;
  a.krs = k_row_stride ? k_row_stride : static_cast<int64_t>(num_kv_heads) * kD;
  a.vrs = v_row_stride ? v_row_stride : static_cast<int64_t>(num_kv_heads) * kD;
  a.qors = q_out_row_stride ? q_out_row_stride : static_cast<int64_t>(num_q_heads) * kD;
  uintptr_t bases = reinterpret_cast<uintptr_t>(k_in) | reinterpret_cast<uintptr_t>(v_in);
  int64_t strides = a.krs | a.vrs;
  if (num_q_heads > 0) {
    bases |= reinterpret_cast<uintptr_t>(q_in) | reinterpret_cast<uintptr_t>(q_out);
    strides |= a.qrs | a.qors;
  }
  if (a.norm) {
    bases |= reinterpret_cast<uintptr_t>(k_norm_w);
    if (num_q_heads > 0) bases |= reinterpret_cast<uintptr_t>(q_norm_w);
  }
  if (bases % 16 != 0 || strides % 8 != 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT,
                     std::string(what) + ": q/k/v rows and weights must start on 16-byte "
                                         "boundaries");
  }
  a.q = static_cast<const __nv_bfloat16 *>(q_in);
  a.k = static_cast<const __nv_bfloat16 *>(k_in);
  a.v = static_cast<const __nv_bfloat16 *>(v_in);
  a.qw = static_cast<const __nv_bfloat16 *>(q_norm_w);
  a.kw = static_cast<const __nv_bfloat16 *>(k_norm_w);
  a.positions = positions;
  a.slots = slot_mapping;
  a.q_out = static_cast<__nv_bfloat16 *>(q_out);
  a.table = static_cast<const uint4 *>(rope_table);
  a.table_len = rope_table_len;
  a.heads = static_cast<uint32_t>(heads);
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.eps = eps;
  build_rope_table(rope_theta, a.freq.inv_freq);
  // row indices of a launch stay below 2^31 (grid-stride steps cannot wrap)
  const int64_t per_launch = (int64_t(1) << 30) / heads;
  const int64_t cap = static_cast<int64_t>(num_sms()) * 8;
  for (int64_t t0 = 0; t0 < num_tokens; t0 += per_launch) {
    a.t_begin = t0;
    a.num_rows = static_cast<uint32_t>(std::min(per_launch, num_tokens - t0) * heads);
    const unsigned grid = static_cast<unsigned>(
        std::min<int64_t>((a.num_rows + kStoreThreads / 8 - 1) / (kStoreThreads / 8), cap));
    if (cache_dtype == VJ_CACHE_INT8) {
      kv_store_quantized_kernel<true><<<grid, kStoreThreads, 0, stream>>>(a);
    } else {
      kv_store_quantized_kernel<false><<<grid, kStoreThreads, 0, stream>>>(a);
    }
    rc = check_launch(what);
    if (rc) return rc;
  }
  return VJ_OK;
}

extern "C" vj_status vj_kv_read_quantized(
    const void *k_cache, const void *v_cache, const void *k_scales, const void *v_scales,
    int32_t cache_dtype, const int32_t *block_tables, const int32_t *context_lens, void *k_out,
    void *v_out, int32_t batch, int32_t max_len, int32_t zero_to, int32_t num_kv_heads,
    int32_t head_dim, int64_t num_blocks, int32_t block_size, int32_t bt_width,
    int32_t bt_stride, int64_t stride_block, int64_t stride_token, int64_t stride_head,
    int64_t scale_stride_block, int64_t scale_stride_head, cudaStream_t stream) {
  using namespace vj;
  const char *what = "vj_kv_read_quantized";
  ReadArgs a;
  a.pool = {static_cast<uint8_t *>(const_cast<void *>(k_cache)),
            static_cast<uint8_t *>(const_cast<void *>(v_cache)),
            static_cast<uint8_t *>(const_cast<void *>(k_scales)),
            static_cast<uint8_t *>(const_cast<void *>(v_scales)),
            stride_block, stride_token, stride_head, scale_stride_block, scale_stride_head,
            num_blocks, block_size};
  int rc = check_pool(what, a.pool, cache_dtype, num_kv_heads, head_dim);
  if (rc) return rc;
  if (batch < 0 || max_len < 0 || zero_to < 0 || bt_width < 0 || bt_stride < bt_width) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, std::string(what) + ": negative size");
  }
  if (batch > 65535) {
    return set_error(VJ_ERR_UNSUPPORTED, std::string(what) + ": more than 65535 sequences");
  }
  if (num_kv_heads > 4096) {
    return set_error(VJ_ERR_UNSUPPORTED, std::string(what) + ": more than 4096 KV heads");
  }
  if (batch == 0 || max_len == 0) return VJ_OK;
  rc = check_pool_memory(what, a.pool);
  if (rc) return rc;
  if (!context_lens || !k_out || !v_out || (bt_width > 0 && !block_tables)) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, std::string(what) + ": null pointer");
  }
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16 != 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT,
                     std::string(what) + ": outputs must be 16-byte aligned");
  }
  a.bt = block_tables;
  a.lens = context_lens;
  a.k_out = static_cast<__nv_bfloat16 *>(k_out);
  a.v_out = static_cast<__nv_bfloat16 *>(v_out);
  a.max_len = max_len;
  a.zero_to = zero_to;
  a.Hkv = num_kv_heads;
  a.bt_stride = bt_stride;
  a.max_tokens = static_cast<int>(
      std::min<int64_t>(static_cast<int64_t>(bt_width) * block_size, INT32_MAX));
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(max_len) + kReadTok - 1) / kReadTok),
                  static_cast<unsigned>(batch));
  if (cache_dtype == VJ_CACHE_INT8) {
    kv_read_quantized_kernel<true><<<grid, kReadThreads, 0, stream>>>(a);
  } else {
    kv_read_quantized_kernel<false><<<grid, kReadThreads, 0, stream>>>(a);
  }
  return check_launch(what);
}
