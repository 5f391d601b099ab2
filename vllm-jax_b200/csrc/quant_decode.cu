// Attention of one new token per sequence over the quantised paged KV cache.
//
//   s_t = scale * q . k_t,  p = softmax(s),  o = sum_t p_t v_t,  t < context
//
// One CTA per (sequence, KV head): its warps take the context's tokens in
// turn, each with a running maximum, sum and output for every query head of
// the group (32 bits), merged at the end.
#include "quant.cuh"

#include <algorithm>
#include <cmath>

namespace vj {
namespace {
using namespace qn;

struct QDecodeArgs {
  Pool pool;
  const __nv_bfloat16 *q;
  __nv_bfloat16 *out;
  const int32_t *bt, *lens;
  int B, Hq, Hkv, g, bt_stride, max_tokens;
  float scale_log2;
};

constexpr int kWarps = 8;

template <bool kInt8>
VJ_DEV float4 load4(const uint8_t *p, float s) {
  const uint32_t w = *reinterpret_cast<const uint32_t *>(p);
  const float2 a = f16x2_to_f32(dequant_f16x2<kInt8, false>(w));
  const float2 b = f16x2_to_f32(dequant_f16x2<kInt8, true>(w));
  return make_float4(a.x * s, a.y * s, b.x * s, b.y * s);
}

template <bool kInt8, int G>
__global__ void __launch_bounds__(kWarps * 32) quant_decode_kernel(const QDecodeArgs a) {
  __shared__ float red_m[kWarps][G], red_l[kWarps][G];
  __shared__ float4 red_o[kWarps][32];
  const int b = blockIdx.x / a.Hkv, h = blockIdx.x % a.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = min(__ldg(a.lens + b), a.max_tokens);
  float4 q[G], o[G];
  float m[G], l[G];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    q[i] = o[i];
    m[i] = -INFINITY;
    l[i] = 0.f;
    if (i < a.g) {
      const uint2 w = *reinterpret_cast<const uint2 *>(
          a.q + (static_cast<int64_t>(b) * a.Hq + h * a.g + i) * kD + lane * 4);
      q[i] = make_float4(bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y));
    }
  }
  for (int t = warp; t < len; t += kWarps) {
    int64_t blk = __ldg(a.bt + static_cast<int64_t>(b) * a.bt_stride + t / a.pool.block_size);
    if (blk < 0 || blk >= a.pool.num_blocks) blk = 0;
    const int64_t off = t % a.pool.block_size;
    const int64_t at = blk * a.pool.sb + off * a.pool.st + h * a.pool.sh + lane * 4;
    const int64_t sat = blk * a.pool.ssb + h * a.pool.ssh + off;
    const float4 k = load4<kInt8>(a.pool.k + at, scale_of(a.pool.ks[sat]));
    const float4 v = load4<kInt8>(a.pool.v + at, scale_of(a.pool.vs[sat]));
#pragma unroll
    for (int i = 0; i < G; ++i) {
      float s = k.x * q[i].x + k.y * q[i].y + k.z * q[i].z + k.w * q[i].w;
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      s *= a.scale_log2;
      const float mn = fmaxf(m[i], s);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float c = exp2f(m[i] - mu), p = exp2f(s - mu);
      m[i] = mn;
      l[i] = l[i] * c + p;
      o[i].x = o[i].x * c + p * v.x;
      o[i].y = o[i].y * c + p * v.y;
      o[i].z = o[i].z * c + p * v.z;
      o[i].w = o[i].w * c + p * v.w;
    }
  }
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < G; ++i) { red_m[warp][i] = m[i]; red_l[warp][i] = l[i]; }
  }
#pragma unroll
  for (int i = 0; i < G; ++i) {
    if (i >= a.g) break;
    __syncthreads();
    red_o[warp][lane] = o[i];
    __syncthreads();
    if (warp != 0) continue;
    float mt = -INFINITY;
    for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, red_m[w][i]);
    const float mu = mt == -INFINITY ? 0.f : mt;
    float lt = 0.f;
    float4 ot = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < kWarps; ++w) {
      const float c = exp2f(red_m[w][i] - mu);
      lt += red_l[w][i] * c;
      const float4 x = red_o[w][lane];
      ot.x += x.x * c; ot.y += x.y * c; ot.z += x.z * c; ot.w += x.w * c;
    }
    const float inv = len > 0 ? 1.f / lt : 0.f;
    *reinterpret_cast<uint2 *>(a.out + (static_cast<int64_t>(b) * a.Hq + h * a.g + i) * kD +
                               lane * 4) =
        make_uint2(pack_bf16(ot.x * inv, ot.y * inv), pack_bf16(ot.z * inv, ot.w * inv));
  }
}

}  // namespace
}  // namespace vj

extern "C" size_t vj_paged_decode_quantized_workspace_size(int32_t batch, int32_t num_q_heads,
                                                           int32_t num_kv_heads,
                                                           int32_t head_dim) {
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim != vj::kD) return 0;
  return 256;
}

extern "C" vj_status vj_paged_decode_quantized(
    const void *q, const void *k_cache, const void *v_cache, const void *k_scales,
    const void *v_scales, int32_t cache_dtype, const int32_t *block_tables,
    const int32_t *context_lens, void *out, int32_t batch, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, int64_t num_blocks, int32_t block_size,
    int32_t bt_width, int32_t bt_stride, int64_t stride_block, int64_t stride_token,
    int64_t stride_head, int64_t scale_stride_block, int64_t scale_stride_head, float scale,
    void *workspace, size_t workspace_bytes, int32_t *error_flag, cudaStream_t stream) {
  using namespace vj;
  const std::string what = "vj_paged_decode_quantized";
  QDecodeArgs a;
  a.pool = {static_cast<uint8_t *>(const_cast<void *>(k_cache)),
            static_cast<uint8_t *>(const_cast<void *>(v_cache)),
            static_cast<uint8_t *>(const_cast<void *>(k_scales)),
            static_cast<uint8_t *>(const_cast<void *>(v_scales)),
            stride_block, stride_token, stride_head, scale_stride_block, scale_stride_head,
            num_blocks, block_size};
  int rc = check_pool(what, a.pool, cache_dtype, num_kv_heads, head_dim);
  if (rc) return rc;
  if (batch < 0 || num_q_heads <= 0 || bt_width < 0 || bt_stride < bt_width) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": negative or zero size");
  }
  if (num_q_heads % num_kv_heads != 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT,
                     what + ": Number of Q heads must be divisible by number of KV heads. Got " +
                         std::to_string(num_q_heads) + " and " + std::to_string(num_kv_heads) + ".");
  }
  if (num_q_heads / num_kv_heads > 16) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": at most 16 query heads per KV head");
  }
  if (num_kv_heads > 1024) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": at most 1024 KV heads");
  }
  if (stride_block != block_size * stride_token) {
    return set_error(VJ_ERR_UNSUPPORTED,
                     what + ": tokens of a block must be evenly strided (stride_block == "
                            "block_size * stride_token)");
  }
  if (batch == 0) return VJ_OK;
  rc = check_pool_memory(what, a.pool);
  if (rc) return rc;
  if (!q || !context_lens || !out || (bt_width > 0 && !block_tables)) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": null pointer");
  }
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 != 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": q and out must be 16-byte aligned");
  }
  const size_t need =
      vj_paged_decode_quantized_workspace_size(batch, num_q_heads, num_kv_heads, head_dim);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
    return set_error(VJ_ERR_WORKSPACE, what + ": workspace needs " + std::to_string(need) +
                                           " bytes, 16-byte aligned");
  }
  (void)error_flag;
  a.q = static_cast<const __nv_bfloat16 *>(q);
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.bt = block_tables;
  a.lens = context_lens;
  a.B = batch;
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.g = num_q_heads / num_kv_heads;
  a.bt_stride = bt_stride;
  a.max_tokens = static_cast<int>(
      std::min<int64_t>(static_cast<int64_t>(bt_width) * block_size, INT32_MAX));
  a.scale_log2 = scale * 1.4426950408889634f;
  if (static_cast<int64_t>(batch) * num_kv_heads > INT32_MAX) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": batch too large");
  }
  const unsigned grid = static_cast<unsigned>(batch) * num_kv_heads;
  const bool i8 = cache_dtype == VJ_CACHE_INT8;
  if (a.g <= 8) {
    if (i8) quant_decode_kernel<true, 8><<<grid, kWarps * 32, 0, stream>>>(a);
    else quant_decode_kernel<false, 8><<<grid, kWarps * 32, 0, stream>>>(a);
  } else {
    if (i8) quant_decode_kernel<true, 16><<<grid, kWarps * 32, 0, stream>>>(a);
    else quant_decode_kernel<false, 16><<<grid, kWarps * 32, 0, stream>>>(a);
  }
  return check_launch("vj_paged_decode_quantized");
}
