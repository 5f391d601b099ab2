// Prefill attention whose keys are split over CTAs: what the parts leave, and the
// kernel that joins them. Args has out, cu, num_seqs, num_tokens, Hq, parts, keep_tail
// (rows past the last sequence stay as they are), part_rows, part_o ([parts]
// [part_rows][Hq][128] sums in 32 bits, not normalised) and part_ml ([parts][part_rows]
// [Hq] maximum (log2) and sum of the weights). Row 0 of the parts is token cu[0].
#pragma once

#include "vj_common.cuh"

#include <algorithm>
#include <cstdint>

namespace vj {
namespace {

// Whether two buffers of this many bytes overlap without being the same: a tile reads
// its own rows of q alone before it writes them, so out may be q, but not lie across it.
inline bool overlap_in_part(const void *x, const void *y, int64_t bytes) {
  const auto p = reinterpret_cast<uintptr_t>(x), r = reinterpret_cast<uintptr_t>(y);
  return p != r && (p < r ? r - p : p - r) < static_cast<uint64_t>(bytes);
}

// Rows of the parts: the call's sequences hold no more tokens. (With those of the whole
// batch, a call for one of its many sequences took gigabytes.)
inline int64_t rows_of_parts(int64_t num_tokens, int64_t num_seqs, int64_t longest) {
  return std::min(num_tokens, num_seqs * longest);
}
// The row of a token in a part, or a negative number where the bound on the new tokens
// that sizes the parts does not hold.
template <class Args>
VJ_DEV int64_t row_of_part(const Args &a, int first, int token) {
  const int rel = token - first;
  return rel >= 0 && rel < a.part_rows ? rel : -1;
}
template <class Args>
VJ_DEV int64_t place_in_parts(const Args &a, int part, int64_t rel, int head) {
  return (part * static_cast<int64_t>(a.part_rows) + rel) * a.Hq + head;
}

constexpr float kLowest = -1e30f;       // a maximum that no key has moved yet

// This CTA's share of the rows past cu_seqlens_q[num_seqs] -> 0, by n of its threads.
template <class Args>
VJ_DEV void zero_tail_share(const Args &a, int i, int n) {
  const int64_t per_row = static_cast<int64_t>(a.Hq) * 16, from = a.cu[a.num_seqs] * per_row;
  const int64_t tail = a.num_tokens * per_row - from;
  if (tail <= 0) return;
  const int64_t cta = (static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  const int64_t ctas = static_cast<int64_t>(gridDim.x) * gridDim.y * gridDim.z;
  uint4 *o = reinterpret_cast<uint4 *>(a.out) + from;
  for (int64_t k = tail * cta / ctas + i; k < tail * (cta + 1) / ctas; k += n) {
    o[k] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// Joins the parts of the rows [cu[0], cu[num_seqs]) and zeroes those behind (unless
// they are kept). kWarps warps take a (token, query head), each every kWarps-th part,
// four of them in flight.
constexpr int kJoinWarps = 8;
template <int kWarps, class Args>
__global__ void __launch_bounds__(kJoinWarps * 32)
prefill_join_kernel(const Args a) {
  __shared__ float4 so[kJoinWarps][32];
  __shared__ float2 sml[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = warp % kWarps;
  const int64_t rows = static_cast<int64_t>(a.part_rows) * a.Hq;
  const int64_t rel = static_cast<int64_t>(blockIdx.x) * (kJoinWarps / kWarps) + warp / kWarps;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t first = static_cast<int64_t>(a.cu[0]) * a.Hq;
  const int64_t end = min(a.cu[a.num_seqs], a.num_tokens) * static_cast<int64_t>(a.Hq);
  const int64_t row = first + rel;
  uint2 *dst = reinterpret_cast<uint2 *>(a.out + row * 128) + lane;
  const bool mine = rel < rows && row < end;
  if (!a.keep_tail) zero_tail_share(a, threadIdx.x, kJoinWarps * 32);
  float m = kLowest, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float2 ml, float4 x) {
    if (ml.y == 0.f) return;            // no key of the part: its sums may not be there
    const float top = fmaxf(m, ml.x), f0 = exp2f(m - top), f1 = exp2f(ml.x - top);
    m = top;
    l = fmaf(ml.y, f1, l * f0);
    o.x = fmaf(x.x, f1, o.x * f0); o.y = fmaf(x.y, f1, o.y * f0);
    o.z = fmaf(x.z, f1, o.z * f0); o.w = fmaf(x.w, f1, o.w * f0);
  };
  if (mine) {
    constexpr int kFly = 4;
    for (int i0 = w; i0 < a.parts; i0 += kFly * kWarps) {
      float2 ml[kFly];
      float4 x[kFly];
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        const int i = i0 + k * kWarps;
        ml[k] = make_float2(kLowest, 0.f);
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < a.parts) {
          const int64_t at = i * rows + rel;
          ml[k] = a.part_ml[at];
          x[k] = reinterpret_cast<const float4 *>(a.part_o + at * 128)[lane];
        }
      }
#pragma unroll
      for (int k = 0; k < kFly; ++k) add(ml[k], x[k]);
    }
  }
  if constexpr (kWarps > 1) {
    so[warp][lane] = o;
    if (lane == 0) sml[warp] = make_float2(m, l);
    __syncthreads();
    if (w != 0) return;
    for (int k = 1; k < kWarps; ++k) add(sml[warp + k], so[warp + k][lane]);
  }
  if (!mine) return;
  const float inv = 1.f / l;
  *dst = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
}

template <class Args>
int launch_join(const char *what, const Args &a, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.part_rows) * a.Hq;
  const bool few = rows <= 8 * num_sms();       // eight warps each
  const int64_t blocks = few ? rows : (rows + kJoinWarps - 1) / kJoinWarps;
  return launch_dependent(what, few ? prefill_join_kernel<kJoinWarps, Args> : prefill_join_kernel<1, Args>,
                          dim3(static_cast<unsigned>(blocks)), kJoinWarps * 32, 0, stream, a);
}

}  // namespace
}  // namespace vj
