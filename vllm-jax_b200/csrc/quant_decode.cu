// Attention of one new token per sequence over the quantised paged KV cache.
//
//   s_t = scale * q . k_t,  p = softmax(s),  o = sum_t p_t v_t,  t < context
//
// HBM-bound: every cached row is read once (129 bytes a row, K and V), for all
// query heads of its KV head together.
//
// The work is cut into pages of 16 tokens. All sequences' pages in a row,
// numbered 0..T-1, are split evenly over groups of Hkv warps; the warps of a
// group walk the same pages, each for its own KV head, so a page's rows (which
// lie side by side) are read at about the same time. Every CTA finds its
// warps' ranges from the context lengths by itself, so there is no planning
// launch, no work counter and nothing to reset between calls. A sequence whose
// pages fall to one group is finished there; otherwise each group leaves a
// partial result (its output in 32 bits, maximum and sum), at most two per
// warp, and quant_combine_kernel joins them.
//
// A warp streams its pages through a ring of its own in shared memory (TMA
// boxes of 16 rows x 128 bytes, 128-byte swizzle, and the rows' scale bytes).
// Products run on mma.sync m16n8k16 in f16 with 32-bit sums, with the tokens,
// then the dimensions, as the 16 rows and the query heads of the group as the 8
// columns:
//   S^T[tok][head] = K[tok][d] Q^T[d][head]     (8 steps of 16 dims)
//   O^T[d][head]  += V^T[d][tok] W^T[tok][head]  (8 tiles of 16 dims)
// The elements of both types are exact in f16. Which 16 dims make a step is
// free as long as q agrees, and which dims make a tile of O too, so a lane
// takes 32 consecutive bytes of a K row and 16 of a V row with 16-byte loads,
// and V^T needs only bytes of neighbouring tokens interleaved before the
// conversion: no transposing loads.
//   q is brought to [1, 2) by a power of two per head before it is rounded to
// f16 (8 significant bits fit; what falls below f16's range is 2^-24 of the
// head's largest element or less).
//   The row scales of K multiply the scores. Those of V are put into the
// weights, w_t = p_t * 2^(ev_t), against a running maximum of their own, so
// that rows of any scale keep 11 bits; the sum of p stays in 32 bits.
// The running maxima only move when a score passes them by 2^11 (a vote per
// page instead of shuffles and rescaling): weights are kept 2^4 up in f16, so
// they stay below 2^15, and one 2^-28 of the maximum is still a number.
#include "quant.cuh"

#include <algorithm>
#include <cmath>

namespace vj {
namespace {
using namespace qn;

constexpr int kTok = 16;                      // tokens per page
constexpr int kHalf = kTok * kD;              // bytes of a page's K (or V) rows
constexpr int kStage = 2 * kHalf;
constexpr int kMinPages = 4;                  // pages of a group, at least
constexpr float kSlack = 11.0f;               // log2 of what a score may pass the maximum by
constexpr float kUp = 4.0f;                   // log2 of the weight at the maximum

template <int NT>
struct Shape {                                // NT tiles of 8 query heads
  static constexpr int kWarps = NT == 1 ? 16 : 8;
  static constexpr int kStages = NT == 1 ? 3 : 6;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRing = kWarps * kStages;
  // pages, scale bytes, page infos, barriers, scan
  static constexpr size_t kSmem =
      1024 + (size_t)kRing * (kStage + 32 + 16 + 8) + (kThreads + 1 + kWarps) * 4;
};

struct Scratch {
  int32_t *prefix;    // [B + 1] first page of each sequence
  float2 *ml;         // [2 * groups][Hq] maximum (log2), sum
  float *o;           // [2 * groups][Hq][128]
};

inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

inline size_t scratch_bytes(int64_t B, int64_t Hq, int64_t groups) {
  return up256(4 * (B + 1)) + up256(2 * groups * Hq * sizeof(float2)) +
         2 * groups * Hq * kD * sizeof(float);
}

struct QDecodeArgs {
  const __nv_bfloat16 *q;
  __nv_bfloat16 *out;
  const int32_t *bt, *lens;
  const uint8_t *ks, *vs;
  int64_t ssb, ssh;
  int B, Hq, Hkv, g, bt_stride, pages_per_block, block_size, max_pages, num_blocks, head_major;
  int groups;         // warps of the grid / Hkv
  float scale_log2;
  Scratch ws;
  int32_t *err;
};

// Groups in use, and the page range of group G: [first(G), first(G + 1)).
VJ_DEV int groups_of(int total, int groups) {
  return min(groups, (total + kMinPages - 1) / kMinPages);
}
VJ_DEV int first_page(int G, int total, int n) {
  return static_cast<int>(static_cast<int64_t>(G) * total / n);
}
VJ_DEV int group_of(int page, int total, int n) {
  return static_cast<int>((static_cast<int64_t>(page + 1) * n - 1) / total);
}

VJ_DEV int pages_of(int len, int max_pages) {
  const int p = len > 0 ? (len - 1) / kTok + 1 : 0;
  return min(p, max_pages);
}

VJ_DEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                    uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
VJ_DEV uint32_t transpose8x8(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
VJ_DEV uint32_t pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
VJ_DEV uint32_t bytes(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}
VJ_DEV uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}
VJ_DEV float max3_over_rows(float v) {        // over the lanes that share lane & 3
#pragma unroll
  for (int o = 4; o <= 16; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The pages of a warp's range in order. Every lane holds the same state but
// the two windows: 32 sequences' lengths, and 32 entries of the current
// sequence's block table.
struct Walk {
  int base, len_w;        // window: lane i has sequence base + i
  int b, p, np;           // current sequence, next page, its pages
  int left;               // pages left in the range
  int start;              // first page of the current segment
  int entry, blk_w;       // table window: lane i has entry + i
};

VJ_DEV int walk_len(const QDecodeArgs &a, int base, int lane) {
  return base + lane < a.B ? __ldg(a.lens + base + lane) : 0;
}
VJ_DEV void walk_enter(Walk &w, const QDecodeArgs &a, int b, int p) {
  w.b = b;
  w.p = w.start = p;
  w.np = pages_of(__shfl_sync(0xffffffffu, w.len_w, b - w.base), a.max_pages);
  w.entry = -64;
}
// Next sequence that has pages; there is one while pages are left.
VJ_DEV void walk_next(Walk &w, const QDecodeArgs &a, int lane) {
  int from = w.b + 1 - w.base;
  while (true) {
    const unsigned have = __ballot_sync(
        0xffffffffu, lane >= from && pages_of(w.len_w, a.max_pages) > 0);
    if (have) {
      walk_enter(w, a, w.base + __ffs(have) - 1, 0);
      return;
    }
    w.base += 32;
    if (w.base >= a.B) { w.left = 0; return; }
    w.len_w = walk_len(a, w.base, lane);
    from = 0;
  }
}

// What a stage holds. flags: 1 first page of its segment, 2 last page of its
// segment, 4 the segment starts at the sequence's first page, 8 it ends at
// its last one.
struct PageInfo {
  int b, page, len, flags;
};

template <bool kInt8, int NT>
__global__ void __launch_bounds__(Shape<NT>::kThreads, 1)
quant_decode_kernel(const __grid_constant__ CUtensorMap tmk,
                    const __grid_constant__ CUtensorMap tmv, const QDecodeArgs a) {
  using S = Shape<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t *scales = smem + S::kRing * kStage;
  PageInfo *infos = reinterpret_cast<PageInfo *>(scales + S::kRing * 32);
  uint64_t *bars = reinterpret_cast<uint64_t *>(infos + S::kRing);
  int *scan = reinterpret_cast<int *>(bars + S::kRing);       // [kThreads + 1]
  int *warp_sum = scan + S::kThreads + 1;                     // [kWarps]

  // ---- pages before each run of `per` sequences
  const int per = (a.B + S::kThreads - 1) / S::kThreads;
  int mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < a.B) mine += pages_of(__ldg(a.lens + b), a.max_pages);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  if (lane == 0) {
    for (int s = 0; s < S::kStages; ++s) mbar_init(&bars[warp * S::kStages + s], 1);
    fence_mbar_init();
  }
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < S::kWarps; ++w) {
    const int v = warp_sum[w];
    before += w < warp ? v : 0;
    total += v;
  }
  scan[tid] = before + incl - mine;
  __syncthreads();
  if (blockIdx.x == 0) {                      // for the combine kernel
    int run = scan[tid];
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      if (b >= a.B) break;
      a.ws.prefix[b] = run;
      run += pages_of(__ldg(a.lens + b), a.max_pages);
    }
    if (tid == 0) a.ws.prefix[a.B] = total;
  }

  // ---- this warp's KV head and pages
  const int id = warp * gridDim.x + blockIdx.x;
  const int G = id / a.Hkv, h = id - G * a.Hkv;
  const int n_groups = groups_of(total, a.groups);
  if (G >= n_groups) return;
  const int s0 = first_page(G, total, n_groups);
  Walk w;
  w.left = first_page(G + 1, total, n_groups) - s0;
  const int n_pages = w.left;
  {
    int lo = 0;                               // last run that starts at or before s0
#pragma unroll
    for (int step = S::kThreads / 2; step >= 1; step >>= 1) {
      if (scan[lo + step] <= s0) lo += step;
    }
    int cum = scan[lo];
    w.base = lo * per;
    while (true) {
      w.len_w = walk_len(a, w.base, lane);
      const int pg = pages_of(w.len_w, a.max_pages);
      int in = pg;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, cum + in > s0);
      if (past) {
        const int i = __ffs(past) - 1;
        walk_enter(w, a, w.base + i, s0 - cum - __shfl_sync(0xffffffffu, in - pg, i));
        break;
      }
      cum += __shfl_sync(0xffffffffu, in, 31);
      w.base += 32;
      if (w.base >= a.B) return;              // cannot happen: s0 < total
    }
  }

  uint8_t *ring = smem + warp * S::kStages * kStage;
  uint8_t *sc_ring = scales + warp * S::kStages * 32;
  PageInfo *info = infos + warp * S::kStages;
  uint64_t *full = bars + warp * S::kStages;

  // issue the walk's next page into stage s
  auto produce = [&](int s) {
    if (w.left == 0) return;
    const int e = w.p / a.pages_per_block;
    if (e >= w.entry + 32 || e < w.entry) {
      w.entry = e;
      const int last = (w.np - 1) / a.pages_per_block;
      int blk = __ldg(a.bt + static_cast<int64_t>(w.b) * a.bt_stride + min(e + lane, last));
      w.blk_w = blk < 0 || blk >= a.num_blocks ? 0 : blk;
    }
    const int blk = __shfl_sync(0xffffffffu, w.blk_w, e - w.entry);
    const int len = __shfl_sync(0xffffffffu, w.len_w, w.b - w.base);
    if (lane == 0) {
      const int off = (w.p - e * a.pages_per_block) * kTok;
      const int flags = (w.p == w.start ? 1 : 0) | (w.p + 1 == w.np || w.left == 1 ? 2 : 0) |
                        (w.start == 0 ? 4 : 0) | (w.p + 1 == w.np ? 8 : 0);
      info[s] = {w.b, w.p, len, flags};
      uint8_t *dst = ring + s * kStage;
      mbar_arrive_expect_tx(&full[s], kStage + 32);
      const int tok = blk * a.block_size + off;
      const int c1 = a.head_major ? h : tok, c2 = a.head_major ? tok : h;
      tma_load_3d(dst, &tmk, &full[s], 0, c1, c2);
      tma_load_3d(dst + kHalf, &tmv, &full[s], 0, c1, c2);
      const int64_t so = blk * a.ssb + h * a.ssh + off;
      bulk_g2s(sc_ring + s * 32, a.ks + so, 16, &full[s]);
      bulk_g2s(sc_ring + s * 32 + 16, a.vs + so, 16, &full[s]);
    }
    ++w.p;
    --w.left;
    if (w.left > 0 && w.p == w.np) walk_next(w, a, lane);
  };
#pragma unroll
  for (int s = 0; s < S::kStages; ++s) produce(s);

  const int r = lane >> 2, qd = lane & 3;
  uint32_t qf[NT][16];                  // Q^T fragments: dims 32*qd + 4*j + {0,1}, {2,3}
  float qs[NT][2];                      // score factor of heads 2*qd, 2*qd + 1
  float acc[NT][8][4];                  // O^T: dims 16*r + 2*i, + 1; heads 2*qd, 2*qd + 1
  float m[NT][2], mw[NT][2], l[NT][2];  // log2: maximum of s, of s + ev; sum of p
  bool fail = false;
  int it = 0;
  for (; it < n_pages; ++it) {
    const int s = it % S::kStages;
    if (!mbar_wait(&full[s], (it / S::kStages) & 1)) { fail = true; break; }
    const PageInfo pi = info[s];
    if (pi.flags & 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int head = t * 8 + r;
        uint4 x[4] = {};
        if (head < a.g) {
          const uint4 *row = reinterpret_cast<const uint4 *>(
              a.q + (static_cast<int64_t>(pi.b) * a.Hq + h * a.g + head) * kD + qd * 32);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = __ldg(row + j);
        }
        const uint32_t *xw = reinterpret_cast<const uint32_t *>(x);
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          amax = max(amax, max((xw[j] << 16) & 0x7fffffffu, xw[j] & 0x7fff0000u));
        }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int ex = min(max(static_cast<int>(amax >> 23) - 127, -126), 126);
        const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
        const float up = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          qf[t][j] = pack_f16(bf16_lo(xw[j]) * down, bf16_hi(xw[j]) * down);
        }
        qs[t][0] = __shfl_sync(0xffffffffu, up, 8 * qd);
        qs[t][1] = __shfl_sync(0xffffffffu, up, 8 * qd + 4);
#pragma unroll
        for (int j = 0; j < 2; ++j) { m[t][j] = mw[t][j] = -INFINITY; l[t][j] = 0.f; }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[t][i][j] = 0.f;
        }
      }
    }
    const uint32_t kb = smem_u32(ring + s * kStage), vb = kb + kHalf;
    // ---- S^T = K Q^T
    float sc[NT][4];
    {
      float s0a[NT][4], s1a[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s0a[t][j] = s1a[t][j] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {         // 16-byte chunk 2*qd + c of rows r and r + 8
        const uint4 lo = lds128(kb + sw128(r, 2 * qd + c));
        const uint4 hi = lds128(kb + sw128(r + 8, 2 * qd + c));
        const uint32_t lw[4] = {lo.x, lo.y, lo.z, lo.w}, hw[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a0 = dequant_f16x2<kInt8, false>(lw[j]);
          const uint32_t a1 = dequant_f16x2<kInt8, false>(hw[j]);
          const uint32_t a2 = dequant_f16x2<kInt8, true>(lw[j]);
          const uint32_t a3 = dequant_f16x2<kInt8, true>(hw[j]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16(j & 1 ? s1a[t] : s0a[t], a0, a1, a2, a3, qf[t][8 * c + 2 * j],
                    qf[t][8 * c + 2 * j + 1]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[t][j] = s0a[t][j] + s1a[t][j];
      }
    }
    // ---- scores of tokens r, r + 8 and heads 2*qd, 2*qd + 1
    const uint8_t *sb = sc_ring + s * 32;
    const bool in0 = pi.page * kTok + r < pi.len, in1 = pi.page * kTok + r + 8 < pi.len;
    const float ks0 = scale_of(sb[r]), ks1 = scale_of(sb[r + 8]);
    const uint32_t vb0 = sb[16 + r], vb1 = sb[24 + r];
    const float ev0 = vb0 == 255u ? __uint_as_float(0x7fffffffu) : static_cast<float>(static_cast<int>(vb0) - 127);
    const float ev1 = vb1 == 255u ? __uint_as_float(0x7fffffffu) : static_cast<float>(static_cast<int>(vb1) - 127);
    bool moves = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sc[t][j] = in0 ? sc[t][j] * ks0 * qs[t][j] : -INFINITY;
        sc[t][2 + j] = in1 ? sc[t][2 + j] * ks1 * qs[t][j] : -INFINITY;
        const float most = fmaxf(sc[t][j], sc[t][2 + j]);
        const float most_w = fmaxf(in0 ? sc[t][j] + ev0 : -INFINITY,
                                   in1 ? sc[t][2 + j] + ev1 : -INFINITY);
        moves |= most > m[t][j] + kSlack || most_w > mw[t][j] + kSlack;
      }
    }
    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float top = fmaxf(m[t][j], max3_over_rows(fmaxf(sc[t][j], sc[t][2 + j])));
          const float top_w =
              fmaxf(mw[t][j], max3_over_rows(fmaxf(in0 ? sc[t][j] + ev0 : -INFINITY,
                                                   in1 ? sc[t][2 + j] + ev1 : -INFINITY)));
          if (top > m[t][j]) {
            l[t][j] *= exp2f(m[t][j] - top);
            m[t][j] = top;
          }
          if (top_w > mw[t][j]) {
            const float f = exp2f(mw[t][j] - top_w);
#pragma unroll
            for (int i = 0; i < 8; ++i) { acc[t][i][j] *= f; acc[t][i][2 + j] *= f; }
            mw[t][j] = top_w;
          }
        }
      }
    }
    // ---- weights
    uint32_t wb[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float p[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[t][j] += fast_exp2(sc[t][j] - m[t][j]) + fast_exp2(sc[t][2 + j] - m[t][j]);
        const float d = mw[t][j] - kUp;
        p[j] = in0 ? fast_exp2(sc[t][j] + ev0 - d) : 0.f;
        p[2 + j] = in1 ? fast_exp2(sc[t][2 + j] + ev1 - d) : 0.f;
      }
      wb[t][0] = transpose8x8(pack_f16(p[0], p[1]));
      wb[t][1] = transpose8x8(pack_f16(p[2], p[3]));
    }
    // ---- O^T += V^T W^T: tokens 2*qd, + 1, + 8, + 9; dims 16*r .. + 15
    {
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 2 * qd + (j & 1) + (j >> 1) * 8;
        v[j] = lds128(vb + sw128(row, r));
      }
      if (pi.page * kTok + kTok > pi.len) {      // rows past the context hold anything
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (pi.page * kTok + 2 * qd + (j & 1) + (j >> 1) * 8 >= pi.len) v[j] = make_uint4(0, 0, 0, 0);
        }
      }
      const uint32_t *w0 = reinterpret_cast<const uint32_t *>(&v[0]);
      const uint32_t *w1 = reinterpret_cast<const uint32_t *>(&v[1]);
      const uint32_t *w2 = reinterpret_cast<const uint32_t *>(&v[2]);
      const uint32_t *w3 = reinterpret_cast<const uint32_t *>(&v[3]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {              // dims 16*r + 2*i, + 1
        const uint32_t sel = i & 1 ? 0x7362u : 0x5140u;
        const uint32_t x = bytes(w0[i >> 1], w1[i >> 1], sel);
        const uint32_t y = bytes(w2[i >> 1], w3[i >> 1], sel);
        const uint32_t a0 = dequant_f16x2<kInt8, false>(x), a1 = dequant_f16x2<kInt8, true>(x);
        const uint32_t a2 = dequant_f16x2<kInt8, false>(y), a3 = dequant_f16x2<kInt8, true>(y);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16(acc[t][i], a0, a1, a2, a3, wb[t][0], wb[t][1]);
      }
    }
    __syncwarp();
    produce(s);                // refill: every lane has read the stage

    if (pi.flags & 2) {
      const bool whole = (pi.flags & 12) == 12;
      const int64_t slot = 2ll * G + (pi.flags & 4 ? 1 : 0);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float sum = l[t][j];
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const int head = t * 8 + 2 * qd + j;
          if (head >= a.g) continue;
          float f = exp2f(mw[t][j] - m[t][j] - kUp);
          float o[16];
          if (whole) f /= sum;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            o[2 * i] = acc[t][i][j] * f;
            o[2 * i + 1] = acc[t][i][2 + j] * f;
          }
          const int hq = h * a.g + head;
          if (whole) {
            uint4 *dst = reinterpret_cast<uint4 *>(
                a.out + (static_cast<int64_t>(pi.b) * a.Hq + hq) * kD + 16 * r);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              dst[i] = make_uint4(pack_bf16(o[8 * i], o[8 * i + 1]),
                                  pack_bf16(o[8 * i + 2], o[8 * i + 3]),
                                  pack_bf16(o[8 * i + 4], o[8 * i + 5]),
                                  pack_bf16(o[8 * i + 6], o[8 * i + 7]));
            }
          } else {
            float4 *dst =
                reinterpret_cast<float4 *>(a.ws.o + (slot * a.Hq + hq) * kD + 16 * r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
            if (r == 0) a.ws.ml[slot * a.Hq + hq] = make_float2(m[t][j], sum);
          }
        }
      }
    }
  }
  if (fail) {
    // the ring's copies still in flight must land before the CTA ends
    for (int k = it; k < n_pages - w.left; ++k) {
      mbar_wait(&full[k % S::kStages], (k / S::kStages) & 1);
    }
    if (lane == 0 && a.err != nullptr) atomicExch(a.err, 1);
  }
}

// Joins the partial results of split sequences and writes the zeros of empty
// ones. kSplit warps share a (sequence, query head), each taking every
// kSplit-th partial; 8 of them for small batches, whose sequences have many
// partials, one where there are enough rows to fill the GPU.
constexpr int kCombineWarps = 8;

template <int kSplit>
__global__ void __launch_bounds__(kCombineWarps * 32) quant_combine_kernel(const QDecodeArgs a) {
  constexpr int kRows = kCombineWarps / kSplit;
  __shared__ float4 so[kCombineWarps][32];
  __shared__ float sm[kCombineWarps], sl[kCombineWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % kSplit;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + warp / kSplit;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool live = row < static_cast<int64_t>(a.B) * a.Hq;
  const int b = live ? static_cast<int>(row / a.Hq) : 0;
  const int head = static_cast<int>(row - static_cast<int64_t>(b) * a.Hq);
  const int p0 = a.ws.prefix[b], p1 = live ? a.ws.prefix[b + 1] : p0;
  const int total = a.ws.prefix[a.B];
  uint2 *dst = reinterpret_cast<uint2 *>(a.out + row * kD) + lane;
  int first = 0, count = 0;      // slots: 2 * first + 1, then 2 * (first + i)
  if (p1 > p0) {
    const int n = groups_of(total, a.groups);
    first = group_of(p0, total, n);
    count = group_of(p1 - 1, total, n) - first + 1;
  } else if (live && part == 0) {
    *dst = make_uint2(0u, 0u);
  }
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (count > 1) {
    auto at = [&](int i) { return (2ll * (first + i) + (i == 0 ? 1 : 0)) * a.Hq + head; };
    for (int i = part + lane * kSplit; i < count; i += 32 * kSplit) m = fmaxf(m, a.ws.ml[at(i)].x);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float mu = m == -INFINITY ? 0.f : m;
    for (int i0 = part; i0 < count; i0 += 4 * kSplit) {
      float4 x[4];
      float2 ml[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * kSplit;
        if (i < count) {
          ml[j] = a.ws.ml[at(i)];
          x[j] = reinterpret_cast<const float4 *>(a.ws.o + at(i) * kD)[lane];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (i0 + j * kSplit < count) {
          const float f = exp2f(ml[j].x - mu);
          l = fmaf(f, ml[j].y, l);
          o.x = fmaf(f, x[j].x, o.x); o.y = fmaf(f, x[j].y, o.y);
          o.z = fmaf(f, x[j].z, o.z); o.w = fmaf(f, x[j].w, o.w);
        }
      }
    }
  }
  if constexpr (kSplit > 1) {
    so[warp][lane] = o;
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
    __syncthreads();
    if (part != 0 || count < 2) return;
    for (int i = 1; i < kSplit; ++i) m = fmaxf(m, sm[warp + i]);
    const float mu = m == -INFINITY ? 0.f : m;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < kSplit; ++i) {
      const float f = exp2f(sm[warp + i] - mu);
      const float4 x = so[warp + i][lane];
      l = fmaf(f, sl[warp + i], l);
      o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y);
      o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
    }
  }
  if (count < 2) return;          // finished by its group
  const float inv = 1.f / l;
  *dst = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
}

template <bool kInt8, int NT>
int launch_decode(const CUtensorMap &tmk, const CUtensorMap &tmv, const QDecodeArgs &a, int grid,
                  cudaStream_t stream) {
  using S = Shape<NT>;
  static_assert(S::kSmem <= 227 * 1024, "shared memory");
  const char *what = "vj_paged_decode_quantized";
  cudaError_t e = cudaFuncSetAttribute(quant_decode_kernel<kInt8, NT>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(S::kSmem));
  if (e != cudaSuccess) {
    return set_error(VJ_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  quant_decode_kernel<kInt8, NT><<<grid, S::kThreads, S::kSmem, stream>>>(tmk, tmv, a);
  return check_launch(what);
}

// Grid and groups of a shape, from head counts and the GPU's size alone.
void decode_grid(int g, int num_kv_heads, int *grid, int *groups) {
  const int warps = g <= 8 ? Shape<1>::kWarps : Shape<2>::kWarps;
  *grid = std::max(num_sms(), (num_kv_heads + warps - 1) / warps);
  *groups = *grid * warps / num_kv_heads;
}

}  // namespace
}  // namespace vj

extern "C" size_t vj_paged_decode_quantized_workspace_size(int32_t batch, int32_t num_q_heads,
                                                           int32_t num_kv_heads,
                                                           int32_t head_dim) {
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim != vj::kD) return 0;
  int grid, groups;
  vj::decode_grid((num_q_heads + num_kv_heads - 1) / num_kv_heads, num_kv_heads, &grid, &groups);
  return vj::scratch_bytes(batch, num_q_heads, groups);
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
  const Pool pool = {static_cast<uint8_t *>(const_cast<void *>(k_cache)),
            static_cast<uint8_t *>(const_cast<void *>(v_cache)),
            static_cast<uint8_t *>(const_cast<void *>(k_scales)),
            static_cast<uint8_t *>(const_cast<void *>(v_scales)),
            stride_block, stride_token, stride_head, scale_stride_block, scale_stride_head,
            num_blocks, block_size};
  QDecodeArgs a;
  int rc = check_pool(what, pool, cache_dtype, num_kv_heads, head_dim);
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
  const int64_t table_pages = static_cast<int64_t>(bt_width) * (block_size / kTok);
  if (static_cast<int64_t>(batch) * table_pages > INT32_MAX ||
      static_cast<int64_t>(batch) * num_q_heads > INT32_MAX) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": batch or block tables too large (2^31 pages)");
  }
  if (batch == 0) return VJ_OK;
  rc = check_pool_memory(what, pool);
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
  CUtensorMap tmk, tmv;
  const uint64_t ntok = static_cast<uint64_t>(num_blocks) * block_size;
  // the two outer dims in the order of their strides
  const bool head_major = stride_head < stride_token;
  for (int i = 0; i < 2; ++i) {
    CUtensorMap *m = i ? &tmv : &tmk;
    const void *base = i ? v_cache : k_cache;
    rc = head_major ? encode_tmap_3d_u8(m, base, kD, num_kv_heads, ntok, stride_head, stride_token,
                                        kD, 1, kTok, true)
                    : encode_tmap_3d_u8(m, base, kD, ntok, num_kv_heads, stride_token, stride_head,
                                        kD, kTok, 1, true);
    if (rc) return rc;
  }
  a.q = static_cast<const __nv_bfloat16 *>(q);
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.bt = block_tables;
  a.lens = context_lens;
  a.ks = pool.ks;
  a.vs = pool.vs;
  a.ssb = scale_stride_block;
  a.ssh = scale_stride_head;
  a.B = batch;
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.g = num_q_heads / num_kv_heads;
  a.bt_stride = bt_stride;
  a.pages_per_block = block_size / kTok;
  a.block_size = block_size;
  a.max_pages = static_cast<int>(table_pages);
  a.num_blocks = static_cast<int>(num_blocks);
  a.head_major = head_major ? 1 : 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = error_flag;
  int grid;
  decode_grid(a.g, num_kv_heads, &grid, &a.groups);
  char *w = static_cast<char *>(workspace);
  a.ws.prefix = reinterpret_cast<int32_t *>(w);
  w += up256(4 * (static_cast<size_t>(batch) + 1));
  a.ws.ml = reinterpret_cast<float2 *>(w);
  w += up256(2 * static_cast<size_t>(a.groups) * num_q_heads * sizeof(float2));
  a.ws.o = reinterpret_cast<float *>(w);
  const bool i8 = cache_dtype == VJ_CACHE_INT8;
  if (a.g <= 8) {
    rc = i8 ? launch_decode<true, 1>(tmk, tmv, a, grid, stream)
            : launch_decode<false, 1>(tmk, tmv, a, grid, stream);
  } else {
    rc = i8 ? launch_decode<true, 2>(tmk, tmv, a, grid, stream)
            : launch_decode<false, 2>(tmk, tmv, a, grid, stream);
  }
  if (rc) return rc;
  const int64_t rows = static_cast<int64_t>(batch) * num_q_heads;
  if (rows < 4 * kCombineWarps * num_sms()) {
    quant_combine_kernel<kCombineWarps>
        <<<static_cast<unsigned>(rows), kCombineWarps * 32, 0, stream>>>(a);
  } else {
    quant_combine_kernel<1><<<static_cast<unsigned>((rows + kCombineWarps - 1) / kCombineWarps),
                              kCombineWarps * 32, 0, stream>>>(a);
  }
  return check_launch("vj_paged_decode_quantized");
}
