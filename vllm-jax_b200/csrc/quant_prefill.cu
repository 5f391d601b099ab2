// Prefill attention straight from the quantised pages, for few new tokens: causal
// attention of each sequence's new tokens over its cached context.
//
// A tile of 128 rows (tokens x query heads of one KV head) meets key tiles of 128 on
// tcgen05.mma in bf16. Eight warps read the pages and write bf16 tiles to shared memory,
// element times scale, which rounds nothing; 8 lanes read a row of 128 bytes. Reading
// the context back to bf16 in a launch of its own and taking it in from there does that
// work once instead of once per row tile, and costs its launch and 4 bytes per element
// of traffic: the caller takes that way where there are many row tiles.
//   The keys of a row tile are split over as many CTAs as leave no SM idle; their
// results are joined by prefill_join_kernel.
//
//   TMEM columns: [0,128) S of even key tiles | [128,256) of odd ones | [256,384) O of
//   the first 64 keys of every tile | [384,512) of the others; P (bf16 pairs) overwrites
//   the first half of its 64 columns of S.
// Warps: 0-3 softmax of the first 64 keys of a tile (a row a thread), 4-7 of the others,
// 8-11 K tiles, 12-15 V tiles, 16 the products (and q by TMA). The two halves are two
// softmaxes with maxima, sums and outputs of their own, joined at the end: one thread a
// row took 2.1 us a key tile, since one warp is then all that a quarter of the SM has
// for it. Pages travel two tiles ahead through shared memory (loads held in registers
// one tile ahead: 2.1 us; four warps for K and V together: 2.5).
// The weights enter their product rounded to bf16 (half a step: 2^-8 of each), since its
// two operands have one type and V's rows, element times scale, need bf16's range; their
// sum, which divides them, and all outputs up to the last rounding are in 32 bits.
// S(j+1) is computed while the softmax of S(j) runs; O is rescaled only where a row's
// maximum grows by more than 2^8, and then behind PV(j - 1).
// Latency-bound: a few key tiles a CTA, each load -> convert -> scores -> softmax ->
// product; 1.8 us a key tile in the steady state (16 sequences of 30 tokens after up to
// 2000: 34.5 us, issue rate 0.46, DRAM 11%, tensor pipe 10%).
//   One token after 1421 cached ones, 32 / 8 heads: 11.9 us (15.5 with the context read
// back first); 32 after 11129: 22.3 (35.6); four prompts of up to 269 tokens: 13 (16.5).
#include "prefill_join.cuh"
#include "quant.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

namespace vj {
namespace {
using namespace qn;

constexpr int kRows = 128, kKeys = 128;
constexpr int kHalfTile = 128 * 128;           // 128 rows of 64 bf16, 128-byte swizzle
constexpr int kTileBytes = 2 * kHalfTile;
constexpr int kRing = 2;                       // tiles of K, and of V
constexpr int kOffK = kTileBytes, kOffV = kOffK + kRing * kTileBytes;
// pages on their way: [2 tiles][K, V][4 warps][8 pages][32 lanes] 16 bytes
constexpr int kOffRaw = kOffV + kRing * kTileBytes, kRawHalf = 4 * 8 * 512;
constexpr int kOffBars = kOffRaw + 4 * kRawHalf;
constexpr int kPrefillThreads = 17 * 32;
constexpr uint32_t kColO = 256;                // + 128 for the second half of the keys
constexpr float kGrow = 8.0f;                  // log2 of what a maximum may grow by unseen

struct PrefillBars {
  uint64_t q_full, k_full[kRing], k_empty[kRing], v_full[kRing], v_empty[kRing];
  uint64_t s_full[2], p_full[2], pv_done[2];
  uint32_t tmem;
};
constexpr size_t kPrefillSmem = 1024 + kOffBars + sizeof(PrefillBars);
static_assert(kPrefillSmem <= 227 * 1024, "shared memory");

struct QPrefillArgs {
  Pool pool;
  __nv_bfloat16 *out;
  const int32_t *bt, *cu, *lens;
  int Hq, Hkv, g, tt;                          // tt = tokens of a row tile = 128 / g
  int bt_stride, pages_per_block, max_pages, num_tokens, num_seqs;
  float scale_log2;
  int32_t *err;
  int parts, part_rows, keep_tail;             // prefill_join.cuh
  float *part_o;
  float2 *part_ml;
};

VJ_DEV uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
VJ_DEV void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}
VJ_DEV uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// 16 bytes from global to shared memory, of which `bytes` (0 or 16) are read, the rest 0.
VJ_DEV void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
VJ_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
VJ_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
VJ_DEV uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
VJ_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// What brings a pair of to_bf16 to its value times the row's scale, and the byte up to
// which one bf16 number holds it (beyond: 2^127 and the rest). NaN for byte 255.
template <bool kInt8>
constexpr uint32_t kScaleUp = kInt8 ? 0 : 120;
template <bool kInt8>
VJ_DEV uint32_t scale_pair(uint32_t byte) {
  const uint32_t b = byte == 255u ? 0x7fffu
                     : kInt8 && byte == 0u ? 0x0040u               // 2^-127
                                           : min(byte + kScaleUp<kInt8>, 254u) << 7;
  return b * 0x10001u;
}
// The elements in the low or high half of a word as a pair of bf16 numbers, exactly.
// int8: 128 + its low 7 bits, less 128 or (negative) 256. e4m3: 2^-120 times it, since
// bf16 gives the 4 bits of the exponent 2^(x - 127) instead of 2^(x - 7). (By way of
// f16, whose bits are moved, it takes twice the instructions of the busiest pipe.)
template <bool kInt8, bool kHi>
VJ_DEV uint32_t to_bf16(uint32_t w) {
  uint32_t y;                                  // a byte in each half
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(y) : "r"(w), "n"(kHi ? 0x4342 : 0x4140));
  if constexpr (kInt8) {
    return sub_bf16x2((y & 0x007f007fu) | 0x43004300u, (y & 0x00800080u) | 0x43004300u);
  } else {
    return y * 16u + (y & 0x00800080u) * 240u;   // sign to bit 15, the rest to bits 10 .. 4
  }
}

// The K (v = 0) or V tiles of one CTA into their ring, by four warps: warp cw takes rows
// 4 cw .. + 3 of every page, 8 lanes a row. `limit`: tokens from there on are zeros.
// False if a wait ran out.
template <bool kInt8>
VJ_DEV bool convert_tiles(const QPrefillArgs &a, uint8_t *smem, PrefillBars &bar, int v, int s, int h,
                          int j0, int n, int limit, int cw, int lane) {
  const int c = lane & 7, r0 = 4 * cw + (lane >> 3);
  const bool upper = c >= 4;                   // dims 64 and up
  const int32_t *bt = a.bt + static_cast<int64_t>(s) * a.bt_stride;
  const int64_t row_at = h * a.pool.sh + r0 * a.pool.st + c * 16, scale_at = h * a.pool.ssh + 4 * cw;
  // where this lane's 32 bytes of bf16 go in a tile (16 rows on, the swizzle is the same).
  // The half of the lanes that has dims 64 and up starts with its second 16 bytes, so
  // that 8 lanes store to 8 different bank groups.
  const uint32_t to = smem_u32(smem) + (upper ? kHalfTile : 0);
  const uint32_t to0 = to + sw128(r0, 2 * (c & 3) + (upper ? 1 : 0));
  const uint32_t to1 = to + sw128(r0, 2 * (c & 3) + (upper ? 0 : 1));
  // this lane's 16 bytes of a page on its way (it reads what it copied itself)
  const uint32_t raw = smem_u32(smem) + kOffRaw + v * kRawHalf + cw * (8 * 512) + lane * 16;
  const uint8_t *const rows = (v ? a.pool.v : a.pool.k) + row_at;
  const uint8_t *const scale_bytes = (v ? a.pool.vs : a.pool.ks) + scale_at;
  uint64_t *const empty = v ? bar.v_empty : bar.k_empty, *const full = v ? bar.v_full : bar.k_full;
  // where page `lane & 7` of a key tile lies: its table entry is read two tiles before
  // its rows are needed, and the scale bytes of the warp's four rows with the rows
  int64_t at_rows = 0;
  int ahead_blk = 0, ahead_off = 0;
  auto look_up = [&](int j) {
    const int page = (j0 + j) * 8 + c;
    ahead_blk = ahead_off = 0;
    if (j < n && page < a.max_pages) {
      const int entry = page / a.pages_per_block;
      ahead_off = (page - entry * a.pages_per_block) * 16;
      ahead_blk = bt[entry];
    }
  };
  auto looked_up = [&]() {                     // leaves at_rows; the scale bytes
    // (blocks that are none are read as block 0, as the other attention kernels do)
    const int blk = ahead_blk < 0 || ahead_blk >= a.pool.num_blocks ? 0 : ahead_blk;
    at_rows = blk * a.pool.sb + ahead_off * a.pool.st;
    return *reinterpret_cast<const uint32_t *>(scale_bytes + blk * a.pool.ssb + ahead_off);
  };
  auto load = [&](int j) {                     // a key tile's pages
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t rp = __shfl_sync(0xffffffffu, at_rows, i);
      const bool there = j < n && (j0 + j) * kKeys + i * 16 + r0 < limit;
      cp_async16(raw + (j & 1) * (2 * kRawHalf) + i * 512, rows + rp, there ? 16 : 0);
    }
    cp_async_commit();
  };
  look_up(0);
  uint32_t scales = looked_up();
  look_up(1);
  load(0);
  uint32_t next_scales = looked_up();
  look_up(2);
  load(1);
  for (int j = 0; j < n; ++j) {
    const int st = j % kRing;
    const uint32_t last_scales = looked_up();  // of tile j + 2
    look_up(j + 3);
    cp_async_wait<1>();                      // this tile's pages; the next one's travel
    const bool ok = j < kRing || mbar_wait(&empty[st], (j / kRing - 1) & 1);
    if (!__all_sync(0xffffffffu, ok)) {
      cp_async_wait<0>();
      return false;
    }
    const uint32_t tile = (v ? kOffV : kOffK) + st * kTileBytes;
    const uint32_t from = raw + (j & 1) * (2 * kRawHalf);
    // the scales first, then no branches: the pages' chains run into one another
    uint32_t f2[8];
    bool beyond = false;                     // e4m3: rows beyond 2^7
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m = __shfl_sync(0xffffffffu, scales, i) >> (lane & 24) & 0xffu;
      if ((j0 + j) * kKeys + i * 16 + r0 >= limit) m = 127u;
      f2[i] = scale_pair<kInt8>(m);
      beyond |= !kInt8 && m > 254u - kScaleUp<kInt8> && m != 255u;
    }
    auto convert = [&](auto big) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4 y = lds128(from + i * 512);
        const uint32_t w[4] = {upper ? y.z : y.x, upper ? y.w : y.y,
                               upper ? y.x : y.z, upper ? y.y : y.w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[2 * k] = mul_bf16x2(to_bf16<kInt8, false>(w[k]), f2[i]);
          o[2 * k + 1] = mul_bf16x2(to_bf16<kInt8, true>(w[k]), f2[i]);
        }
        if constexpr (big.value) {           // the rest of the scale
          uint32_t m = __shfl_sync(0xffffffffu, scales, i) >> (lane & 24) & 0xffu;
          if ((j0 + j) * kKeys + i * 16 + r0 >= limit) m = 127u;
          const uint32_t rest = m == 255u ? 127u : max(m + kScaleUp<kInt8>, 254u) - 254u + 127u;
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = mul_bf16x2(o[k], (rest << 7) * 0x10001u);
        }
        const uint32_t at = tile + i * (16 * 128);
        sts128(to0 + at, o[0], o[1], o[2], o[3]);
        sts128(to1 + at, o[4], o[5], o[6], o[7]);
      }
    };
    if (__any_sync(0xffffffffu, beyond)) convert(std::true_type{});
    else convert(std::false_type{});
    fence_proxy_async_smem();
    mbar_arrive(&full[st]);
    load(j + 2);                               // into the place that is read now
    scales = next_scales;
    next_scales = last_scales;
  }
  cp_async_wait<0>();
  return true;
}

// Grid: row tiles, KV heads, (sequence, part).
template <bool kInt8>
__global__ void __launch_bounds__(kPrefillThreads, 1)
quant_prefill_kernel(const __grid_constant__ CUtensorMap tmq, const QPrefillArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  PrefillBars &bar = *reinterpret_cast<PrefillBars *>(smem + kOffBars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y, s = blockIdx.z / a.parts, part = blockIdx.z - s * a.parts;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmq);
    mbar_init(&bar.q_full, 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&bar.k_full[i], 128);
      mbar_init(&bar.v_full[i], 128);
      mbar_init(&bar.k_empty[i], 1);
      mbar_init(&bar.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_full[i], 2 * kRows);
      mbar_init(&bar.pv_done[i], 1);
    }
    fence_mbar_init();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (a.parts > 1) asm volatile("griddepcontrol.launch_dependents;");
  if (a.num_seqs == 0) {
    zero_tail_share(a, threadIdx.x, kPrefillThreads);
    return;
  }
  const int first = a.cu[0], q0 = a.cu[s], q1 = a.cu[s + 1];
  int ctx = a.lens[s];
  const int n = q1 - q0;
  const int tq0 = (gridDim.x - 1 - blockIdx.x) * a.tt;     // first token of the row tile
  if (tq0 >= n) {              // the whole CTA
    if (a.parts == 1) zero_tail_share(a, threadIdx.x, kPrefillThreads);
    return;
  }
  ctx = max(ctx, n);
  const int p0 = ctx - n;                                  // cached prefix
  const int all = (p0 + min(n, tq0 + a.tt) + kKeys - 1) / kKeys;
  const int j0 = static_cast<int>(static_cast<int64_t>(all) * part / a.parts);
  const int nkv = static_cast<int>(static_cast<int64_t>(all) * (part + 1) / a.parts) - j0;
  // this thread's row and half of the keys, in the softmax warps
  const int half = threadIdx.x / kRows, r = threadIdx.x % kRows, tq = tq0 + r / a.g;
  const bool valid = half < 2 && tq < n && q0 + tq < a.num_tokens;
  const int64_t row = static_cast<int64_t>(q0 + tq) * a.Hq + h * a.g + r % a.g;
  const int64_t rel = row_of_part(a, first, q0 + tq);
  const bool in_parts = valid && rel >= 0;
  const int64_t part_row = place_in_parts(a, part, rel, h * a.g + r % a.g);
  if (nkv == 0) {              // more parts than key tiles
    if (in_parts && half == 0) a.part_ml[part_row] = make_float2(kLowest, 0.f);
    return;
  }
  if (warp == 16) tmem_alloc(&bar.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem;
  bool ok = true;

  if (warp >= 8 && warp < 16) {
    ok = convert_tiles<kInt8>(a, smem, bar, warp >= 12, s, h, j0, nkv, min(ctx, a.max_pages * 16),
                              warp & 3, lane);
    if (a.parts == 1 && warp == 15) zero_tail_share(a, lane, 32);
  } else if (warp == 16) {
    if (lane == 0) {
      mbar_arrive_expect_tx(&bar.q_full, kTileBytes);
      tma_load_3d(smem, &tmq, &bar.q_full, 0, h * a.g, q0 + tq0);
      tma_load_3d(smem + kHalfTile, &tmq, &bar.q_full, 64, h * a.g, q0 + tq0);
      constexpr uint32_t idesc_qk = umma_idesc_bf16(kRows, kKeys, false);
      constexpr uint32_t idesc_pv = umma_idesc_bf16(kRows, kD, true);
      const uint32_t sq = smem_u32(smem), sk = smem_u32(smem + kOffK), sv = smem_u32(smem + kOffV);
      auto qk = [&](int j) {                   // S = Q K^T
        const uint32_t kb = sk + (j % kRing) * kTileBytes;
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * kHalfTile + (kk & 3) * 32;
          umma_ss(tmem + (j & 1) * kKeys, umma_desc_sw128(sq + off, 16, 1024),
                  umma_desc_sw128(kb + off, 16, 1024), idesc_qk, kk > 0 ? 1u : 0u);
        }
        umma_commit(&bar.s_full[j & 1]);
        umma_commit(&bar.k_empty[j % kRing]);
      };
      ok = mbar_wait(&bar.q_full, 0);
      for (int j = 0; j < min(nkv, 2) && ok; ++j) {
        ok = mbar_wait(&bar.k_full[j], 0);
        if (!ok) break;
        tc_fence_after();
        qk(j);
      }
      for (int j = 0; j < nkv && ok; ++j) {
        const int st = j % kRing;
        ok = mbar_wait(&bar.p_full[j & 1], (j >> 1) & 1) &&
             mbar_wait(&bar.v_full[st], (j / kRing) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t vb = sv + st * kTileBytes;
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk) {              // O += P V, a half of the keys each
          const int hf = kk >> 2, k4 = kk & 3;
          umma_ts(tmem + kColO + hf * kD, tmem + (j & 1) * kKeys + hf * 64 + k4 * 8,
                  umma_desc_sw128(vb + kk * 2048, kHalfTile, 1024), idesc_pv,
                  (j > 0 || k4 > 0) ? 1u : 0u);
        }
        umma_commit(&bar.v_empty[st]);
        umma_commit(&bar.pv_done[j & 1]);
        if (j + 2 < nkv) {                     // S(j) is read: in issue order behind it
          ok = mbar_wait(&bar.k_full[(j + 2) % kRing], ((j + 2) / kRing) & 1);
          if (!ok) break;
          tc_fence_after();
          qk(j + 2);
        }
      }
    }
  } else {
    // ---- softmax: a row and half of the keys a thread
    const int qpos = p0 + tq, qpos_min = p0 + tq0;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lanes + kColO;
    float m_run = kLowest, l_run = 0.f;
    for (int j = 0; j < nkv; ++j) {
      const uint32_t tS = tmem + lanes + (j & 1) * kKeys + half * 64;
      ok = mbar_wait(&bar.s_full[j & 1], (j >> 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after();
      float v[64];
      tmem_ld64(tS, v);
      const int kbase = (j0 + j) * kKeys + half * 64;
      if (kbase + 63 > qpos_min) {
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          if (kbase + i > qpos) v[i] = -INFINITY;
        }
      }
      float mx[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) mx[k] = max3(v[k], v[k + 4], v[k + 8]);
#pragma unroll
      for (int i = 12; i < 60; i += 8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], v[i + k], v[i + 4 + k]);
      }
      const float top = max3(max3(mx[0], mx[1], v[60]), max3(mx[2], mx[3], v[61]), fmaxf(v[62], v[63]));
      const float m_new = fmaxf(m_run, top * a.scale_log2);
      const bool grown = m_new - m_run > kGrow;
      const float m_use = j == 0 || grown ? m_new : m_run;
      const float corr = j == 0 ? 0.f : fast_exp2(m_run - m_use);
      uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
      const uint64_t sc2 = f32x2(a.scale_log2, a.scale_log2), nm2 = f32x2(-m_use, -m_use);
      uint32_t pw[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float x0, x1;
        f32x2_split(f32x2_fma(f32x2(v[2 * i], v[2 * i + 1]), sc2, nm2), x0, x1);
        const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
        sum2[i & 3] = f32x2_add(sum2[i & 3], f32x2(e0, e1));
        pw[i] = pack_bf16(e0, e1);
      }
      tmem_st32u_nowait(tS, pw);
      float u[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) f32x2_split(sum2[k], u[2 * k], u[2 * k + 1]);
      l_run = l_run * corr + (((u[0] + u[1]) + (u[2] + u[3])) + ((u[4] + u[5]) + (u[6] + u[7])));
      m_run = m_use;
      if (j > 0 && __any_sync(0xffffffffu, grown)) {
        ok = mbar_wait(&bar.pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1);       // O holds PV(j - 1)
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
#pragma unroll 1
        for (int k = 0; k < kD / 32; ++k) {
          float o[32];
          tmem_ld32(tO + half * kD + k * 32, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= corr;
          tmem_st32(tO + half * kD + k * 32, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bar.p_full[j & 1]);
    }
    if (ok) ok = mbar_wait(&bar.pv_done[(nkv - 1) & 1], ((nkv - 1) >> 1) & 1);
    // ---- the halves of the keys together: half of the dims a thread
    float2 *const ml = reinterpret_cast<float2 *>(smem);   // q's place, which no product reads now
    ml[half * kRows + r] = make_float2(m_run, l_run);
    named_bar_sync(1, 2 * kRows);
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      const float2 ml0 = ml[r], ml1 = ml[kRows + r];
      const float m = fmaxf(ml0.x, ml1.x), g0 = exp2f(ml0.x - m), g1 = exp2f(ml1.x - m);
      const float l = ml0.y * g0 + ml1.y * g1, inv = a.parts > 1 ? 1.f : 1.f / l;
      const float f0 = g0 * inv, f1 = g1 * inv;
      if (a.parts > 1 && in_parts && half == 0) a.part_ml[part_row] = make_float2(m, l);
#pragma unroll 1
      for (int k = 2 * half; k < 2 * half + 2; ++k) {
        float o[32], o1[32];
        tmem_ld32(tO + k * 32, o);
        tmem_ld32(tO + kD + k * 32, o1);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = o[i] * f0 + o1[i] * f1;
        if (a.parts > 1 && in_parts) {
          float4 *dst = reinterpret_cast<float4 *>(a.part_o + part_row * kD + k * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        } else if (a.parts == 1 && valid) {
          uint4 *dst = reinterpret_cast<uint4 *>(a.out + row * kD + k * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            dst[i] = make_uint4(pack_bf16(o[8 * i], o[8 * i + 1]),
                                pack_bf16(o[8 * i + 2], o[8 * i + 3]),
                                pack_bf16(o[8 * i + 4], o[8 * i + 5]),
                                pack_bf16(o[8 * i + 6], o[8 * i + 7]));
          }
        }
        __syncwarp();
      }
    } else {
      ok = false;
    }
  }
  if (!ok && a.err != nullptr) atomicExch(a.err, 1);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) tmem_dealloc(tmem, 512);
}

// Parts of a row tile's key tiles: as many as fill the GPU, of two key tiles or more
// each where there are many.
int quant_prefill_parts(int64_t tiles, int64_t num_kv_heads, int64_t num_seqs,
                        int64_t max_context_len) {
  const int64_t ctas = tiles * num_kv_heads * num_seqs, keys = (max_context_len + kKeys - 1) / kKeys;
  if (ctas == 0 || keys < 8) return 1;
  return static_cast<int>(std::max<int64_t>(1, std::min(num_sms() / ctas, keys / 2)));
}

template <bool kInt8>
int launch_quant_prefill(const std::string &what, const CUtensorMap &tmq, const QPrefillArgs &a,
                         dim3 grid, cudaStream_t stream) {
  // the shared-memory opt-in is a per-device attribute of the kernel
  static std::atomic<bool> opted[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !opted[dev].load(std::memory_order_acquire))) {
    e = cudaFuncSetAttribute(quant_prefill_kernel<kInt8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kPrefillSmem));
    if (e == cudaSuccess && dev < 64) opted[dev].store(true, std::memory_order_release);
  }
  if (e != cudaSuccess) return set_error(VJ_ERR_CUDA, what + ": " + cudaGetErrorString(e));
  return launch_dependent(what.c_str(), quant_prefill_kernel<kInt8>, grid, kPrefillThreads,
                          kPrefillSmem, stream, tmq, a);
}

}  // namespace
}  // namespace vj

extern "C" size_t vj_paged_prefill_quantized_workspace_size(int64_t num_tokens, int32_t num_seqs,
                                                            int32_t num_q_heads,
                                                            int32_t num_kv_heads, int32_t head_dim,
                                                            int32_t max_seqlen_q,
                                                            int32_t max_context_len) {
  if (num_tokens <= 0 || num_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      head_dim != vj::kD || max_context_len < 0 || num_q_heads % num_kv_heads != 0 ||
      vj::kRows % (num_q_heads / num_kv_heads) != 0) {
    return 0;
  }
  const int64_t tt = vj::kRows / (num_q_heads / num_kv_heads);
  const int64_t longest = max_seqlen_q > 0 ? max_seqlen_q : num_tokens;
  const int parts = vj::quant_prefill_parts((longest + tt - 1) / tt, num_kv_heads, num_seqs,
                                            max_context_len);
  return parts == 1 ? 0
                    : static_cast<size_t>(parts) * vj::rows_of_parts(num_tokens, num_seqs, longest) *
                          num_q_heads *
                          (vj::kD * sizeof(float) + sizeof(float2));
}

extern "C" vj_status vj_paged_prefill_quantized(
    const void *q, const void *k_cache, const void *v_cache, const void *k_scales,
    const void *v_scales, int32_t cache_dtype, const int32_t *block_tables,
    const int32_t *cu_seqlens_q, const int32_t *context_lens, void *out, int64_t num_tokens,
    int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int64_t num_blocks, int32_t block_size, int32_t bt_width, int32_t bt_stride,
    int64_t stride_block, int64_t stride_token, int64_t stride_head, int64_t scale_stride_block,
    int64_t scale_stride_head, int32_t max_seqlen_q, int32_t max_context_len, float scale,
    void *workspace, size_t workspace_bytes, int32_t *error_flag, cudaStream_t stream) {
  using namespace vj;
  const std::string what = "vj_paged_prefill_quantized";
  QPrefillArgs a;
  a.pool = {static_cast<uint8_t *>(const_cast<void *>(k_cache)),
            static_cast<uint8_t *>(const_cast<void *>(v_cache)),
            static_cast<uint8_t *>(const_cast<void *>(k_scales)),
            static_cast<uint8_t *>(const_cast<void *>(v_scales)),
            stride_block, stride_token, stride_head, scale_stride_block, scale_stride_head,
            num_blocks, block_size};
  int rc = check_pool(what, a.pool, cache_dtype, num_kv_heads, head_dim);
  if (rc) return rc;
  if (num_tokens < 0 || num_seqs < 0 || num_q_heads <= 0 || bt_width < 0 || bt_stride < bt_width ||
      max_context_len < 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": negative or zero size");
  }
  if (num_q_heads % num_kv_heads != 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT,
                     what + ": Number of Q heads must be divisible by number of KV heads. Got " +
                         std::to_string(num_q_heads) + " and " + std::to_string(num_kv_heads) + ".");
  }
  a.g = num_q_heads / num_kv_heads;
  if (kRows % a.g != 0) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": query heads per KV head must divide 128");
  }
  // the row maximum is taken of q.k, before the scale; 0 times a masked key's -inf is NaN
  if (!(scale > 0.f) || std::isinf(scale)) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": scale must be positive and finite");
  }
  if (num_tokens == 0) return VJ_OK;
  rc = check_pool_memory(what, a.pool);
  if (rc) return rc;
  if (!q || !cu_seqlens_q || !out || (num_seqs > 0 && (!context_lens || !block_tables))) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": null pointer");
  }
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 != 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": q and out must be 16-byte aligned");
  }
  if (overlap_in_part(q, out, num_tokens * num_q_heads * kD * 2)) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": out must be q or not overlap it");
  }
  a.tt = kRows / a.g;
  const int64_t longest = max_seqlen_q > 0 ? max_seqlen_q : num_tokens;
  const int64_t tiles = num_seqs > 0 ? (longest + a.tt - 1) / a.tt : 1;
  a.parts = quant_prefill_parts(num_seqs > 0 ? tiles : 0, num_kv_heads, num_seqs, max_context_len);
  const int64_t z = std::max<int64_t>(static_cast<int64_t>(num_seqs) * a.parts, 1);
  const int64_t rows = num_tokens * num_q_heads;
  if (tiles > INT32_MAX || num_kv_heads > 65535 || z > 65535 || rows > INT32_MAX ||
      static_cast<int64_t>(bt_width) * block_size > INT32_MAX - kKeys) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": grid too large");
  }
  if (a.parts > 1) {
    const size_t need = vj_paged_prefill_quantized_workspace_size(
        num_tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, max_seqlen_q, max_context_len);
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
      return set_error(VJ_ERR_WORKSPACE, what + ": workspace needs " + std::to_string(need) +
                                             " bytes, 16-byte aligned");
    }
  }
  CUtensorMap tmq;
  rc = encode_tmap_3d(&tmq, q, kD, num_q_heads, num_tokens, kD * 2,
                      static_cast<uint64_t>(num_q_heads) * kD * 2, 64, a.g, a.tt, true);
  if (rc) return rc;
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.bt = block_tables;
  a.cu = cu_seqlens_q;
  a.lens = context_lens;
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.bt_stride = bt_stride;
  a.pages_per_block = block_size / 16;
  a.max_pages = bt_width * a.pages_per_block;
  a.num_tokens = static_cast<int>(num_tokens);
  a.num_seqs = num_seqs;
  a.keep_tail = 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = error_flag;
  a.part_o = static_cast<float *>(workspace);
  a.part_rows = static_cast<int>(rows_of_parts(num_tokens, num_seqs, longest));
  a.part_ml = a.parts > 1 ? reinterpret_cast<float2 *>(
                                a.part_o + static_cast<int64_t>(a.parts) * a.part_rows * num_q_heads * kD)
                          : nullptr;
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(num_kv_heads),
                  static_cast<unsigned>(z));
  rc = cache_dtype == VJ_CACHE_INT8 ? launch_quant_prefill<true>(what, tmq, a, grid, stream)
                                    : launch_quant_prefill<false>(what, tmq, a, grid, stream);
  if (rc || a.parts == 1) return rc;
  return launch_join(what.c_str(), a, stream);
}
