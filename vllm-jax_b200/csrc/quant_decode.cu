// Attention of one new token per sequence over the quantised paged KV cache.
//
//   s_t = scale * q . k_t,  p = softmax(s),  o = sum_t p_t v_t,  t < context
//
// HBM-bound: every cached row is read once (129 bytes a row, K and V), for all
// query heads of its KV head together.
//
// The work is cut into pages of 16 tokens. All sequences' pages in a row are
// split evenly over the warps that serve a KV head; the warps of the other heads
// walk the same pages at the same time, so a page's rows, which lie side by
// side, are read together. A sequence's start (its q, its own results) costs a
// warp about as much as three pages, so the split counts that many places before
// every sequence's pages: without them a warp with six short sequences among 64
// of 1 to 8192 tokens took 26 us where most took 18. Every CTA finds its warps'
// ranges from the context lengths by itself: there is no planning launch.
//   Little work (below kDealt pages a warp): eight warps with neighbouring
// ranges form a unit and join the sequences they share in shared memory; a
// sequence that more than one unit shares leaves a partial result in each (its
// output in 32 bits, maximum and sum).
//   Much work: SMs do not get equal shares of a saturated memory (even ranges
// of 157 pages a warp ended between 212 and 281 us), so a warp keeps only the
// first 4/5 of its range for sure. The rest is three pieces, which a warp takes
// one by one from its own range, and then from ranges of warps that are behind,
// by counting up the range's word. A range's warp sets that word to 0 before
// anything else; one that looks at a word before that takes no piece, or one
// that will be done twice with the same result, so the words need no launch of
// their own to be cleared. Pieces depend on the lengths alone and each leaves
// its own partial results: who does which changes no result.
//   quant_combine_kernel joins the partial results, at most two of a unit,
// range or piece, in the order of the pages.
//   Where the block tables hold at most kWhole pages a row and there is a unit for
// every sequence and KV head, a unit takes a whole sequence: nothing is left to
// join, and there is one launch (17 tokens: 5.4 us against 7.5; at 125 pages, 16 a
// warp, it would be 21 against 11).
//
// A warp streams its pages through a ring of its own in shared memory: one TMA
// box of 16 rows x 128 bytes of K and of V (128-byte swizzle; the distance from
// the one to the other is the box's fourth dimension) and one of their scale
// bytes. Where a page lies (sequence ends, block tables) is looked up for 32
// pages at once, a page a lane, and that lane issues its copies. Products run on mma.sync m16n8k16 in f16 with
// 32-bit sums, with the tokens, then the dimensions, as the 16 rows and the
// query heads of the group as the 8 columns:
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
#include <atomic>
#include <cmath>

namespace vj {
namespace {
using namespace qn;

constexpr int kTok = 16;                      // tokens per page
constexpr int kHalf = kTok * kD;              // bytes of a page's K (or V) rows
constexpr int kStage = 2 * kHalf;
constexpr int kScaleStage = 128;              // 32 bytes; a TMA destination is 128-byte aligned
constexpr int kStart = 3;                     // places in front of a sequence's pages
constexpr int kWhole = 32;                    // pages up to which a unit takes a sequence
constexpr int kDealt = 32;                    // pages a warp from which on a part is dealt
constexpr uint32_t kFresh = 127;              // scale byte of rows that nothing was stored to
constexpr float kSlack = 11.0f;               // log2 of what a score may pass the maximum by
constexpr float kUp = 4.0f;                   // log2 of the weight at the maximum

// A page: what its lane looked up.
struct Page {
  int b;             // sequence
  int valid_flags;   // tokens inside the context (1..16), and kFirst.. below << 8
  int tok, blk;      // first token's place in the pool, its block
};
// What the consumer of a stage needs to know of it.
struct Info {
  int b, valid_flags, h, segment;
};
constexpr int kFirst = 1;      // first page of its segment (the part of a sequence in a range)
constexpr int kLast = 2;       // last page of its segment
constexpr int kHead = 4;       // the segment starts with the sequence
constexpr int kTail = 8;       // the segment ends with the sequence
constexpr int kEnd = 16;       // last page of the range

// What a warp leaves for its unit to join.
struct Left {
  int b0;         // sequence of a segment that began before the range, or -1
  int ends0;      // whether that sequence ends in it
  int far0;       // whether the record is in the workspace (pages came after it) or the ring
  int b1;         // sequence of a segment that began in the range and goes on behind it, or -1
};

// A sequence and a page of it.
struct Place {
  int b, p, np, len;      // p of np pages, of a context of len tokens
};

// How all places are split: n ranges of neighbouring ones, the first `more` of
// them of pages + 1, the others of `pages` (in both, the kStart places in front of
// a sequence count as pages). Where pieces are dealt, a range is cut in kCuts parts.
constexpr int kCuts = 4;
struct Split {
  int n, pages, more, dealt;
};

template <int NT>
struct Shape {                                // NT tiles of 8 query heads
  static constexpr int kUnit = 8;                             // warps that join their results
  static constexpr int kWarps = NT == 1 ? 16 : 8;
  static constexpr int kStages = NT == 1 ? 3 : 6;
  static constexpr int kThreads = kWarps * 32;                // a power of two
  static constexpr int kRing = kWarps * kStages;
  static constexpr int kUnits = kWarps / kUnit;
  static constexpr int kHeads = NT * 8;
  // pages, scale bytes, barriers, left records, scan
  static constexpr size_t kSmem = 1024 + (size_t)kRing * (kStage + kScaleStage + sizeof(Info) + 8) +
                                  kWarps * sizeof(Left) + kUnits * (sizeof(Split) + sizeof(Place)) +
                                  (kThreads + kWarps) * 4;
  // a record in a warp's ring: kHeads x 128 outputs, kHeads (maximum, sum)
  static_assert(kHeads * (kD + 2) * 4 <= kStages * kStage, "a record fits the ring");
};

struct Scratch {
  int32_t *taken;     // [groups][Hkv] pieces of a range that are taken
  int2 *segments;     // [B] first unit (or range or piece) of a sequence, and how many hold it
  float2 *ml;         // [records][Hq] maximum (log2), sum
  float *o;           // [records][Hq][128]
};

inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Records: with units, two of each and one of each warp (a sequence that ends
// in the middle of a warp's range); else two of each part of each range.
inline size_t carve(Scratch *s, void *base, size_t B, size_t Hq, size_t Hkv, size_t groups,
                    size_t unit, bool may_deal) {
  const size_t records = may_deal ? 2 * kCuts * groups : 2 * (groups / unit) + groups;
  char *p = static_cast<char *>(base);
  size_t off = 0;
  auto take = [&](size_t n) { char *at = p + off; off += up256(n); return at; };
  Scratch t;
  t.taken = reinterpret_cast<int32_t *>(take(may_deal ? groups * Hkv * sizeof(int32_t) : 0));
  t.segments = reinterpret_cast<int2 *>(take(B * sizeof(int2)));
  t.ml = reinterpret_cast<float2 *>(take(records * Hq * sizeof(float2)));
  t.o = reinterpret_cast<float *>(take(records * Hq * kD * sizeof(float)));
  if (s) *s = t;
  return off;
}

struct QDecodeArgs {
  const __nv_bfloat16 *q;
  __nv_bfloat16 *out;
  const int32_t *bt, *lens;
  int B, Hq, Hkv, g, bt_stride, pages_per_block, ppb_shift, block_size, max_pages, num_blocks;
  int head_major;     // order of the pages' outer dimensions: heads, tokens
  int v_half, v_scale_half;   // where V's rows and scales lie in a stage: 0 first, 1 second
  int unit;           // warps of a unit
  int groups;         // warps that serve a KV head, a multiple of unit
  int whole;          // whether a unit takes a whole sequence
  int may_deal;       // whether the tables could hold enough to deal pieces
  float scale_log2;
  Scratch ws;
  int32_t *err;
};

VJ_DEV Split split_pages(int total, int groups, int may_deal) {
  const int n = max(min(groups, total), 1);
  return {total > 0 ? n : 0, total / n, total % n, may_deal && total / groups >= kDealt ? 1 : 0};
}
// First place of range G (no division: every warp waits for it).
VJ_DEV int first_page(int G, const Split &t) { return G * t.pages + min(G, t.more); }
VJ_DEV int range_of(int page, const Split &t) {
  const int longer = t.more * (t.pages + 1);
  return page < longer ? page / (t.pages + 1) : t.more + (page - longer) / t.pages;
}
// First page of part i (0..kCuts) of a range of `pages`: 4/5 of it, 3/25, 1/25, 1/25.
VJ_DEV int part_page(int i, int pages) {
  const int a = pages * 4 / 5, b = a + (pages - a) * 3 / 5, c = b + (pages - b) / 2;
  return i == 0 ? 0 : i == 1 ? a : i == 2 ? b : i == 3 ? c : pages;
}
VJ_DEV int range_id(int G, int h, int Hkv) { return G * Hkv + h; }
// The range, or the part of one (kCuts of a range), that holds a page.
VJ_DEV int segment_of(int page, const Split &t) {
  const int G = range_of(page, t);
  if (!t.dealt) return G;
  const int at = page - first_page(G, t), pages = first_page(G + 1, t) - first_page(G, t);
  return G * kCuts + (at >= part_page(1, pages)) + (at >= part_page(2, pages)) +
         (at >= part_page(3, pages));
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
VJ_DEV void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
               : "r"(addr)
               : "memory");
  return v;
}
VJ_DEV uint32_t lds8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
VJ_DEV float max_over_rows(float v) {        // over the lanes that share lane & 3
#pragma unroll
  for (int o = 4; o <= 16; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Places of a sequence of `pages` pages.
VJ_DEV int places_of(int pages) { return pages > 0 ? pages + kStart : 0; }

// The sequence at place s of all places, and its page there (negative: in front
// of its pages); scan[i] = places before sequence i * per.
template <int kRuns>
VJ_DEV Place locate(const QDecodeArgs &a, const int *scan, int per, int s) {
  int lo = 0;                               // last run that starts at or before s
#pragma unroll
  for (int step = kRuns / 2; step >= 1; step >>= 1) {
    if (scan[lo + step] <= s) lo += step;
  }
  Place w;
  int cum = scan[lo];
  for (w.b = lo * per;; ++w.b) {            // s lies in this run
    w.len = a.lens[w.b];
    w.np = pages_of(w.len, a.max_pages);
    const int places = places_of(w.np);
    if (s < cum + places || w.b + 1 >= a.B) break;
    cum += places;
  }
  w.p = s - cum - kStart;
  return w;
}

// Whether rows r and r + 8 of a page of V (at shared address vb) are zeros: bits 0 and 1. Not
// inlined: it is hardly ever called, and its registers are not the loop's.
template <bool kInt8>
__device__ __noinline__ uint32_t zero_rows(uint32_t vb) {
  const int r = (threadIdx.x & 31) >> 2, qd = threadIdx.x & 3;
  uint32_t zero = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 x = lds128(vb + sw128(r + 8 * i, 2 * qd)), y = lds128(vb + sw128(r + 8 * i, 2 * qd + 1));
    uint32_t any = (x.x | x.y | x.z | x.w | y.x | y.y | y.z | y.w) & (kInt8 ? ~0u : 0x7f7f7f7fu);
    any |= __shfl_xor_sync(0xffffffffu, any, 1);       // four lanes look at a row
    any |= __shfl_xor_sync(0xffffffffu, any, 2);
    zero |= any == 0 ? 1u << i : 0u;
  }
  return zero;
}

template <bool kInt8, int NT>
__global__ void __launch_bounds__(Shape<NT>::kThreads, 1)
quant_decode_kernel(const __grid_constant__ CUtensorMap tm_rows,
                    const __grid_constant__ CUtensorMap tm_scales, const QDecodeArgs a) {
  using S = Shape<NT>;
  constexpr int kStages = S::kStages, kUnit = S::kUnit;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t *scales = smem + S::kRing * kStage;
  Info *infos = reinterpret_cast<Info *>(scales + S::kRing * kScaleStage);
  uint64_t *full = reinterpret_cast<uint64_t *>(infos + S::kRing);
  Left *lefts = reinterpret_cast<Left *>(full + S::kRing);
  Split *splits = reinterpret_cast<Split *>(lefts + S::kWarps);     // [kUnits]
  Place *wholes = reinterpret_cast<Place *>(splits + S::kUnits);    // [kUnits]
  int *scan = reinterpret_cast<int *>(wholes + S::kUnits);          // [kThreads]
  int *warp_sum = scan + S::kThreads;                               // [kWarps]

  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[warp * kStages + s], 1);
    fence_mbar_init();
    if (warp == 0) { tma_prefetch_desc(&tm_rows); tma_prefetch_desc(&tm_scales); }
  }
  // nothing of the caller's is read before the kernel ahead is done (and none of
  // it by read-only loads, which need data that stands still from the launch on);
  // the combine kernel may be made ready as soon as every CTA of this one runs
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int unit = (warp / kUnit) * gridDim.x + blockIdx.x;
  const int per = (a.B + S::kThreads - 1) / S::kThreads;
  if (!a.whole) {
    // ---- places before each run of `per` sequences
    int mine = 0;
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      if (b < a.B) mine += places_of(pages_of(a.lens[b], a.max_pages));
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w) {
      const int v = warp_sum[w];
      before += w < warp ? v : 0;
      total += v;
    }
    scan[tid] = before + incl - mine;
    if (tid < S::kUnits) splits[tid] = split_pages(total, a.groups, a.may_deal);
    __syncthreads();
  } else {
    // ---- the unit's sequence, as if it were all there is
    const int b = unit / a.Hkv;
    const int len = b < a.B ? a.lens[b] : 0, pages = pages_of(len, a.max_pages);
    if (b >= a.B) return;        // the whole unit
    if (pages == 0) {
      const int i = tid % (kUnit * 32), h = unit - b * a.Hkv;
      uint4 *dst = reinterpret_cast<uint4 *>(
          a.out + (static_cast<int64_t>(b) * a.Hq + h * a.g) * kD);
      if (i < a.g * (kD / 8)) dst[i] = make_uint4(0, 0, 0, 0);
      return;
    }
    // every warp writes the same; the ranges go to the unit's first warps
    if (lane == 0) {
      wholes[warp / kUnit] = {b, 0, pages, len};
      splits[warp / kUnit] = split_pages(pages, kUnit, 0);
    }
    __syncwarp();
  }
  const Split &split = splits[warp / kUnit];
  const bool dealt = split.dealt != 0;
  const int SG = a.whole ? 0 : unit / a.Hkv;
  const int h = unit % a.Hkv;
  // where each sequence's results will lie, for the combine kernel: a run of
  // sequences a thread, spread over the CTAs
  auto tell_combine = [&]() {
    if (tid % gridDim.x != blockIdx.x) return;
    int run = scan[tid];
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      if (b >= a.B) break;
      const int pages = pages_of(a.lens[b], a.max_pages);
      int2 in = make_int2(0, 0);
      if (pages > 0) {
        const int of = dealt ? 1 : kUnit;
        in.x = segment_of(run + kStart, split) / of;
        in.y = segment_of(run + kStart + pages - 1, split) / of - in.x + 1;
      }
      a.ws.segments[b] = in;
      run += places_of(pages);
    }
  };
  if (!a.whole && SG * kUnit >= split.n && !dealt) {      // the unit has nothing to do
    tell_combine();
    return;
  }
  const int G = SG * kUnit + warp % kUnit;
  const int r = lane >> 2, qd = lane & 3;
  uint8_t *const my_ring = smem + warp * kStages * kStage;
  uint8_t *const my_scales = scales + warp * kStages * kScaleStage;
  Info *const my_info = infos + warp * kStages;
  uint64_t *const my_full = full + warp * kStages;

  // the range or piece whose pages are being issued
  int seg = dealt ? G * kCuts : G, seg_h = h, seg_at = 0, seg_end = 0, seg_first = 0;
  if (G < split.n) {
    if (dealt && lane == 0) atomicExch(a.ws.taken + range_id(G, h, a.Hkv), 0);
    seg_at = seg_first = first_page(G, split);
    seg_end = first_page(G + 1, split);
    if (dealt) seg_end = seg_at + part_page(1, seg_end - seg_at);
  }
  Page page = {};                       // lane i: the page at place i of 32
  unsigned there = 0;                   // lanes whose places have pages yet to issue
  int issued = 0;
  int own = dealt && G < split.n ? 1 : 0, misses = 0;
  auto issue = [&](int s) {             // the next page, if there is one, into stage s
    while (there == 0) {
      if (seg_at >= seg_end) {
        if (!dealt || misses >= 3) return;
        const int ranges = split.n * a.Hkv;
        int range = range_id(G, h, a.Hkv);
        if (!own) {
          // look at 32 ranges' words, a lane each, and choose one with the least taken
          range = static_cast<int>((static_cast<uint32_t>(unit * kUnit + warp + 97 * issued) * 61u +
                                    (lane + 32 * misses) * 73u) % static_cast<uint32_t>(ranges));
          const uint32_t taken = static_cast<uint32_t>(__ldcg(a.ws.taken + range));
          unsigned who = 0;
#pragma unroll
          for (uint32_t i = 0; i + 1 < kCuts; ++i) {
            const unsigned at = __ballot_sync(0xffffffffu, taken == i);
            if (who == 0) who = at;
          }
          if (who == 0) { ++misses; continue; }
          range = __shfl_sync(0xffffffffu, range, __ffs(who) - 1);
        }
        uint32_t i = 0;
        if (lane == 0) i = static_cast<uint32_t>(atomicAdd(a.ws.taken + range, 1));
        i = __shfl_sync(0xffffffffu, i, 0);
        if (i + 1 >= kCuts) {                      // none left
          if (own) own = 0; else ++misses;
          continue;
        }
        const int g = range / a.Hkv, part = static_cast<int>(i) + 1;
        seg = g * kCuts + part;
        seg_h = range - g * a.Hkv;
        const int at = first_page(g, split), pages = first_page(g + 1, split) - at;
        seg_at = seg_first = at + part_page(part, pages);
        seg_end = at + part_page(part + 1, pages);
      }
      // the next 32 places, one a lane
      const int at = seg_at + lane;
      bool has_page = false;
      if (at < seg_end) {
        Place w;
        if (a.whole) {
          w = wholes[warp / kUnit];
          w.p = at;
        } else {
          w = locate<S::kThreads>(a, scan, per, at);
        }
        has_page = w.p >= 0;
        if (has_page) {
          const int entry = a.ppb_shift >= 0 ? w.p >> a.ppb_shift : w.p / a.pages_per_block;
          const int off = (w.p - entry * a.pages_per_block) * kTok;
          int blk = a.bt[static_cast<int64_t>(w.b) * a.bt_stride + entry];
          if (blk < 0 || blk >= a.num_blocks) blk = 0;   // as the other attention kernels read it
          const bool seq_end = w.p + 1 == w.np;
          const bool end = at + 1 + (seq_end ? kStart : 0) >= seg_end;    // no page after it
          page.b = w.b;
          page.valid_flags =
              min(w.len - w.p * kTok, kTok) |
              ((w.p == 0 || at == seg_first ? kFirst : 0) | (seq_end || end ? kLast : 0) |
               (at - w.p >= seg_first ? kHead : 0) | (seq_end ? kTail : 0) | (end ? kEnd : 0)) << 8;
          page.tok = blk * a.block_size + off;
          page.blk = blk;
        }
      }
      there = __ballot_sync(0xffffffffu, has_page);
      seg_at += 32;
    }
    const int who = __ffs(there) - 1;
    there &= there - 1;
    if (lane == who) {
      my_info[s] = {page.b, page.valid_flags, seg_h, seg};
      uint8_t *dst = my_ring + s * kStage;
      mbar_arrive_expect_tx(&my_full[s], kStage + 32);
      const int c1 = a.head_major ? seg_h : page.tok, c2 = a.head_major ? page.tok : seg_h;
      tma_load_4d(dst, &tm_rows, &my_full[s], 0, c1, c2, 0);
      tma_load_4d(my_scales + s * kScaleStage, &tm_scales, &my_full[s],
                  page.tok - page.blk * a.block_size, seg_h, page.blk, 0);
    }
    ++issued;
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) issue(s);
  if (!a.whole) tell_combine();         // while the pages travel

  const uint32_t ring = smem_u32(my_ring), sc_ring = smem_u32(my_scales);
  const uint32_t v_rows = a.v_half ? kHalf : 0, v_scales = a.v_scale_half ? 16 : 0;
  uint32_t qf[NT][16];                  // Q^T fragments: dims 32*qd + 4*j + {0,1}, {2,3}
  float qs[NT][2];                      // score factor of heads 2*qd, 2*qd + 1
  float acc[NT][8][4];                  // O^T: dims 16*r + 2*i, + 1; heads 2*qd, 2*qd + 1
  // log2, negated: maximum of s; of s + ev, less kUp. Sum of p (this lane's tokens)
  float nm[NT][2], nw[NT][2], l[NT][2];
  // q of a segment's query heads (head 8*t + r, dims 32*qd .. + 31), nothing summed yet
  auto begin = [&](int b, int h) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int head = t * 8 + r;
      uint4 x[4] = {};
      if (head < a.g) {
        const uint4 *src = reinterpret_cast<const uint4 *>(
            a.q + (static_cast<int64_t>(b) * a.Hq + h * a.g + head) * kD + qd * 32);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = src[j];
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
      for (int j = 0; j < 2; ++j) { nm[t][j] = nw[t][j] = INFINITY; l[t][j] = 0.f; }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][i][j] = 0.f;
      }
    }
  };
  __syncwarp();
  if (issued > 0) begin(my_info[0].b, my_info[0].h);      // while the pages travel
  Left mine_left = {-1, 0, 0, -1};
  int stage = 0;
  uint32_t parity = 0;
  for (int it = 0; it < issued; ++it) {
    // (all lanes together: what follows are warp-wide products)
    if (!__all_sync(0xffffffffu, mbar_wait(&my_full[stage], parity))) {
      // bounded: the copies still in flight must land before the CTA ends
      for (int k = it + 1; k < issued; ++k) {
        mbar_wait(&my_full[k % kStages], (k / kStages) & 1);
      }
      if (lane == 0 && a.err != nullptr) atomicExch(a.err, 1);
      break;
    }
    const Info info = my_info[stage];
    const int seq = info.b, valid = info.valid_flags & 0xff, flags = info.valid_flags >> 8;
    const uint32_t kb = ring + stage * kStage + (kHalf - v_rows), vb = ring + stage * kStage + v_rows;
    const uint32_t ksb = sc_ring + stage * kScaleStage + (16 - v_scales);
    const uint32_t vsb = sc_ring + stage * kScaleStage + v_scales;
    if (it > 0 && (flags & kFirst)) begin(seq, info.h);
    // ---- S^T = K Q^T, two chains of sums
    float sc[NT][4];
    {
      float sa[NT][4], sz[NT][4];
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
            const uint32_t b0 = qf[t][8 * c + 2 * j], b1 = qf[t][8 * c + 2 * j + 1];
            if (c == 0 && j < 2) mma_f16_first(j ? sz[t] : sa[t], a0, a1, a2, a3, b0, b1);
            else mma_f16(j & 1 ? sz[t] : sa[t], a0, a1, a2, a3, b0, b1);
          }
        }
      }
      // tokens r, r + 8 (heads 2*qd, + 1 each), times the rows' scales
      const float ks0 = __uint_as_float(max(lds8(ksb + r) << 23, 0x00400000u));
      const float ks1 = __uint_as_float(max(lds8(ksb + r + 8) << 23, 0x00400000u));
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[t][j] = (sa[t][j] + sz[t][j]) * (j < 2 ? ks0 : ks1);
      }
    }
    const uint32_t vb0 = lds8(vsb + r), vb1 = lds8(vsb + r + 8);
    float ev0 = vb0 == 255u ? __uint_as_float(0x7fffffffu)
                                  : __uint_as_float(0x4b000000u | vb0) - 8388735.0f;   // vb0 - 127
    float ev1 = vb1 == 255u ? __uint_as_float(0x7fffffffu)
                                  : __uint_as_float(0x4b000000u | vb1) - 8388735.0f;
    // ---- arguments of the exponentials, against the running maxima
    float ap[NT][4], aw[NT][4];
    auto arguments = [&]() {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ap[t][j] = fmaf(sc[t][j], qs[t][j & 1], nm[t][j & 1]);
          aw[t][j] = fmaf(sc[t][j], qs[t][j & 1], (j < 2 ? ev0 : ev1) + nw[t][j & 1]);
        }
      }
      if (valid < kTok) {            // what lies past the context may be anything
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (r + (j < 2 ? 0 : 8) >= valid) {
#pragma unroll
            for (int t = 0; t < NT; ++t) ap[t][j] = aw[t][j] = -INFINITY;
          }
        }
      }
    };
    arguments();
    float over = -INFINITY, over_w = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        over = fmaxf(over, ap[t][j]);
        over_w = fmaxf(over_w, aw[t][j]);
      }
    }
    if (__any_sync(0xffffffffu, over > kSlack || over_w > kSlack + kUp)) {
      // rows that nothing was stored to have the scale 1, but must move no maximum: zeros
      // of that scale count with the smallest, as stored ones have it. (Looked at here alone,
      // where a maximum may move: 0 to 1% longer, 2% with 16 heads a KV head; for every
      // page 1 to 2%, and all rows of zeros here, inlined, up to 3%.)
      if (__any_sync(0xffffffffu, vb0 == kFresh || vb1 == kFresh)) {
        const uint32_t zero = zero_rows<kInt8>(vb);
        if ((zero & 1) && vb0 == kFresh) ev0 = -126.f;
        if ((zero & 2) && vb1 == kFresh) ev1 = -126.f;
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float s0 = sc[t][j] * qs[t][j], s1 = sc[t][2 + j] * qs[t][j];
          float w0 = s0 + ev0, w1 = s1 + ev1;
          if (r >= valid) s0 = w0 = -INFINITY;
          if (r + 8 >= valid) s1 = w1 = -INFINITY;
          const float top = max_over_rows(fmaxf(s0, s1)), top_w = max_over_rows(fmaxf(w0, w1));
          if (-top < nm[t][j]) {
            l[t][j] *= exp2f(-top - nm[t][j]);
            nm[t][j] = -top;
          }
          if (kUp - top_w < nw[t][j]) {
            const float f = exp2f(kUp - top_w - nw[t][j]);
#pragma unroll
            for (int i = 0; i < 8; ++i) { acc[t][i][j] *= f; acc[t][i][2 + j] *= f; }
            nw[t][j] = kUp - top_w;
          }
        }
      }
      arguments();
    }
    // ---- weights
    uint32_t wb[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int j = 0; j < 2; ++j) l[t][j] += fast_exp2(ap[t][j]) + fast_exp2(ap[t][2 + j]);
      wb[t][0] = transpose8x8(pack_f16(fast_exp2(aw[t][0]), fast_exp2(aw[t][1])));
      wb[t][1] = transpose8x8(pack_f16(fast_exp2(aw[t][2]), fast_exp2(aw[t][3])));
    }
    // ---- O^T += V^T W^T: tokens 2*qd, + 1, + 8, + 9; dims 16*r .. + 15
    {
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = lds128(vb + sw128(2 * qd + (j & 1) + (j >> 1) * 8, r));
      if (valid < kTok) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (2 * qd + (j & 1) + (j >> 1) * 8 >= valid) v[j] = make_uint4(0, 0, 0, 0);
        }
      }
      // every lane has read the stage: refill it. V is still on its way to the registers
      // here, and the copy is the async proxy's, which a barrier of the warp alone does
      // not order behind the reads: in some builds of this kernel one page in two million
      // was read while it was refilled. With the fence: none, and the same time.
      fence_proxy_async_smem();
      __syncwarp();
      issue(stage);
      const uint32_t *w0 = reinterpret_cast<const uint32_t *>(&v[0]);
      const uint32_t *w1 = reinterpret_cast<const uint32_t *>(&v[1]);
      const uint32_t *w2 = reinterpret_cast<const uint32_t *>(&v[2]);
      const uint32_t *w3 = reinterpret_cast<const uint32_t *>(&v[3]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {              // dims 16*r + 2*i, + 1
        const uint32_t sel = i & 1 ? 0x7362u : 0x5140u;
        const uint32_t y = bytes(w0[i >> 1], w1[i >> 1], sel);
        const uint32_t z = bytes(w2[i >> 1], w3[i >> 1], sel);
        const uint32_t a0 = dequant_f16x2<kInt8, false>(y), a1 = dequant_f16x2<kInt8, true>(y);
        const uint32_t a2 = dequant_f16x2<kInt8, false>(z), a3 = dequant_f16x2<kInt8, true>(z);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_f16(acc[t][i], a0, a1, a2, a3, wb[t][0], wb[t][1]);
      }
    }
    if (++stage == kStages) { stage = 0; parity ^= 1; }

    if (flags & kLast) {
      const bool whole = (flags & (kHead | kTail)) == (kHead | kTail);
      const bool end = (flags & kEnd) != 0;
      float2 *ml = nullptr;
      float *o = nullptr;
      if (!whole) {
        int64_t record = 2ll * info.segment + (flags & kHead ? 1 : 0);
        if (!dealt) {
          if (flags & kHead) {
            mine_left.b1 = seq;          // goes on behind the range: its end
          } else {
            mine_left.b0 = seq;
            mine_left.ends0 = flags & kTail;
            mine_left.far0 = !end;
          }
          record = 2ll * (a.groups / kUnit) + G;
        }
        if (!dealt && end) {             // into the ring, whose pages are all read
          o = reinterpret_cast<float *>(my_ring);
          ml = reinterpret_cast<float2 *>(o + S::kHeads * kD);
        } else {
          o = a.ws.o + (record * a.Hq + info.h * a.g) * kD;
          ml = a.ws.ml + record * a.Hq + info.h * a.g;
        }
        __syncwarp();
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float sum = l[t][j];
#pragma unroll
          for (int d = 4; d <= 16; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          const int head = t * 8 + 2 * qd + j;
          if (head >= a.g) continue;
          // maximum of s + ev less that of s, and the 2^kUp taken off
          float f = exp2f(nm[t][j] - nw[t][j]);
          if (whole) f /= sum;
          float y[16];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[2 * i] = acc[t][i][j] * f;
            y[2 * i + 1] = acc[t][i][2 + j] * f;
          }
          if (whole) {
            uint4 *dst = reinterpret_cast<uint4 *>(
                a.out + (static_cast<int64_t>(seq) * a.Hq + info.h * a.g + head) * kD + 16 * r);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              dst[i] = make_uint4(pack_bf16(y[8 * i], y[8 * i + 1]),
                                  pack_bf16(y[8 * i + 2], y[8 * i + 3]),
                                  pack_bf16(y[8 * i + 4], y[8 * i + 5]),
                                  pack_bf16(y[8 * i + 6], y[8 * i + 7]));
            }
          } else {
            float4 *dst = reinterpret_cast<float4 *>(o + head * kD + 16 * r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              dst[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
            }
            if (r == 0) ml[head] = make_float2(-nm[t][j], sum);
          }
        }
      }
    }
  }

  if (dealt) return;
  // ---- the unit joins what its warps left, in the order of the pages
  if (lane == 0) lefts[warp] = mine_left;
  named_bar_sync(1 + warp / kUnit, kUnit * 32);
  const int w0 = warp / kUnit * kUnit;
  for (int i = tid - w0 * 32; i < a.g * (kD / 4); i += kUnit * 32) {
    const int head = i / (kD / 4), d = i % (kD / 4);
    const int hq = h * a.g + head;
    bool open = false, before_unit = false;
    int b = 0;
    float m = 0.f, sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 ml, float4 y) {
      const float top = fmaxf(m, ml.x);
      const float base = top == -INFINITY ? 0.f : top;
      const float f0 = exp2f(m - base), f1 = exp2f(ml.x - base);
      m = top;
      sum = sum * f0 + ml.y * f1;
      o.x = o.x * f0 + y.x * f1; o.y = o.y * f0 + y.y * f1;
      o.z = o.z * f0 + y.z * f1; o.w = o.w * f0 + y.w * f1;
    };
    auto begin = [&](int seq, bool earlier) {
      open = true;
      before_unit = earlier;
      b = seq;
      m = -INFINITY;
      sum = 0.f;
      o = make_float4(0.f, 0.f, 0.f, 0.f);
    };
    auto partial = [&]() {
      const int64_t at = (2ll * SG + (before_unit ? 0 : 1)) * a.Hq + hq;
      if (d == 0) a.ws.ml[at] = make_float2(m, sum);
      reinterpret_cast<float4 *>(a.ws.o + at * kD)[d] = o;
    };
    for (int w = w0; w < w0 + kUnit; ++w) {
      const Left lf = lefts[w];
      const float *near_o = reinterpret_cast<const float *>(smem + w * kStages * kStage);
      const float2 *near_ml = reinterpret_cast<const float2 *>(near_o + S::kHeads * kD);
      if (lf.b0 >= 0) {
        if (!open) begin(lf.b0, true);
        const int64_t far = (2ll * (a.groups / kUnit) + SG * kUnit + w - w0) * a.Hq + hq;
        if (lf.far0) {
          add(a.ws.ml[far], reinterpret_cast<const float4 *>(a.ws.o + far * kD)[d]);
        } else {
          add(near_ml[head], reinterpret_cast<const float4 *>(near_o + head * kD)[d]);
        }
        if (lf.ends0) {
          if (before_unit) {
            partial();
          } else {
            const float inv = 1.f / sum;
            reinterpret_cast<uint2 *>(a.out + (static_cast<int64_t>(b) * a.Hq + hq) * kD)[d] =
                make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
          }
          open = false;
        }
      }
      if (lf.b1 >= 0) {
        begin(lf.b1, false);
        add(near_ml[head], reinterpret_cast<const float4 *>(near_o + head * kD)[d]);
      }
    }
    if (open) partial();
  }
}

// Joins the partial results of sequences that several units (or ranges and
// pieces) shared, and writes the zeros of empty ones. kSplit warps take a
// (sequence, query head), each every kSplit-th partial, several of them in
// flight: as many warps as fit the GPU at once, since a row's time is its chain
// of memory round trips. Launched while the decode kernel runs and held by
// griddepcontrol until that is done.
template <int kSplit>
constexpr int kCombineWarps = kSplit > 8 ? kSplit : 8;

template <int kSplit>
__global__ void __launch_bounds__(kCombineWarps<kSplit> * 32) quant_combine_kernel(const QDecodeArgs a) {
  constexpr int kWarps = kCombineWarps<kSplit>, kRows = kWarps / kSplit, kFly = kSplit > 8 ? 4 : 8;
  __shared__ float4 so[kWarps][32];
  __shared__ float sm[kWarps], sl[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % kSplit;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + warp / kSplit;
  const bool live = row < static_cast<int64_t>(a.B) * a.Hq;
  const int b = live ? static_cast<int>(row / a.Hq) : 0;
  const int head = static_cast<int>(row - static_cast<int64_t>(b) * a.Hq);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int2 in = live ? a.ws.segments[b] : make_int2(0, 1);
  const int first = in.x, count = in.y;      // records: 2 * first + 1, then 2 * (first + i)
  uint2 *dst = reinterpret_cast<uint2 *>(a.out + row * kD) + lane;
  if (count == 0 && part == 0) *dst = make_uint2(0u, 0u);
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (count > 1) {               // 1: finished in one place
    for (int i0 = part; i0 < count; i0 += kFly * kSplit) {
      float4 x[kFly];
      float2 ml[kFly];
#pragma unroll
      for (int j = 0; j < kFly; ++j) {
        const int i = i0 + j * kSplit;
        ml[j] = make_float2(-INFINITY, 0.f);
        x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < count) {
          const int64_t at = (2ll * (first + i) + (i == 0 ? 1 : 0)) * a.Hq + head;
          ml[j] = a.ws.ml[at];
          x[j] = reinterpret_cast<const float4 *>(a.ws.o + at * kD)[lane];
        }
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < kFly; ++j) top = fmaxf(top, ml[j].x);
      const float base = top == -INFINITY ? 0.f : top;
      const float c = exp2f(m - base);
      m = top;
      l *= c;
      o.x *= c; o.y *= c; o.z *= c; o.w *= c;
#pragma unroll
      for (int j = 0; j < kFly; ++j) {
        const float f = exp2f(ml[j].x - base);
        l = fmaf(f, ml[j].y, l);
        o.x = fmaf(f, x[j].x, o.x); o.y = fmaf(f, x[j].y, o.y);
        o.z = fmaf(f, x[j].z, o.z); o.w = fmaf(f, x[j].w, o.w);
      }
    }
  }
  if constexpr (kSplit > 1) {
    so[warp][lane] = o;
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
    __syncthreads();
    if (part != 0 || count < 2) return;
#pragma unroll
    for (int i = 1; i < kSplit; ++i) m = fmaxf(m, sm[warp + i]);
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kSplit; ++i) {
      const float f = exp2f(sm[warp + i] - base);
      const float4 x = so[warp + i][lane];
      l = fmaf(f, sl[warp + i], l);
      o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y);
      o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
    }
  }
  if (count < 2) return;
  const float inv = 1.f / l;
  *dst = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
}

template <int kSplit>
int launch_combine(const QDecodeArgs &a, int64_t rows, cudaStream_t stream) {
  constexpr int kRows = kCombineWarps<kSplit> / kSplit;
  return launch_dependent("vj_paged_decode_quantized", quant_combine_kernel<kSplit>,
                          dim3(static_cast<unsigned>((rows + kRows - 1) / kRows)),
                          kCombineWarps<kSplit> * 32, 0, stream, a);
}

template <bool kInt8, int NT>
int launch_decode(const CUtensorMap &tm_rows, const CUtensorMap &tm_scales, const QDecodeArgs &a, int grid,
                  cudaStream_t stream) {
  using S = Shape<NT>;
  static_assert(S::kSmem <= 227 * 1024, "shared memory");
  // the shared-memory opt-in is a per-device attribute of the kernel
  static std::atomic<bool> opted[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !opted[dev].load(std::memory_order_acquire))) {
    e = cudaFuncSetAttribute(quant_decode_kernel<kInt8, NT>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(S::kSmem));
    if (e == cudaSuccess && dev < 64) opted[dev].store(true, std::memory_order_release);
  }
  if (e != cudaSuccess) {
    return set_error(VJ_ERR_CUDA,
                     std::string("vj_paged_decode_quantized: ") + cudaGetErrorString(e));
  }
  return launch_dependent("vj_paged_decode_quantized", quant_decode_kernel<kInt8, NT>,
                          dim3(static_cast<unsigned>(grid)), S::kThreads, S::kSmem, stream, tm_rows,
                          tm_scales, a);
}

// Grid, warps of a unit and groups, from head counts and the GPU's size alone.
void decode_grid(int g, int num_kv_heads, int *grid, int *unit, int *groups) {
  const int units = g <= 8 ? Shape<1>::kUnits : Shape<2>::kUnits;      // of a CTA
  *unit = g <= 8 ? Shape<1>::kUnit : Shape<2>::kUnit;
  *grid = std::max(num_sms(), (num_kv_heads + units - 1) / units);
  *groups = *grid * units / num_kv_heads * *unit;
}

// Whether a unit takes a whole sequence, so that there is nothing to join.
bool whole_sequences(int64_t batch, int64_t num_kv_heads, int64_t table_pages, int grid, int g) {
  const int units = g <= 8 ? Shape<1>::kUnits : Shape<2>::kUnits;
  return table_pages <= kWhole && batch * num_kv_heads <= static_cast<int64_t>(grid) * units;
}

// Whether block tables this large could hold enough pages to deal pieces.
bool may_deal(int64_t batch, int64_t bt_width, int64_t block_size, int64_t groups) {
  return batch * (bt_width * block_size / kTok) / groups >= kDealt;
}

}  // namespace
}  // namespace vj

extern "C" size_t vj_paged_decode_quantized_workspace_size(int32_t batch, int32_t num_q_heads,
                                                           int32_t num_kv_heads,
                                                           int32_t head_dim, int32_t bt_width,
                                                           int32_t block_size) {
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim != vj::kD || bt_width < 0 ||
      block_size <= 0) {
    return 0;
  }
  int grid, unit, groups;
  vj::decode_grid((num_q_heads + num_kv_heads - 1) / num_kv_heads, num_kv_heads, &grid, &unit,
                  &groups);
  return vj::carve(nullptr, nullptr, batch, num_q_heads, num_kv_heads, groups, unit,
                   vj::may_deal(batch, bt_width, block_size, groups));
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
  // places are counted in 32 bits, and looked up 32 at a time
  if (static_cast<int64_t>(batch) * (table_pages + kStart) > INT32_MAX - 64 ||
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
      vj_paged_decode_quantized_workspace_size(batch, num_q_heads, num_kv_heads, head_dim, bt_width,
                                               block_size);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
    return set_error(VJ_ERR_WORKSPACE, what + ": workspace needs " + std::to_string(need) +
                                           " bytes, 16-byte aligned");
  }
  // one map for the rows of K and V, one for their scales: the fourth dimension
  // leads from the lower address to the higher one
  CUtensorMap tm_rows, tm_scales;
  const uint64_t ntok = static_cast<uint64_t>(num_blocks) * block_size, hkv = num_kv_heads;
  const bool head_major = stride_head < stride_token;    // outer dims in the order of strides
  auto apart = [](const void *x, const void *y) {
    const auto p = reinterpret_cast<uintptr_t>(x), r = reinterpret_cast<uintptr_t>(y);
    return static_cast<uint64_t>(p < r ? r - p : p - r);
  };
  const uint64_t rows_apart = apart(k_cache, v_cache), scales_apart = apart(k_scales, v_scales);
  if (rows_apart == 0 || scales_apart == 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": K and V must not be the same memory");
  }
  if (rows_apart >= (1ull << 40) || scales_apart >= (1ull << 40)) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": K and V lie 2^40 bytes apart or more");
  }
  // a sequence's q is read again after another part of its results is written
  const uint64_t rows_bytes = static_cast<uint64_t>(batch) * num_q_heads * kD * 2;
  if (apart(q, out) < rows_bytes) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": out must not overlap q");
  }
  a.v_half = v_cache > k_cache ? 1 : 0;
  a.v_scale_half = v_scales > k_scales ? 1 : 0;
  const uint64_t st = stride_token, sh = stride_head;
  const uint32_t box_tok = kTok;
  rc = head_major
           ? encode_tmap_4d_u8(&tm_rows, a.v_half ? k_cache : v_cache, {kD, hkv, ntok, 2},
                               {sh, st, rows_apart}, {kD, 1, box_tok, 2}, true)
           : encode_tmap_4d_u8(&tm_rows, a.v_half ? k_cache : v_cache, {kD, ntok, hkv, 2},
                               {st, sh, rows_apart}, {kD, box_tok, 1, 2}, true);
  if (rc) return rc;
  rc = encode_tmap_4d_u8(
      &tm_scales, a.v_scale_half ? k_scales : v_scales,
      {static_cast<uint64_t>(block_size), hkv, static_cast<uint64_t>(num_blocks), 2},
      {static_cast<uint64_t>(scale_stride_head), static_cast<uint64_t>(scale_stride_block),
       scales_apart},
      {box_tok, 1, 1, 2}, false);
  if (rc) return rc;
  a.q = static_cast<const __nv_bfloat16 *>(q);
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.bt = block_tables;
  a.lens = context_lens;
  a.B = batch;
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.g = num_q_heads / num_kv_heads;
  a.bt_stride = bt_stride;
  a.pages_per_block = block_size / kTok;
  a.ppb_shift = (a.pages_per_block & (a.pages_per_block - 1)) == 0
                    ? __builtin_ctz(a.pages_per_block) : -1;
  a.block_size = block_size;
  a.max_pages = static_cast<int>(table_pages);
  a.num_blocks = static_cast<int>(num_blocks);
  a.head_major = head_major ? 1 : 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = error_flag;
  int grid;
  decode_grid(a.g, num_kv_heads, &grid, &a.unit, &a.groups);
  a.whole = whole_sequences(batch, num_kv_heads, table_pages, grid, a.g) ? 1 : 0;
  a.may_deal = !a.whole && may_deal(batch, bt_width, block_size, a.groups) ? 1 : 0;
  carve(&a.ws, workspace, batch, num_q_heads, num_kv_heads, a.groups, a.unit, a.may_deal != 0);
  const bool i8 = cache_dtype == VJ_CACHE_INT8;
  if (a.g <= 8) {
    rc = i8 ? launch_decode<true, 1>(tm_rows, tm_scales, a, grid, stream)
            : launch_decode<false, 1>(tm_rows, tm_scales, a, grid, stream);
  } else {
    rc = i8 ? launch_decode<true, 2>(tm_rows, tm_scales, a, grid, stream)
            : launch_decode<false, 2>(tm_rows, tm_scales, a, grid, stream);
  }
  if (rc || a.whole) return rc;
  const int64_t rows = static_cast<int64_t>(batch) * num_q_heads;
  // warps that can be resident at once: 32 an SM at this kernel's registers
  const int64_t room = 32ll * num_sms();
  rc = rows * 32 <= room  ? launch_combine<32>(a, rows, stream)
       : rows * 8 <= room ? launch_combine<8>(a, rows, stream)
       : rows * 4 <= room ? launch_combine<4>(a, rows, stream)
       : rows * 2 <= room ? launch_combine<2>(a, rows, stream)
                          : launch_combine<1>(a, rows, stream);
  if (rc) return rc;
  return check_launch("vj_paged_decode_quantized");
}
