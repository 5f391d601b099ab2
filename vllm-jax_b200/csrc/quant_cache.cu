// Quantised KV cache: the store (q/k RMSNorm + RoPE + rounding of k and v to 8
// bits, in one launch) and the read-back to bf16.
//
// Store, per token and head row x of 128:
//   y = rope(x * w / sqrt(mean(x^2) + eps))        (q and k; v: y = x)
//   q_out = bf16(y)
//   e = smallest integer with max|y| <= qmax * 2^e;  cached = RN8(y * 2^-e), byte e + 127
// A cached row is the correctly rounded one, whatever order a sum was taken in,
// so two programs (or two ranks, or a recomputed prefix) that cache the same
// token hold the same bytes. For k that takes more than 32 bits near a rounding
// border: a row is computed in 32 bits, and again in 64 where one of its
// elements lies so close to a border that 32 bits do not decide (about one
// step of four rows in a hundred).
#include "kv_row.cuh"
#include "quant.cuh"

#include <algorithm>
#include <atomic>

namespace vj {
namespace {
using namespace qn;

struct StoreArgs {
  const __nv_bfloat16 *q, *k, *v, *qw, *kw;
  const int32_t *positions, *slots;
  __nv_bfloat16 *q_out;
  const uint4 *table;
  Pool pool;
  int64_t num_tokens;
  int parts, rows;        // units of a token, head rows of a unit (a multiple of 4)
  int step_t, step_part;  // from a warp's unit to its next one: tokens, and units
  int bs_shift;           // log2 of the block size, or -1
  int Hq, Hkv, table_len;
  int64_t qrs, krs, vrs, qors;
  double eps;
  bool norm, rope;
  int32_t *err;
  RopeTable freq;
};

VJ_DEV uint32_t group_max(unsigned mask, uint32_t v) {
#pragma unroll
  for (int o = 4; o >= 1; o >>= 1) v = max(v, __shfl_xor_sync(mask, v, o));
  return v;
}


// What turns and weighs the pairs (2i, 2i + 1) of a row, two pairs a word:
//   y0 = (x0 * w0 c - x1 * w1 s) / rms,  y1 = (x0 * w0 s + x1 * w1 c) / rms
// Products of two bf16 numbers are exact in 32 bits.
struct Turn {
  uint64_t a[4], nb[4], c[4], d[4];     // w0 c, -w1 s, w0 s, w1 c
};

VJ_DEV Turn make_turn(const RowSlice &w, const RowSlice &cs) {
  Turn t;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t w0 = f32x2(bf16_lo(w.w[2 * j]), bf16_lo(w.w[2 * j + 1]));
    const uint64_t w1 = f32x2(bf16_hi(w.w[2 * j]), bf16_hi(w.w[2 * j + 1]));
    const uint64_t c = f32x2(bf16_lo(cs.w[2 * j]), bf16_lo(cs.w[2 * j + 1]));
    const uint64_t s = f32x2(bf16_hi(cs.w[2 * j]), bf16_hi(cs.w[2 * j + 1]));
    const uint64_t ns = f32x2(-bf16_hi(cs.w[2 * j]), -bf16_hi(cs.w[2 * j + 1]));
    t.a[j] = f32x2_mul(w0, c);
    t.nb[j] = f32x2_mul(w1, ns);
    t.c[j] = f32x2_mul(w0, s);
    t.d[j] = f32x2_mul(w1, c);
  }
  return t;
}

// A row turned and normalised in 32 bits: elements 2i of the lane's 8 pairs in
// u, 2i + 1 in z. Relative error below 12.5 * 2^-24: the sum of squares adds
// 128 exact squares in at most 11 roundings, then eps (its own cast and one
// more), which the root halves to 6.25; rsqrtf 4, the turn 1 (its products are
// exact), the last product 1. That holds where decided_range() does. Returns 1 / rms.
VJ_DEV float turn_row(uint64_t (&u)[4], uint64_t (&z)[4], const RowSlice &x, const Turn &t,
                     unsigned mask, const StoreArgs &a) {
  uint64_t x0[4], x1[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x0[j] = f32x2(bf16_lo(x.w[2 * j]), bf16_lo(x.w[2 * j + 1]));
    x1[j] = f32x2(bf16_hi(x.w[2 * j]), bf16_hi(x.w[2 * j + 1]));
  }
  float inv = 1.0f;
  if (a.norm) {
    uint64_t s2 = f32x2_mul(x0[0], x0[0]);
    s2 = f32x2_fma(x1[0], x1[0], s2);
#pragma unroll
    for (int j = 1; j < 4; ++j) s2 = f32x2_fma(x1[j], x1[j], f32x2_fma(x0[j], x0[j], s2));
    float ss, hi;
    f32x2_split(s2, ss, hi);
    ss += hi;
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    inv = rsqrtf(fmaf(ss, 1.0f / kD, static_cast<float>(a.eps)));
  }
  const uint64_t inv2 = f32x2(inv, inv);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    u[j] = f32x2_mul(x0[j], t.a[j]);
    z[j] = f32x2_mul(x1[j], t.d[j]);
    if (a.rope) {
      u[j] = f32x2_fma(x1[j], t.nb[j], u[j]);
      z[j] = f32x2_fma(x0[j], t.c[j], z[j]);
    }
    u[j] = f32x2_mul(u[j], inv2);
    z[j] = f32x2_mul(z[j], inv2);
  }
  return inv;
}
// Whether nothing of a row in turn_row has left the range of 32 bits so far that its bound
// fails: 1 / rms in 2^-40 .. 2^20 (squares of a mean above 2^-40 that are subnormal, off by
// 2^-150 each, do not count in it), the result's largest magnitude in 2^-80 .. 2^120 (before
// the last product it is then above 2^-100, against which subnormal products, off by 2^-149,
// do not count either), and no negative eps that the mean square cancels with.
VJ_DEV bool decided_range(float inv, uint32_t amax_bits, const StoreArgs &a) {
  return inv >= 0x1p-40f && inv <= 0x1p20f && amax_bits >= (47u << 23) &&
         amax_bits < (247u << 23) && (!a.norm || a.eps >= 0.0);
}

// One row of q: rounded to bf16 at the end.
VJ_DEV RowSlice q_row(const RowSlice &x, const Turn &t, unsigned mask, const StoreArgs &a) {
  uint64_t u[4], z[4];
  turn_row(u, z, x, t, mask, a);
  RowSlice o;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float u0, u1, z0, z1;
    f32x2_split(u[j], u0, u1);
    f32x2_split(z[j], z0, z1);
    o.w[2 * j] = cvt_bf16x2(u0, z0);
    o.w[2 * j + 1] = cvt_bf16x2(u1, z1);
  }
  return o;
}

// High word of a double with its last bit set if the low word is not 0: enough
// to compare with any number of 20 bits.
VJ_DEV uint32_t high_word(double y) {
  return static_cast<uint32_t>(__double2hiint(y)) | min(static_cast<uint32_t>(__double2loint(y)), 1u);
}

// 24 bits of y, truncated, with the last bit set if anything was cut off:
// rounding that to 8 bits equals rounding y itself. |y| below 2^-126 becomes a
// zero (it rounds to one: the smallest step of an element is 2^-9).
VJ_DEV float round_to_odd(double y) {
  const uint32_t hi = static_cast<uint32_t>(__double2hiint(y)), lo = static_cast<uint32_t>(__double2loint(y));
  const uint32_t mag = hi & 0x7fffffffu;
  uint32_t f = __funnelshift_l(lo, mag - (896u << 20), 3) | min(lo & 0x1fffffffu, 1u);
  if (mag < (897u << 20)) f = 0u;
  return __uint_as_float(f | (hi & 0x80000000u));
}

// One row of k in 64 bits. Leaves the elements times 2^-e. Not inlined: its
// registers are not the other rows'.
struct Scaled {
  float v[16];
  int e;
  bool bad;        // an infinity or NaN in the row
};

template <bool kInt8>
__device__ __noinline__ Scaled k_row_64(const uint8_t *row, const __nv_bfloat16 *kw, RowSlice cs,
                                       unsigned mask, double eps, bool norm, bool rope) {
  const int l8 = threadIdx.x & 7;
  const RowSlice x = load_slice(row, l8);
  RowSlice w = {};
  if (norm) w = load_slice(kw, l8);
  Scaled r;
  double y[16];
#pragma unroll
  for (int j = 0; j < 8; ++j) { y[2 * j] = bf16_lo(x.w[j]); y[2 * j + 1] = bf16_hi(x.w[j]); }
  double inv = 1.0;
  if (norm) {
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < 16; ++j) ss = fma(y[j], y[j], ss);
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    const double ms = ss * (1.0 / kD) + eps;
    const float m32 = static_cast<float>(ms);
    if (m32 > 1e-30f && m32 < 1e30f) {
      // 22 bits, and two Newton steps: 1.5 r - 0.5 ms r^3
      inv = static_cast<double>(rsqrtf(m32));
#pragma unroll
      for (int i = 0; i < 2; ++i) inv = inv * fma(-0.5 * ms * inv, inv, 1.5);
    } else {
      inv = 1.0 / sqrt(ms);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    double u = y[2 * j] * inv, z = y[2 * j + 1] * inv;
    if (norm) {
      u *= bf16_lo(w.w[j]);
      z *= bf16_hi(w.w[j]);
    }
    if (rope) {
      const double c = bf16_lo(cs.w[j]), s = bf16_hi(cs.w[j]);
      const double t = fma(u, c, -(z * s));
      z = fma(u, s, z * c);
      u = t;
    }
    y[2 * j] = u;
    y[2 * j + 1] = z;
    top = max(top, max(high_word(u) & 0x7fffffffu, high_word(z) & 0x7fffffffu));
  }
  top = group_max(mask, top);
  r.bad = top >= 0x7ff00000u;
  // scale_exponent of the row: the exponent, and 20 bits of the fraction
  const int ex = static_cast<int>(top >> 20) - 1023;
  const uint32_t frac = top & 0xfffffu;
  int e = kInt8 ? ex - 6 + (frac > 0xfc000u ? 1 : 0) : ex - 8 + (frac > 0xc0000u ? 1 : 0);
  r.e = e = r.bad ? 0 : max(e, -126);
  const double f = __hiloint2double((1023 - e) << 20, 0);      // 2^-e
#pragma unroll
  for (int j = 0; j < 16; ++j) r.v[j] = round_to_odd(y[j] * f);
  return r;
}


// Sixteen elements as four words of the cache.
template <bool kInt8>
VJ_DEV void quantise16(uint32_t (&o)[4], const float (&v)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    o[j] = quantise2<kInt8>(v[4 * j], v[4 * j + 1]) |
           quantise2<kInt8>(v[4 * j + 2], v[4 * j + 3]) << 16;
  }
}

// One row of k, quantised: 32 bits where they decide the rounding, else 64. What 32
// bits give is off by less than 2^-20 of itself, so they decide where an element made
// larger and smaller by that rounds to the same.
template <bool kInt8>
VJ_DEV void k_row(uint32_t (&o)[4], int &e, bool &bad, const uint8_t *row, const RowSlice &cs,
                  const Turn &t, unsigned mask, const StoreArgs &a) {
  uint64_t u[4], z[4];
  const float inv = turn_row(u, z, load_slice(row, threadIdx.x & 7), t, mask, a);
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x0, x1, y0, y1;
    f32x2_split(u[j], x0, x1);
    f32x2_split(z[j], y0, y1);
    amax = max(max(amax, max(__float_as_uint(x0) & 0x7fffffffu, __float_as_uint(x1) & 0x7fffffffu)),
               max(__float_as_uint(y0) & 0x7fffffffu, __float_as_uint(y1) & 0x7fffffffu));
  }
  amax = group_max(mask, amax);
  bad = false;
  e = scale_exponent<kInt8>(amax);
  const float f = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);   // 2^-e
  // undecided too: rows out of 32 bits' range, and the largest element next to where the
  // exponent moves
  bool open = !decided_range(inv, amax, a) ||
              __usad(amax & 0x7fffffu, kInt8 ? 0x7e0000u : 0x600000u, 0u) <= 16u;
  const uint64_t up = f32x2(f * (1.f + 0x1p-20f), f * (1.f + 0x1p-20f));
  const uint64_t down = f32x2(f * (1.f - 0x1p-20f), f * (1.f - 0x1p-20f));
  uint32_t apart = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a0, a1, b0, b1, c0, c1, d0, d1;
    f32x2_split(f32x2_mul(u[j], up), a0, a1);
    f32x2_split(f32x2_mul(z[j], up), b0, b1);
    f32x2_split(f32x2_mul(u[j], down), c0, c1);
    f32x2_split(f32x2_mul(z[j], down), d0, d1);
    o[j] = quantise2<kInt8>(a0, b0) | quantise2<kInt8>(a1, b1) << 16;
    apart |= o[j] ^ (quantise2<kInt8>(c0, d0) | quantise2<kInt8>(c1, d1) << 16);
  }
  if (__any_sync(mask, open || apart != 0u)) {
    const Scaled r = k_row_64<kInt8>(row, a.kw, cs, mask, a.eps, a.norm, a.rope);
    quantise16<kInt8>(o, r.v);
    e = r.e;
    bad = r.bad;
  }
}

// HBM-bound: each head row is read and written once, a token's RoPE row once
// per unit. A unit is up to 32 neighbouring head rows of one token. A warp
// takes units in turn through a ring of its own in shared memory, filled by
// bulk copies (the unit's q, k and v rows and the token's RoPE row, at most
// four copies) a unit ahead: 8 KB a warp, 100 KB an SM in flight, which
// registers could not hold (loads three steps ahead: 4.2 TB/s). Fewer warps
// with enough registers beat more that spill, since the shared memory taken
// leaves next to no L1 for spills (12 warps, 150 registers: 5.9 TB/s; 16 of
// 128: 3.7). 8 lanes own a row: lane l8 holds dims [8*l8, +8) and [64 + 8*l8,
// +8).
constexpr int kStoreWarps = 12;
constexpr int kStoreCtas = 1;        // of an SM
constexpr int kUnitRows = 32;
constexpr int kUnitBytes = (kUnitRows + 1) * 256;      // and the RoPE row
constexpr int kUnitStages = 2;
constexpr int kStoreSmem = kStoreWarps * kUnitStages * (kUnitBytes + 8 + 8);

VJ_DEV RowSlice ones() {
  RowSlice w;
#pragma unroll
  for (int j = 0; j < 8; ++j) w.w[j] = 0x3f803f80u;
  return w;
}

template <bool kInt8>
__global__ void __launch_bounds__(kStoreWarps * 32, kStoreCtas)
kv_store_quantized_kernel(const StoreArgs a) {
  extern __shared__ __align__(128) uint8_t store_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int l8 = lane & 7, grp = lane >> 3;
  const unsigned mask = 0xffu << (8 * grp);
  uint8_t *const ring = store_smem + warp * kUnitStages * kUnitBytes;
  uint64_t *const full =
      reinterpret_cast<uint64_t *>(store_smem + kStoreWarps * kUnitStages * kUnitBytes) +
      warp * kUnitStages;
  int2 *const meta = reinterpret_cast<int2 *>(full + (kStoreWarps - warp) * kUnitStages) +
                     warp * kUnitStages;                   // position, slot
  const int heads = a.Hq + 2 * a.Hkv;
  // a warp's units: number `warp * gridDim.x + blockIdx.x` and every
  // gridDim.x * kStoreWarps-th from there, as token and part (counted, not
  // divided: a 64-bit division costs as much as a row)
  const int first = warp * gridDim.x + blockIdx.x;
  int64_t t = first / a.parts;
  int part = first - static_cast<int>(t) * a.parts;
  asm volatile("griddepcontrol.wait;" ::: "memory");    // the kernel ahead is done
  if (t >= a.num_tokens) return;
  auto advance = [&](int64_t &t, int &part) {
    t += a.step_t;
    part += a.step_part;
    if (part >= a.parts) { part -= a.parts; ++t; }
  };
  if (lane == 0) {
    for (int s = 0; s < kUnitStages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  __syncwarp();

  // the next unit to copy, and its token's position and slot (read one ahead)
  int64_t in_t = t;
  int in_part = part, sent = 0;
  auto read_at = [&]() {
    if (in_t >= a.num_tokens) return make_int2(0, 0);
    return make_int2(a.rope ? a.positions[in_t] : 0, a.slots[in_t]);
  };
  int2 at = read_at();
  auto issue = [&](int s) {
    if (in_t >= a.num_tokens) return;
    const int r0 = in_part * a.rows, r1 = min(r0 + a.rows, heads);
    const bool turned = a.rope && r0 < a.Hq + a.Hkv && at.x >= 0 && at.x < a.table_len;
    uint8_t *dst = ring + s * kUnitBytes;
    if (lane == 0) {
      meta[s] = at;
      mbar_arrive_expect_tx(&full[s], (r1 - r0) * 256 + (turned ? 256 : 0));
    }
    __syncwarp();
    if (lane < 3) {              // lane 0: q rows, 1: k rows, 2: v rows
      const int lo = lane == 0 ? 0 : lane == 1 ? a.Hq : a.Hq + a.Hkv;
      const int from = max(r0, lo);
      const int to = min(r1, lane == 0 ? a.Hq : lane == 1 ? a.Hq + a.Hkv : heads);
      const __nv_bfloat16 *src = lane == 0 ? a.q + in_t * a.qrs
                                 : lane == 1 ? a.k + in_t * a.krs : a.v + in_t * a.vrs;
      if (from < to) {
        bulk_g2s(dst + (from - r0) * 256, src + static_cast<int64_t>(from - lo) * kD,
                 (to - from) * 256, &full[s]);
      }
    } else if (lane == 3 && turned) {
      bulk_g2s(dst + kUnitRows * 256, a.table + static_cast<int64_t>(at.x) * 16, 256, &full[s]);
    }
    ++sent;
    advance(in_t, in_part);
    at = read_at();
  };
#pragma unroll
  for (int s = 0; s < kUnitStages; ++s) issue(s);

  int s = 0;
  uint32_t parity = 0;
#pragma unroll 1
  for (int it = 0; it < sent; ++it) {
    if (!mbar_wait(&full[s], parity)) {
      // bounded: the copies still in flight must land before the CTA ends
      for (int i = it + 1; i < sent; ++i) {
        if (++s == kUnitStages) { s = 0; parity ^= 1; }
        mbar_wait(&full[s], parity);
      }
      if (lane == 0 && a.err != nullptr) atomicExch(a.err, 1);
      return;
    }
    const uint8_t *unit = ring + s * kUnitBytes;
    const int r0 = part * a.rows, r1 = min(r0 + a.rows, heads);
    const int pos = meta[s].x;
    const int slot = meta[s].y;
    RowSlice cs;
    if (!a.rope) {
#pragma unroll
      for (int j = 0; j < 8; ++j) cs.w[j] = 0x3f80u;       // cos 1, sin 0
    } else if (pos >= 0 && pos < a.table_len) {
      cs = load_slice(unit + kUnitRows * 256, l8);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs.w[j] = rope_word(pos, a.freq.inv_freq[(j < 4 ? 0 : 32) + l8 * 4 + (j & 3)]);
      }
    }
    int h = r0 + grp;
    if (h < a.Hq) {
      const Turn turn = make_turn(a.norm ? load_slice(a.qw, l8) : ones(), cs);
      __nv_bfloat16 *out = a.q_out + t * a.qors;
#pragma unroll 4
      for (; h < min(r1, a.Hq); h += 4) {
        stg_slice(out + h * kD, l8, q_row(load_slice(unit + (h - r0) * 256, l8), turn, mask, a),
                  true);
      }
    }
    const bool stored = slot >= 0 && slot < a.pool.num_blocks * a.pool.block_size;
    const int blk = a.bs_shift >= 0 ? slot >> a.bs_shift : slot / a.pool.block_size;
    const int64_t off = slot - blk * a.pool.block_size;
    Turn turn = {};
    if (stored && h < a.Hq + a.Hkv) turn = make_turn(a.norm ? load_slice(a.kw, l8) : ones(), cs);
#pragma unroll 1
    for (; stored && h < r1; h += 4) {
      const bool is_v = h >= a.Hq + a.Hkv;
      const int hk = is_v ? h - a.Hq - a.Hkv : h - a.Hq;
      uint32_t o[4];
      int e;
      bool bad;                            // an infinity or NaN in the row
      if (is_v) {
        const RowSlice x = load_slice(unit + (h - r0) * 256, l8);
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          amax = max(amax, max((x.w[j] << 16) & 0x7fffffffu, x.w[j] & 0x7fff0000u));
        }
        amax = group_max(mask, amax);
        bad = amax >= 0x7f800000u;
        e = bad ? 0 : scale_exponent<kInt8>(amax);
        const float f = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);   // 2^-e
        float y[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          y[2 * j] = bf16_lo(x.w[j]) * f;
          y[2 * j + 1] = bf16_hi(x.w[j]) * f;
        }
        quantise16<kInt8>(o, y);
      } else {
        k_row<kInt8>(o, e, bad, unit + (h - r0) * 256, cs, turn, mask, a);
      }
      if (bad) o[0] = o[1] = o[2] = o[3] = 0u;
      uint8_t *row = (is_v ? a.pool.v : a.pool.k) + blk * a.pool.sb + off * a.pool.st +
                     hk * a.pool.sh + l8 * 8;
      *reinterpret_cast<uint2 *>(row) = make_uint2(o[0], o[1]);
      *reinterpret_cast<uint2 *>(row + 64) = make_uint2(o[2], o[3]);
      if (l8 == 0) {
        uint8_t *sc = (is_v ? a.pool.vs : a.pool.ks) + blk * a.pool.ssb + hk * a.pool.ssh + off;
        *sc = bad ? 255 : static_cast<uint8_t>(e + 127);
      }
    }
    // every lane has read the unit: refill its stage (the copy is the async proxy's, and
    // the fence orders the reads before it)
    fence_proxy_async_smem();
    __syncwarp();
    issue(s);
    if (++s == kUnitStages) { s = 0; parity ^= 1; }
    advance(t, part);
  }
}

// Whether T rows of `out` (out_w elements, out_s from one to the next) may share memory with
// those of x: not where the one is the other (a unit reads its rows before it writes them),
// nor where they are separate columns of one buffer's rows.
bool rows_overlap(const void *out, int64_t out_w, int64_t out_s, const void *x, int64_t x_w,
                  int64_t x_s, int64_t T, bool may_be_same) {
  const auto o = reinterpret_cast<uintptr_t>(out), p = reinterpret_cast<uintptr_t>(x);
  const uint64_t out_bytes = ((T - 1) * out_s + out_w) * 2, x_bytes = ((T - 1) * x_s + x_w) * 2;
  if (o < p ? p - o >= out_bytes : o - p >= x_bytes) return false;
  if (T == 1) return !(may_be_same && o == p);
  if (out_s != x_s || (o - p) % 2 != 0) return true;
  if (o == p) return !may_be_same;
  int64_t column = (static_cast<int64_t>(o - p) / 2) % x_s;       // of out in x's rows
  if (column < 0) column += x_s;
  return column < x_w || column + out_w > x_s;
}

template <bool kInt8>
int launch_store(const StoreArgs &a, unsigned grid, cudaStream_t stream) {
  // the shared-memory opt-in is a per-device attribute of the kernel
  static std::atomic<bool> opted[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !opted[dev].load(std::memory_order_acquire))) {
    e = cudaFuncSetAttribute(kv_store_quantized_kernel<kInt8>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, kStoreSmem);
    if (e == cudaSuccess) {
      e = cudaFuncSetAttribute(kv_store_quantized_kernel<kInt8>,
                               cudaFuncAttributePreferredSharedMemoryCarveout,
                               cudaSharedmemCarveoutMaxShared);
    }
    if (e == cudaSuccess && dev < 64) opted[dev].store(true, std::memory_order_release);
  }
  if (e != cudaSuccess) {
    return set_error(VJ_ERR_CUDA, std::string("vj_kv_store_quantized: ") + cudaGetErrorString(e));
  }
  return launch_dependent("vj_kv_store_quantized", kv_store_quantized_kernel<kInt8>, dim3(grid),
                          kStoreWarps * 32, kStoreSmem, stream, a);
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
  uint32_t Hkv_magic;   // r / Hkv = umulhi(r, magic) for r < 2^16 and Hkv > 1
};

constexpr int kReadThreads = 256;
constexpr int kReadTok = 16;   // tokens of one CTA (within one block)
constexpr int kReadFly = 4;    // rows that a group of lanes has in flight

// HBM-bound. blockIdx.z: K or V.
template <bool kInt8>
__global__ void __launch_bounds__(kReadThreads) kv_read_quantized_kernel(const ReadArgs a) {
  const int b = blockIdx.y;
  const int t0 = blockIdx.x * kReadTok;
  asm volatile("griddepcontrol.wait;" ::: "memory");    // the kernel ahead is done
  const int len = min(min(a.lens[b], a.max_tokens), a.max_len);
  int end = a.max_len;          // rows [len, end) are zeroed
  if (a.zero_to > 0) {
    const int64_t up = (static_cast<int64_t>(max(len, 1)) + a.zero_to - 1) / a.zero_to * a.zero_to;
    if (up < end) end = static_cast<int>(up);
  }
  const int nt = min(kReadTok, end - t0);
  if (nt <= 0) return;
  int64_t blk = 0;
  if (t0 < len) {
    blk = a.bt[static_cast<int64_t>(b) * a.bt_stride + t0 / a.pool.block_size];
    if (blk < 0 || blk >= a.pool.num_blocks) blk = 0;
  }
  const int off0 = t0 % a.pool.block_size;
  const bool is_v = blockIdx.z != 0;
  const int l16 = threadIdx.x & 15;
  const uint8_t *src = (is_v ? a.pool.v : a.pool.k) + blk * a.pool.sb + off0 * a.pool.st + l16 * 8;
  const uint8_t *scales = (is_v ? a.pool.vs : a.pool.ks) + blk * a.pool.ssb + off0;
  __nv_bfloat16 *dst = (is_v ? a.v_out : a.k_out) +
                       (static_cast<int64_t>(b) * a.max_len + t0) * a.Hkv * kD + l16 * 8;
  const int rows = nt * a.Hkv, live = max(0, min(nt, len - t0)) * a.Hkv;
  constexpr int kStep = kReadThreads / 16;
  for (int r0 = threadIdx.x >> 4; r0 < rows; r0 += kStep * kReadFly) {
    uint2 w[kReadFly];
    uint32_t sc[kReadFly];
#pragma unroll
    for (int j = 0; j < kReadFly; ++j) {
      const int r = r0 + j * kStep;
      w[j] = make_uint2(0u, 0u);
      sc[j] = 127u;
      if (r < live) {
        const int tt = a.Hkv == 1 ? r : static_cast<int>(__umulhi(r, a.Hkv_magic));
        const int h = r - tt * a.Hkv;
        w[j] = __ldcs(reinterpret_cast<const uint2 *>(src + tt * a.pool.st + h * a.pool.sh));
        sc[j] = scales[h * a.pool.ssh + tt];
      }
    }
#pragma unroll
    for (int j = 0; j < kReadFly; ++j) {
      const int r = r0 + j * kStep;
      if (r >= rows) break;
      uint4 o = make_uint4(0u, 0u, 0u, 0u);
      if (r < live) {
        const float s = scale_of(sc[j]);
        const float2 f0 = f16x2_to_f32(dequant_f16x2<kInt8, false>(w[j].x));
        const float2 f1 = f16x2_to_f32(dequant_f16x2<kInt8, true>(w[j].x));
        const float2 f2 = f16x2_to_f32(dequant_f16x2<kInt8, false>(w[j].y));
        const float2 f3 = f16x2_to_f32(dequant_f16x2<kInt8, true>(w[j].y));
        o = make_uint4(cvt_bf16x2(f0.x * s, f0.y * s), cvt_bf16x2(f1.x * s, f1.y * s),
                       cvt_bf16x2(f2.x * s, f2.y * s), cvt_bf16x2(f3.x * s, f3.y * s));
      }
      *reinterpret_cast<uint4 *>(dst + static_cast<int64_t>(r) * kD) = o;
    }
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
    int32_t *error_flag, cudaStream_t stream) {
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
  if (num_q_heads > 0) {
    const int64_t qw = static_cast<int64_t>(num_q_heads) * kD, kw = static_cast<int64_t>(num_kv_heads) * kD;
    if (rows_overlap(q_out, qw, a.qors, q_in, qw, a.qrs, num_tokens, true) ||
        rows_overlap(q_out, qw, a.qors, k_in, kw, a.krs, num_tokens, false) ||
        rows_overlap(q_out, qw, a.qors, v_in, kw, a.vrs, num_tokens, false)) {
      return set_error(VJ_ERR_INVALID_ARGUMENT,
                       std::string(what) + ": q_out must be q (with its row stride) or not overlap q, k, v");
    }
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
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.eps = eps;
  a.err = error_flag;
  // 64 powers on the host take longer than the launch: kept for the last theta
  static thread_local float freq_theta = -1.0f;
  static thread_local RopeTable freq;
  if (rope_theta != freq_theta) {
    build_rope_table(rope_theta, freq.inv_freq);
    freq_theta = rope_theta;
  }
  a.freq = freq;
  // units of 32 rows; smaller ones while those would leave half the warps without
  // one (257 tokens of 48 rows: 5.3 us; down to one for every warp 6.2)
  const int64_t warps = static_cast<int64_t>(num_sms()) * kStoreCtas * kStoreWarps;
  a.rows = kUnitRows;
  while (a.rows > 4 && num_tokens * ((heads + a.rows - 1) / a.rows) < warps / 2) a.rows /= 2;
  a.parts = static_cast<int>((heads + a.rows - 1) / a.rows);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(
      num_tokens * a.parts, static_cast<int64_t>(num_sms()) * kStoreCtas));
  a.num_tokens = num_tokens;
  a.step_t = static_cast<int>(grid * kStoreWarps) / a.parts;
  a.step_part = static_cast<int>(grid * kStoreWarps) % a.parts;
  a.bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  return cache_dtype == VJ_CACHE_INT8 ? launch_store<true>(a, grid, stream)
                                      : launch_store<false>(a, grid, stream);
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
  a.Hkv_magic = static_cast<uint32_t>(((1ull << 32) + num_kv_heads - 1) / num_kv_heads);
  a.bt_stride = bt_stride;
  a.max_tokens = static_cast<int>(
      std::min<int64_t>(static_cast<int64_t>(bt_width) * block_size, INT32_MAX));
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(max_len) + kReadTok - 1) / kReadTok),
                  static_cast<unsigned>(batch), 2);
  return cache_dtype == VJ_CACHE_INT8
             ? launch_dependent(what, kv_read_quantized_kernel<true>, grid, kReadThreads, 0, stream, a)
             : launch_dependent(what, kv_read_quantized_kernel<false>, grid, kReadThreads, 0, stream,
                                a);
}
