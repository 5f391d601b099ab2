// The quantised KV cache's number formats, shared by the kernels that write
// it (quant_cache.cu) and the ones that read it (quant_cache.cu,
// quant_decode.cu).
//
// A cached row (token, KV head, K or V) is 128 8-bit elements and one E8M0
// scale byte b; it stands for element * 2^(b - 127). Scales are powers of two
// because then (1) element * scale is a bf16 number for both element types
// (e4m3 has 4 significant bits, int8 has 8), so reading back rounds nothing,
// (2) multiplying by a scale is exact wherever a kernel does it, and (3) e4m3
// loses nothing: its relative precision does not depend on where in its range
// a row lies.
#pragma once

#include "../../include/vjattn.h"
#include "vj_common.cuh"

#include <string>

namespace vj {
namespace {
namespace qn {

constexpr int kD = 128;

// Pages of a quantised pool, as the C entries get them.
struct Pool {
  uint8_t *k, *v;                // elements
  uint8_t *ks, *vs;              // scale bytes
  int64_t sb, st, sh;            // element strides: block, token, head
  int64_t ssb, ssh;              // scale strides: block, head (token stride 1)
  int64_t num_blocks;
  int block_size;
};

// 2^(b - 127); byte 0 is 2^-127 (a subnormal), byte 255 NaN.
VJ_DEV float scale_of(uint32_t b) {
  return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7fffffffu : b << 23);
}

// Scale exponent of a row from the bit pattern of its largest magnitude: the
// smallest e with amax <= 448 * 2^e (448 = 1.75 * 2^8) or 127 * 2^e
// (127 = 1.984375 * 2^6), at least -126 (and so for a row of zeros, whose
// scale must not tower over its neighbours': the decode kernel weighs rows by
// their scales). amax is finite.
template <bool kInt8>
VJ_DEV int scale_exponent(uint32_t amax_bits) {
  const int x = static_cast<int>(amax_bits >> 23) - 127;   // subnormals: far below the clamp
  const uint32_t frac = amax_bits & 0x7fffffu;
  const int e = kInt8 ? x - 6 + (frac > 0x7e0000u ? 1 : 0) : x - 8 + (frac > 0x600000u ? 1 : 0);
  return e < -126 ? -126 : e;
}

// Two floats to two elements (low byte first), round to nearest even.
template <bool kInt8>
VJ_DEV uint32_t quantise2(float lo, float hi) {
  if constexpr (kInt8) {
    // |v| <= 127: adding 1.5 * 2^23 rounds to an integer, whose low byte is
    // the low byte of the sum's bits
    const uint32_t a = __float_as_uint(__fadd_rn(lo, 12582912.0f));
    const uint32_t b = __float_as_uint(__fadd_rn(hi, 12582912.0f));
    return (a & 0xffu) | ((b & 0xffu) << 8);
  } else {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
  }
}

// The two elements in the low (kHi = false) or high half of a word as f16x2.
// Both element types are exact in f16.
template <bool kInt8, bool kHi>
VJ_DEV uint32_t dequant_f16x2(uint32_t w) {
  uint32_t d;
  if constexpr (kInt8) {
    // b + 128 below 0x64 is the f16 number 1024 + (b + 128)
    asm("prmt.b32 %0, %1, %2, %3;"
        : "=r"(d)
        : "r"(w ^ 0x80808080u), "r"(0x64646464u), "r"(kHi ? 0x4342u : 0x4140u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(d), "r"(0x64806480u));   // - 1152
  } else if constexpr (kHi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
        : "=r"(d)
        : "r"(w));
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}"
        : "=r"(d)
        : "r"(w));
  }
  return d;
}
VJ_DEV float2 f16x2_to_f32(uint32_t w) {
  float2 r;
  asm("{\n\t.reg .f16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(w));
  return r;
}

// Checks shared by every entry point of the quantised cache; `what` names it.
inline int check_pool(const std::string &what, const Pool &p, int cache_dtype, int num_kv_heads,
                      int head_dim) {
  if (num_kv_heads <= 0 || p.num_blocks <= 0 || p.block_size <= 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": negative or zero size");
  }
  if (head_dim != kD) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": head_dim must be 128, got " +
                                             std::to_string(head_dim));
  }
  if (cache_dtype != VJ_CACHE_E4M3 && cache_dtype != VJ_CACHE_INT8) {
    return set_error(VJ_ERR_INVALID_ARGUMENT,
                     what + ": cache_dtype must be VJ_CACHE_E4M3 or VJ_CACHE_INT8");
  }
  if (p.block_size % 16 != 0) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": block_size must be a multiple of 16");
  }
  if (p.num_blocks > INT32_MAX / p.block_size) {
    return set_error(VJ_ERR_UNSUPPORTED, what + ": pool larger than 2^31 slots");
  }
  return VJ_OK;
}
// The part of the checks that needs pointers (skipped for empty calls).
inline int check_pool_memory(const std::string &what, const Pool &p) {
  if (!p.k || !p.v || !p.ks || !p.vs) {
    return set_error(VJ_ERR_INVALID_ARGUMENT, what + ": null cache pointer");
  }
  if ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
       reinterpret_cast<uintptr_t>(p.ks) | reinterpret_cast<uintptr_t>(p.vs)) % 16 != 0 ||
      (p.sb | p.st | p.sh | p.ssb | p.ssh) % 16 != 0) {
    return set_error(VJ_ERR_INVALID_ARGUMENT,
                     what + ": cache and scale bases and strides must be multiples of 16 bytes");
  }
  return VJ_OK;
}

}  // namespace qn
}  // namespace
}  // namespace vj
