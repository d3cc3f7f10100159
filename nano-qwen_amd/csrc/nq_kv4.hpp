// The 4-bit page format: rows in blocks of 32 elements, each block E2M1 codes
// ({0, 1/2, 1, 3/2, 2, 3, 4, 6} and a sign) and one scale byte, a power of two with
// bias 127 (E8M0; 255 makes the block NaN).  Two codes a byte, the even element low.
// A page and kv head hold, for P rows of D elements,
//   K codes (P, D/2) | V codes (P, D/2) | K scales (P, D/32) | V scales (P, D/32)
// 17 D / 16 bytes a row: the codes of consecutive rows are adjacent, so a wave's loads
// are whole kilobytes, and every part starts 16-byte aligned (P a multiple of 32).
#pragma once

#include "nq_common.hpp"

namespace nq {

template <int D> struct Kv4 {
  static constexpr int CB = D / 2;        // code bytes of a row
  static constexpr int SB = D / 32;       // scale bytes of a row
  static constexpr int RB = 2 * (CB + SB);  // bytes of a row, K and V
  __device__ static int v_codes(int page) { return page * CB; }
  __device__ static int k_scales(int page) { return page * 2 * CB; }
  __device__ static int v_scales(int page) { return page * (2 * CB + SB); }
};

// The scale of a byte as the conversions take it: a float of that exponent.
__device__ __forceinline__ float kv4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight codes as bf16: exact, a code times a power of two has two significant bits.
__device__ __forceinline__ bf16x8 kv4_bf16x8(uint32_t codes, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The scale byte of a block whose largest magnitude has these bits: the smallest power
// of two of which it is at most 7 times, so that no element is off by more than half of
// the type's widest step (7 rounds to 6).  NaN and infinity order above every number.
__device__ __forceinline__ uint32_t kv4_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const int e = (int)(amax_bits >> 23) - 2 + ((amax_bits & 0x7fffffu) > 0x600000u);
  return (uint32_t)(e < 1 ? 1 : (e > 252 ? 252 : e));  // from 2^-126; 6 * 2^125 is the largest that fp32 holds
}

}  // namespace nq
