// The 4-bit key / value cache: 32 consecutive elements of a head share a power of two, and each is that times an e2m1 number
// (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives).  All of them are bf16 or f16 numbers, so that widening is exact and
// one instruction for two elements.
//
// A page of one kv head: bs token rows of d / 2 bytes (even element in the low half), then their bs * d / 32 scales, each
// the exponent + 127.  Rows and not, as in the wider caches, 8-key groups of V^T: a token's write is then whole bytes, and its V
// has scales of its own.
#pragma once
#include "common.h"

namespace kgc {

__host__ __device__ __forceinline__ int64_t kv4_page_bytes(int bs, int d) { return (int64_t)bs * (d / 2 + d / 32); }

// page of a block table's entry: one that is no page of the pool gives wrong results, never a fault
__device__ __forceinline__ int kv4_page(const int* bt, int i, int bt_stride, int num_blocks) {
  return min(max(kgc_bt(bt, i, bt_stride, num_blocks), 0), num_blocks - 1);
}

// elements 2 * SEL, 2 * SEL + 1 of the 8 in w, times the scale
template <typename T, int SEL> __device__ __forceinline__ uint32_t fp4x2_widen(uint32_t w, float scale) {
  if constexpr (std::is_same_v<T, bf16>)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
}
template <typename T> __device__ __forceinline__ u32x4 fp4x8_widen(uint32_t w, float scale) {
  return u32x4{fp4x2_widen<T, 0>(w, scale), fp4x2_widen<T, 1>(w, scale), fp4x2_widen<T, 2>(w, scale),
               fp4x2_widen<T, 3>(w, scale)};
}
__device__ __forceinline__ float kv4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The scale byte of a block whose largest magnitude is `most`: the power of two under which that is at most 7, since what
// lies between 6 and 7 is as near to 6 as the step there allows.  The ends keep 6 times the scale below the largest number of T, and
// half of it a number of T.
template <typename T> __device__ __forceinline__ uint32_t kv4_scale_byte(float most) {
  constexpr int lo = std::is_same_v<T, bf16> ? -120 : -22, hi = std::is_same_v<T, bf16> ? 125 : 13;
  const uint32_t u = __float_as_uint(most);
  const int e = (int)(u >> 23) - 129 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(min(max(e, lo), hi) + 127);
}

// 8 elements as e2m1 over a scale, ties to the even code; what is over 6 scales is 6
__device__ __forceinline__ uint32_t fp4x8(const float (&x)[8], float scale) {
  const float top = 6.f * scale;
  float c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = fminf(fmaxf(x[j], -top), top);
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, c[0], c[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c[2], c[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c[4], c[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c[6], c[7], scale, 3);
}

// a + b in 24 bits, the last of them set where the others are not all of it: it is above, below or on every number of
// fewer bits that the sum is above, below or on, so that rounding it on is rounding once.
__device__ __forceinline__ float sum_to_odd(double a, double b) {
  const double s = a + b;
  const uint32_t u = __float_as_uint((float)s);
  double off = s - (double)__uint_as_float(u);
  if (off == 0) {                                      // few: what of s is not in 24 bits is more than what of a + b is not in s
    const double t = s - a;
    off = (a - (s - t)) + (b - t);                     // a + b = s + off (Knuth's two-sum)
  }
  // where off's sign is not the sum's, the 24 bits are further from zero than the sum (infinities and NaN: as they are)
  const uint32_t away = ((uint32_t)(__builtin_bit_cast(uint64_t, off) >> 32) ^ u) >> 31;
  return __uint_as_float(__builtin_islessgreater(off, 0.0) ? (u - away) | 1u : u);
}

// l + the two numbers of T in w
template <typename T> __device__ __forceinline__ float kv4_add_pair(uint32_t w, float l) {
  if constexpr (std::is_same_v<T, bf16>)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), bf16x2_t{(bf16)1.f, (bf16)1.f}, l, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, w), f16x2_t{(f16)1.f, (f16)1.f}, l, false);
}

}  // namespace kgc
