// mx4.hpp -- the microscaled 4-bit format on the device: 32 consecutive values
// share a scale 2^e (a byte, e + 127; 255 is no number), each is a code of 4 bits,
// sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, two to a byte, the first in the low
// half.  The conversions are gfx950's: they take the scale as a float, of which
// they read the exponent (255: every value NaN, also that of code 0), round to
// nearest even and cut at 6; measured exact for every scale and code.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace spk_mx4 {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));

constexpr uint32_t kNone = 255;  // scale byte of a block that holds an infinity or NaN

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// The 8 codes of a dword as 16-bit values, in order.
template <bool BF>
__device__ __forceinline__ uint4 expand(uint32_t u, float scale) {
  uint4 r;
  if constexpr (BF) {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 0));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 1));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 2));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 3));
  } else {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(u, scale, 0));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(u, scale, 1));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(u, scale, 2));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(u, scale, 3));
  }
  return r;
}

// 8 values of 16 bits as codes.
template <bool BF>
__device__ __forceinline__ uint32_t codes_of(uint4 v, float scale) {
  uint32_t r = 0;
  if constexpr (BF) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf2_t, v.x), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf2_t, v.y), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf2_t, v.z), scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf2_t, v.w), scale, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(half2_t, v.x), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(half2_t, v.y), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(half2_t, v.z), scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(half2_t, v.w), scale, 3);
  }
  return r;
}

__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float scale) {
  uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], scale, 3);
}

// Of 8 values of 16 bits the largest magnitude's bits; an infinity's or a NaN's are
// larger than any number's.
__device__ __forceinline__ uint32_t most_of(uint4 v) {
  typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
  auto mag = [](uint32_t u) { return __builtin_bit_cast(ushort2_t, u & 0x7fff7fffu); };
  const ushort2_t m = __builtin_elementwise_max(__builtin_elementwise_max(mag(v.x), mag(v.y)),
                                                __builtin_elementwise_max(mag(v.z), mag(v.w)));
  return max((uint32_t)m.x, (uint32_t)m.y);
}

// The scale byte of a block from its largest magnitude's float bits: two binades
// below it, 2^-127 at least.
__device__ __forceinline__ uint32_t scale_byte(uint32_t most) {
  const uint32_t e = most >> 23;
  return e == 255 ? kNone : e > 2 ? e - 2 : 0;
}

// As scale_byte, from the bits of a 16-bit magnitude.
template <bool BF>
__device__ __forceinline__ uint32_t scale_byte16(uint32_t most) {
  if constexpr (BF) return scale_byte(most << 16);
  return most >= 0x7c00u ? kNone : scale_byte(__float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)most)));
}

// A wave's load straight into LDS, side by side at `to`: B bytes of a lane (of one byte
// a dword is written).
template <int B, typename T>
__device__ __forceinline__ void load_lds(const void* from, T* to) {
  const auto g = (const __attribute__((address_space(1))) void*)from;
  const auto l = (__attribute__((address_space(3))) void*)to;
  if constexpr (B == 16)
    __builtin_amdgcn_global_load_lds(g, l, 16, 0, 0);
  else if constexpr (B == 4)
    __builtin_amdgcn_global_load_lds(g, l, 4, 0, 0);
  else
    __builtin_amdgcn_global_load_lds(g, l, 1, 0, 0);
}

// All loads of this wave but the newest N have arrived.  (As a builtin, which the compiler
// takes into account: told in assembly it waits for all of them before it reads what they wrote.)
template <int N>
__device__ __forceinline__ void arrived() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4 | 15 << 8);
  asm volatile("" ::: "memory");
}

}  // namespace spk_mx4
