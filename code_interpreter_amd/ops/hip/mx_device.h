// Device code that the microscaled 4-bit kernels share: the format is
// described in mxfp4_quant.hip.
#pragma once

#include "lm.h"

namespace {

constexpr int kPer = 8;  // elements of a lane

using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
using raw16 = uint32_t __attribute__((ext_vector_type(4), aligned(2)));
using b16x2 = __bf16 __attribute__((ext_vector_type(2)));
using h16x2 = _Float16 __attribute__((ext_vector_type(2)));
using f32x2 = float __attribute__((ext_vector_type(2)));
using u16x2 = uint16_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t lane_max(uint32_t a, uint32_t b) {
  return a > b ? a : b;
}

// the scale byte of a block, from the bits in f32 of its largest magnitude
__device__ __forceinline__ uint32_t scale_of(uint32_t bits) {
  int e = (int)(bits >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}
// the scale that a byte stands for
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// 8 elements in w (f32: w and w2), in f32 bits the largest magnitude
template <LmType T>
__device__ __forceinline__ uint32_t largest(const u32x4& w, const u32x4& w2) {
  if constexpr (T == LmType::F32) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
      m = lane_max(m, lane_max(w[i] & 0x7FFFFFFFu, w2[i] & 0x7FFFFFFFu));
    return m;
  } else {
    // magnitudes order as their bits
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t b = w[i] & 0x7FFF7FFFu;
      u16x2 p;
      __builtin_memcpy(&p, &b, 4);
      m = __builtin_elementwise_max(m, p);
    }
    uint16_t top = m[0] > m[1] ? m[0] : m[1];
    if constexpr (T == LmType::BF16) return (uint32_t)top << 16;
    _Float16 h;
    __builtin_memcpy(&h, &top, 2);
    return __float_as_uint((float)h);
  }
}

// the scale byte of the block whose 32 elements four neighbouring lanes hold
template <LmType T>
__device__ __forceinline__ uint32_t block_scale(const u32x4& w,
                                                const u32x4& w2) {
  uint32_t a = largest<T>(w, w2);
  a = lane_max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0xB1, 15, 15,
                                                     false));  // lane ^ 1
  a = lane_max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x4E, 15, 15,
                                                     false));  // lane ^ 2
  return scale_of(a);
}

template <LmType T>
__device__ __forceinline__ uint32_t encode(const u32x4& w, const u32x4& w2,
                                           float s) {
  uint32_t c = 0;
  if constexpr (T == LmType::F32) {
    auto f = [&](int i) { return __uint_as_float(i < 4 ? w[i] : w2[i - 4]); };
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(0), f(1), s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(2), f(3), s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(4), f(5), s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f(6), f(7), s, 3);
  } else if constexpr (T == LmType::BF16) {
    b16x2 p[4];
    __builtin_memcpy(p, &w, 16);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[0], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[1], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[2], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, p[3], s, 3);
  } else {
    h16x2 p[4];
    __builtin_memcpy(p, &w, 16);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, p[0], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, p[1], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, p[2], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, p[3], s, 3);
  }
  return c;
}

template <LmType T>
struct Size {
  static constexpr int value = T == LmType::F32 ? 4 : 2;
};

// elements [at, at + 8) of a row of k elements, zeros behind its end
template <LmType T>
__device__ __forceinline__ void load8(const char* row, int64_t at, int64_t k,
                                      u32x4& w, u32x4& w2) {
  const char* p = row + at * Size<T>::value;
  if (at + kPer <= k) {
    w = *(const raw16*)p;
    if constexpr (T == LmType::F32) w2 = *(const raw16*)(p + 16);
    return;
  }
  w = w2 = u32x4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    if (at + i >= k) continue;
    if constexpr (T == LmType::F32) {
      uint32_t b = ((const uint32_t*)p)[i];
      if (i < 4)
        w[i] = b;
      else
        w2[i - 4] = b;
    } else {
      w[i >> 1] |= (uint32_t)((const uint16_t*)p)[i] << (16 * (i & 1));
    }
  }
}

}  // namespace
