// Microscaled 4-bit floating point: quantisation and read-back.
//
// 32 elements along the last axis share a scale, a power of two held as its
// exponent + 127 in a byte. An element is e2m1: sign, and one of 0, 0.5, 1,
// 1.5, 2, 3, 4, 6. Two share a byte, the earlier in the low half. With a the
// block's largest magnitude the scale is 2^(floor(log2 a) - 2), so that a
// falls in [4, 8); elements are rounded to the nearest, ties to the even
// code, and what lies above 6 becomes 6. That saturation and the rounding
// are the format's own choices. The exponent stops at -127: smaller blocks
// keep that scale. A block with a NaN or an infinity has scale byte 255,
// which stands for NaN in all of its elements, and codes of 0.
//
// Both directions move bytes and little else: 2 + 17/32 bytes an element of
// a 16-bit tensor. A lane takes 8 elements, 4 neighbouring lanes a block,
// so that loads are 16 bytes a lane in order and the block's largest
// magnitude takes two lane exchanges. The hardware's conversion divides by
// the scale and rounds as above, for every scale from 2^-127 on and for
// subnormal elements too. 8192 x 8192 bf16: 34.8 us, 4.9 TB/s (a large copy:
// 4.8); back 25.8 us, 6.6 TB/s, part of it from the chip's cache.

#include "mx_device.h"

namespace {

constexpr int kThreads = 256;
// A thread takes groups of 8 elements, `kUnroll` of them a block apart.
// groups = rows * per_row, per_row = 4 * blocks of a row.
template <LmType T, int kUnroll>
__global__ __launch_bounds__(kThreads) void quantize_kernel(
    const char* __restrict__ x, int64_t stride, int64_t k, int64_t per_row,
    int64_t groups, bool flat, uint32_t* __restrict__ codes,
    uint8_t* __restrict__ scales) {
  const int64_t first =
      (int64_t)blockIdx.x * (kThreads * kUnroll) + threadIdx.x;
  u32x4 w[kUnroll], w2[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; i++) {
    int64_t g = first + i * kThreads;
    if (g >= groups) break;
    if (flat) {  // rows of whole blocks, one behind the other
      load8<T>(x, g * kPer, g * kPer + kPer, w[i], w2[i]);
    } else {
      int64_t row = g / per_row;
      load8<T>(x + row * stride * Size<T>::value, (g - row * per_row) * kPer,
               k, w[i], w2[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kUnroll; i++) {
    int64_t g = first + i * kThreads;
    if (g >= groups) break;  // groups is a multiple of 4: whole blocks
    uint32_t byte = block_scale<T>(w[i], w2[i]);
    codes[g] = byte == 255 ? 0u : encode<T>(w[i], w2[i], scale_value(byte));
    if ((g & 3) == 0) scales[g >> 2] = (uint8_t)byte;
  }
}

template <LmType T>
__device__ __forceinline__ void decode8(uint32_t c, float s, u32x4& w,
                                        u32x4& w2) {
  if constexpr (T == LmType::F32) {
    f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0),
                  __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1),
                  __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2),
                  __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3)};
    __builtin_memcpy(&w, p, 16);
    __builtin_memcpy(&w2, p + 2, 16);
  } else if constexpr (T == LmType::BF16) {
    b16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0),
                  __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1),
                  __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2),
                  __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3)};
    __builtin_memcpy(&w, p, 16);
  } else {
    h16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 0),
                  __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 1),
                  __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 2),
                  __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 3)};
    __builtin_memcpy(&w, p, 16);
  }
}

template <LmType T, int kUnroll>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(
    const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
    int64_t k, int64_t per_row, int64_t groups, bool flat,
    char* __restrict__ out) {
  constexpr uint32_t kNan = T == LmType::F32    ? 0x7FC00000u
                            : T == LmType::BF16 ? 0x7FC07FC0u
                                                : 0x7E007E00u;
  const int64_t first =
      (int64_t)blockIdx.x * (kThreads * kUnroll) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kUnroll; i++) {
    int64_t g = first + i * kThreads;
    if (g >= groups) break;
    uint32_t byte = scales[g >> 2];
    u32x4 w, w2;
    decode8<T>(codes[g], scale_value(byte), w, w2);
    if (byte == 255) w = w2 = u32x4{kNan, kNan, kNan, kNan};
    int64_t at = g * kPer, left = kPer;
    if (!flat) {
      int64_t row = g / per_row, col = (g - row * per_row) * kPer;
      at = row * k + col;
      left = k - col;
    }
    char* p = out + at * Size<T>::value;
    if (left >= kPer) {
      *(raw16*)p = w;
      if constexpr (T == LmType::F32) *(raw16*)(p + 16) = w2;
    } else {
#pragma unroll
      for (int j = 0; j < kPer; j++) {
        if (j >= left) continue;
        if constexpr (T == LmType::F32)
          ((uint32_t*)p)[j] = j < 4 ? w[j] : w2[j - 4];
        else
          ((uint16_t*)p)[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
      }
    }
  }
}

constexpr int kUnroll = 4;

dim3 grid_of(int64_t groups) {
  int64_t per = (int64_t)kThreads * kUnroll;
  return lm_grid((groups + per - 1) / per, kThreads);
}

}  // namespace

void launch_mx_quantize(LmType t, const void* x, int64_t stride,
                        uint8_t* codes, uint8_t* scales, int64_t rows,
                        int64_t k, hipStream_t stream) {
  const int64_t per_row = mx_blocks(k) * 4, groups = rows * per_row;
  const bool flat = k % kMxBlock == 0 && (stride == k || rows == 1);
  const dim3 grid = grid_of(groups);
  auto* x8 = (const char*)x;
  auto* c32 = (uint32_t*)codes;
  switch (t) {
    case LmType::F32:
      quantize_kernel<LmType::F32, kUnroll><<<grid, kThreads, 0, stream>>>(
          x8, stride, k, per_row, groups, flat, c32, scales);
      break;
    case LmType::BF16:
      quantize_kernel<LmType::BF16, kUnroll><<<grid, kThreads, 0, stream>>>(
          x8, stride, k, per_row, groups, flat, c32, scales);
      break;
    case LmType::F16:
      quantize_kernel<LmType::F16, kUnroll><<<grid, kThreads, 0, stream>>>(
          x8, stride, k, per_row, groups, flat, c32, scales);
      break;
  }
  HIP_CHECK(hipGetLastError());
}

void launch_mx_dequantize(LmType t, const uint8_t* codes,
                          const uint8_t* scales, void* out, int64_t rows,
                          int64_t k, hipStream_t stream) {
  const int64_t per_row = mx_blocks(k) * 4, groups = rows * per_row;
  const bool flat = k % kMxBlock == 0;
  const dim3 grid = grid_of(groups);
  auto* c32 = (const uint32_t*)codes;
  switch (t) {
    case LmType::F32:
      dequantize_kernel<LmType::F32, kUnroll><<<grid, kThreads, 0, stream>>>(
          c32, scales, k, per_row, groups, flat, (char*)out);
      break;
    case LmType::BF16:
      dequantize_kernel<LmType::BF16, kUnroll><<<grid, kThreads, 0, stream>>>(
          c32, scales, k, per_row, groups, flat, (char*)out);
      break;
    case LmType::F16:
      dequantize_kernel<LmType::F16, kUnroll><<<grid, kThreads, 0, stream>>>(
          c32, scales, k, per_row, groups, flat, (char*)out);
      break;
  }
  HIP_CHECK(hipGetLastError());
}
