// The product of microscaled 4-bit operands: y[m][n] = sum_k x[m][k] w[n][k]
// + bias[n], on gfx950's scaled matrix instructions, which take the 4-bit
// codes and the block scales as they are stored and add in f32. y is rounded
// once, in the epilogue.
//
// The order of blocks of 32 along k does not matter as long as both operands
// keep the same one. So a lane takes *neighbouring* blocks from a row where
// an instruction's lanes would in memory order be given every second or
// fourth one: a lane then loads its scales as one 4-byte word and picks a
// byte of it by the instruction's selector.
//
// The weights are the instruction's first operand: a lane's accumulators are
// then 4 neighbouring outputs of one token, stored at once.

#include <algorithm>
#include <type_traits>

#include "mx_device.h"

namespace {

using v8i = int __attribute__((ext_vector_type(8)));
using v4f = float __attribute__((ext_vector_type(4)));
using v16f = float __attribute__((ext_vector_type(16)));
using raw4 = uint32_t __attribute__((aligned(1)));
using lds_void = __attribute__((address_space(3))) void;
using global_void = const __attribute__((address_space(1))) void;

constexpr uint32_t kUnit = 0x7F7F7F7Fu;  // four scales of 1

__device__ __forceinline__ v8i operand(const u32x4& w) {
  return v8i{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
}

// scales [at, at + 4) of a row, 1 in the place of those behind its end
__device__ __forceinline__ uint32_t load_scales(const uint8_t* row, int at,
                                                int nb) {
  if (at + 4 <= nb) return *(const raw4*)(row + at);
  uint32_t s = kUnit;
  for (int i = 0; i < 4; i++)
    if (at + i < nb)
      s = (s & ~(0xFFu << (8 * i))) | (uint32_t)row[at + i] << (8 * i);
  return s;
}

// outputs n .. n + 3 of a row
template <LmType T>
__device__ __forceinline__ void store4(void* y, int64_t at, const float* f,
                                       int valid) {
  using E = typename std::conditional<
      T == LmType::F32, float,
      typename std::conditional<T == LmType::BF16, __bf16, _Float16>::type>::
      type;
  using E4 = E __attribute__((ext_vector_type(4)));
  E* p = (E*)y + at;
  if (valid >= 4) {
    struct __attribute__((packed, aligned(2))) Loose {
      E4 v;
    };
    ((Loose*)p)->v = E4{(E)f[0], (E)f[1], (E)f[2], (E)f[3]};
  } else {
    for (int i = 0; i < valid; i++) p[i] = (E)f[i];
  }
}

template <LmType T>
__device__ __forceinline__ float bias_at(const void* bias, int64_t i) {
  if constexpr (T == LmType::F32) return ((const float*)bias)[i];
  if constexpr (T == LmType::BF16) return (float)((const __bf16*)bias)[i];
  return (float)((const _Float16*)bias)[i];
}

// ---------------------------------------------------------------------------
// tiles: many tokens
// ---------------------------------------------------------------------------
// A block of WM x WN waves makes BM tokens x BN outputs; a wave FM x FN
// tiles of 32 x 32. A step takes 256 elements of k, 128 bytes of a row, into
// one of two buffers of shared memory by asynchronous loads of 16 bytes a
// lane, while the other one is read. In shared memory the 8 units of 16
// bytes of row r stand at their index ^ (r & 7), so that 8 lanes that read
// the same unit of 8 rows touch all of the banks once.
template <LmType T, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM* WN * 64) void tile_kernel(
    const uint8_t* __restrict__ xc, const uint8_t* __restrict__ xs,
    const uint8_t* __restrict__ wc, const uint8_t* __restrict__ ws,
    const void* __restrict__ bias, void* __restrict__ y, int64_t m, int64_t n,
    int nb, int tiles_m, int tiles_n) {
  constexpr int kWaves = WM * WN;
  constexpr int BM = WM * FM * 32, BN = WN * FN * 32;
  constexpr int kRow = 128;
  constexpr int kBuf = (BM + BN) * kRow;
  constexpr int kLoadsX = BM / 8 / kWaves, kLoadsW = BN / 8 / kWaves;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0, "");
  extern __shared__ __attribute__((aligned(16))) char smem[];

  // A chiplet gets every eighth block; it is given neighbouring tiles, in
  // columns of 8 tiles of tokens, so that its cache holds what they share.
  int id = blockIdx.x;
  {
    const int all = tiles_m * tiles_n, q = all / 8, r = all % 8;
    const int xcd = id % 8, idx = id / 8;
    id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  }
  const int per = 8 * tiles_n, group = id / per;
  const int high = min(8, tiles_m - group * 8);
  const int64_t m0 = (int64_t)(group * 8 + (id % per) % high) * BM;
  const int64_t n0 = (int64_t)((id % per) / high) * BN;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const int l31 = lane & 31, h = lane >> 5;
  const int64_t row_bytes = (int64_t)nb * kMxBytes;

  // this lane's rows of each load, clamped to the last one: what is made of
  // a row behind it is not stored
  const uint8_t* xb = xc + m0 * row_bytes;
  const uint8_t* wb = wc + n0 * row_bytes;
  uint32_t xo[kLoadsX], wo[kLoadsW];
#pragma unroll
  for (int i = 0; i < kLoadsX; i++) {
    int64_t r = (i * kWaves + wave) * 8 + (lane >> 3);
    xo[i] = (uint32_t)(min(r, m - 1 - m0) * row_bytes);
  }
#pragma unroll
  for (int i = 0; i < kLoadsW; i++) {
    int64_t r = (i * kWaves + wave) * 8 + (lane >> 3);
    wo[i] = (uint32_t)(min(r, n - 1 - n0) * row_bytes);
  }
  const int unit = (lane & 7) ^ (lane >> 3);
  const int steps = (nb + 7) / 8;
  const int rest = nb - (steps - 1) * 8;  // blocks of the last step, 1 to 8

  auto stage = [&](int t) {
    char* to = smem + (t & 1) * kBuf + wave * 1024;
    const uint32_t u =
        (uint32_t)(t == steps - 1 ? min(unit, rest - 1) : unit) * 16;
    const uint8_t* xt = xb + (int64_t)t * kRow;
    const uint8_t* wt = wb + (int64_t)t * kRow;
#pragma unroll
    for (int i = 0; i < kLoadsW; i++)
      __builtin_amdgcn_global_load_lds((global_void*)(wt + wo[i] + u),
                                       (lds_void*)(to + i * kWaves * 1024),
                                       16, 0, 0);
#pragma unroll
    for (int i = 0; i < kLoadsX; i++)
      __builtin_amdgcn_global_load_lds(
          (global_void*)(xt + xo[i] + u),
          (lds_void*)(to + BN * kRow + i * kWaves * 1024), 16, 0, 0);
  };

  const uint8_t* xsr[FM];
  const uint8_t* wsr[FN];
#pragma unroll
  for (int i = 0; i < FM; i++)
    xsr[i] = xs + min(m0 + (wm * FM + i) * 32 + l31, m - 1) * nb;
#pragma unroll
  for (int i = 0; i < FN; i++)
    wsr[i] = ws + min(n0 + (wn * FN + i) * 32 + l31, n - 1) * nb;

  v16f acc[FN][FM] = {};
  uint32_t sx[FM], sw[FN];
  auto scales = [&](int t, uint32_t* dx, uint32_t* dw) {
#pragma unroll
    for (int i = 0; i < FM; i++) dx[i] = load_scales(xsr[i], t * 8 + 4 * h, nb);
#pragma unroll
    for (int i = 0; i < FN; i++) dw[i] = load_scales(wsr[i], t * 8 + 4 * h, nb);
  };

  // Instruction s multiplies blocks s (lower lanes) and 4 + s (upper ones)
  // of the step. Behind the row's end codes and scales are made 0 and 1.
  auto multiply = [&](int t, auto last) {
    const char* from = smem + (t & 1) * kBuf;
    auto one = [&](auto step) {
      constexpr int s = decltype(step)::value;
      if (decltype(last)::value && s >= rest) return;
      const int at = ((s + 4 * h) ^ (lane & 7)) * 16 + l31 * kRow;
      const bool in = !decltype(last)::value || s + 4 * h < rest;
      v8i a[FN], b[FM];
#pragma unroll
      for (int i = 0; i < FN; i++) {
        u32x4 w = *(const u32x4*)(from + (wn * FN + i) * 32 * kRow + at);
        a[i] = operand(in ? w : u32x4{0, 0, 0, 0});
      }
#pragma unroll
      for (int i = 0; i < FM; i++) {
        u32x4 w =
            *(const u32x4*)(from + (BN + (wm * FM + i) * 32) * kRow + at);
        b[i] = operand(in ? w : u32x4{0, 0, 0, 0});
      }
#pragma unroll
      for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
              a[i], b[j], acc[i][j], 4, 4, s, (int)sw[i], s, (int)sx[j]);
    };
    one(std::integral_constant<int, 0>{});
    one(std::integral_constant<int, 1>{});
    one(std::integral_constant<int, 2>{});
    one(std::integral_constant<int, 3>{});
  };

  stage(0);
  scales(0, sx, sw);
  for (int t = 0; t < steps; t++) {
    // this wave's loads of step t have landed; then every wave's have, and
    // every wave is through with step t - 1, whose buffer is filled next
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    uint32_t nx[FM], nw[FN];
    if (t + 1 < steps) {
      stage(t + 1);
      scales(t + 1, nx, nw);
      multiply(t, std::false_type{});
#pragma unroll
      for (int i = 0; i < FM; i++) sx[i] = nx[i];
#pragma unroll
      for (int i = 0; i < FN; i++) sw[i] = nw[i];
    } else if (rest == 8) {
      multiply(t, std::false_type{});
    } else {
      multiply(t, std::true_type{});
    }
  }

#pragma unroll
  for (int i = 0; i < FN; i++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int64_t col = n0 + (wn * FN + i) * 32 + 8 * g + 4 * h;
      const int valid = (int)min((int64_t)4, n - col);
      if (valid <= 0) continue;
      float add[4] = {};
      if (bias)
        for (int r = 0; r < 4; r++)
          if (r < valid) add[r] = bias_at<T>(bias, col + r);
#pragma unroll
      for (int j = 0; j < FM; j++) {
        const int64_t row = m0 + (wm * FM + j) * 32 + l31;
        if (row >= m) continue;
        float f[4];
#pragma unroll
        for (int r = 0; r < 4; r++) f[r] = acc[i][j][4 * g + r] + add[r];
        store4<T>(y, row * n + col, f, valid);
      }
    }
}

// ---------------------------------------------------------------------------
// few tokens
// ---------------------------------------------------------------------------
// The weights are read once, from memory into registers, and bound the time;
// 16 * MT tokens are held against them. A block makes 16 * NT outputs of all
// tokens: its 8 waves take turns along k, 512 elements a turn, a lane 4
// neighbouring blocks (64 bytes) of one row, and add up through shared
// memory at the end, in a fixed order. The tokens come from memory as codes
// (packed), or are quantised by each block into its shared memory, which
// saves a launch and costs the more the more tokens there are.
template <LmType T, int MT, int NT, bool kPacked>
__global__ __launch_bounds__(512) void few_kernel(
    const void* __restrict__ x, int64_t stride,
    const uint8_t* __restrict__ xc, const uint8_t* __restrict__ xs,
    const uint8_t* __restrict__ wc, const uint8_t* __restrict__ ws,
    const void* __restrict__ bias, void* __restrict__ y, int m, int64_t n,
    int64_t k, int nb) {
  constexpr int kWaves = 8;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l15 = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);
  const int turns = (nb + 15) / 16;

  const uint8_t* wrow[NT];
  const uint8_t* srow[NT];
#pragma unroll
  for (int i = 0; i < NT; i++) {
    int64_t r = min(n0 + i * 16 + l15, n - 1);
    wrow[i] = wc + r * nb * kMxBytes;
    srow[i] = ws + r * nb;
  }
  struct Turn {
    u32x4 c[NT][4];
    uint32_t s[NT];
  };
  auto load = [&](int turn, Turn& to) {
    const int at = turn * 16 + 4 * q;
#pragma unroll
    for (int i = 0; i < NT; i++) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        to.c[i][j] = at + j < nb
                         ? *(const u32x4*)(wrow[i] + (int64_t)(at + j) * 16)
                         : u32x4{0, 0, 0, 0};
      to.s[i] = load_scales(srow[i], at, nb);
    }
  };
  Turn next;
  if (wave < turns) load(wave, next);

  // codes of a token stand (nb + 1) * 16 bytes apart: 8 lanes that read the
  // same unit of 8 tokens touch all banks once
  const int crow = (nb + 1) * 16, sstride = ((nb + 3) & ~3) + 4;
  uint8_t* lds_s = (uint8_t*)smem + m * crow;
  if constexpr (!kPacked) {
    const uint32_t per_row = (uint32_t)nb * 4, groups = per_row * m;
    for (uint32_t g = threadIdx.x; g < groups; g += 512) {
      const uint32_t row = g / per_row, col = g - row * per_row;
      u32x4 w, w2;
      load8<T>((const char*)x + row * stride * Size<T>::value,
               (int64_t)col * kPer, k, w, w2);
      uint32_t byte = block_scale<T>(w, w2);
      *(uint32_t*)(smem + row * crow + col * 4) =
          byte == 255 ? 0u : encode<T>(w, w2, scale_value(byte));
      if ((g & 3) == 0) lds_s[row * sstride + (col >> 2)] = (uint8_t)byte;
    }
    // scales of 1 up to the end of a row's last whole word
    for (uint32_t g = threadIdx.x; g < 4u * m; g += 512) {
      const uint32_t col = nb + (g & 3);
      if (col < (uint32_t)sstride) lds_s[(g >> 2) * sstride + col] = 0x7F;
    }
    __syncthreads();
  }

  v4f acc[NT][MT] = {};
  for (int turn = wave; turn < turns; turn += kWaves) {
    Turn now = next;
    if (turn + kWaves < turns) load(turn + kWaves, next);
    const int at = turn * 16 + 4 * q;
#pragma unroll
    for (int j = 0; j < MT; j++) {
      const int token = min(j * 16 + l15, m - 1);
      u32x4 c[4];
      uint32_t s;
      if constexpr (kPacked) {
        const uint8_t* p = xc + ((int64_t)token * nb + at) * 16;
#pragma unroll
        for (int b = 0; b < 4; b++)
          c[b] = at + b < nb ? *(const u32x4*)(p + b * 16)
                             : u32x4{0, 0, 0, 0};
        s = load_scales(xs + (int64_t)token * nb, at, nb);
      } else {
        const char* p = smem + token * crow + at * 16;
#pragma unroll
        for (int b = 0; b < 4; b++)
          c[b] = at + b < nb ? *(const u32x4*)(p + b * 16)
                             : u32x4{0, 0, 0, 0};
        s = at < nb ? *(const uint32_t*)(lds_s + token * sstride + at) : kUnit;
      }
#pragma unroll
      for (int i = 0; i < NT; i++) {
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            operand(now.c[i][0]), operand(c[0]), acc[i][j], 4, 4, 0,
            (int)now.s[i], 0, (int)s);
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            operand(now.c[i][1]), operand(c[1]), acc[i][j], 4, 4, 1,
            (int)now.s[i], 1, (int)s);
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            operand(now.c[i][2]), operand(c[2]), acc[i][j], 4, 4, 2,
            (int)now.s[i], 2, (int)s);
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            operand(now.c[i][3]), operand(c[3]), acc[i][j], 4, 4, 3,
            (int)now.s[i], 3, (int)s);
      }
    }
  }

  __syncthreads();  // the tokens' place is taken by the partial sums
  v4f* part = (v4f*)smem;  // [wave][NT][MT][64]
#pragma unroll
  for (int i = 0; i < NT; i++)
#pragma unroll
    for (int j = 0; j < MT; j++)
      part[((wave * NT + i) * MT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int e = threadIdx.x; e < NT * MT * 64; e += 512) {
    const int j = (e >> 6) % MT, i = (e >> 6) / MT;
    const int token = j * 16 + (e & 15);
    const int64_t col = n0 + i * 16 + 4 * ((e & 63) >> 4);
    const int valid = (int)min((int64_t)4, n - col);
    if (token >= m || valid <= 0) continue;
    v4f sum = part[e];
    for (int w = 1; w < kWaves; w++) sum += part[w * NT * MT * 64 + e];
    float f[4];
    for (int r = 0; r < 4; r++)
      f[r] = sum[r] + (bias && r < valid ? bias_at<T>(bias, col + r) : 0.f);
    store4<T>(y, (int64_t)token * n + col, f, valid);
  }
}

// ---------------------------------------------------------------------------
// launching
// ---------------------------------------------------------------------------
constexpr int kFewTokens = 64;
constexpr int64_t kFusedLds = 64 << 10;

int64_t few_lds(int64_t m, int64_t nb) {
  return m * ((nb + 1) * 16 + ((nb + 3) & ~3) + 4);
}

bool fuses(int64_t m, int64_t nb) {
  return m <= kFewTokens && few_lds(m, nb) <= kFusedLds;
}

template <LmType T, int WM, int WN, int FM, int FN>
void run_tile(const uint8_t* xc, const uint8_t* xs, const uint8_t* wc,
              const uint8_t* ws, const void* bias, void* y, int64_t m,
              int64_t n, int nb, hipStream_t stream) {
  constexpr int BM = WM * FM * 32, BN = WN * FN * 32;
  int64_t tm = (m + BM - 1) / BM, tn = (n + BN - 1) / BN;
  if (tm * tn >= (int64_t)1 << 28)
    throw std::runtime_error("product too large for one launch");
  tile_kernel<T, WM, WN, FM, FN>
      <<<dim3((unsigned)(tm * tn)), WM * WN * 64, 2 * (BM + BN) * 128,
         stream>>>(xc, xs, wc, ws, bias, y, m, n, nb, (int)tm, (int)tn);
  HIP_CHECK(hipGetLastError());
}

template <LmType T>
void run_linear(const void* x, int64_t stride, const uint8_t* xc,
                const uint8_t* xs, const uint8_t* wc, const uint8_t* ws,
                const void* bias, void* y, int64_t m, int64_t n, int64_t k,
                void* scratch, hipStream_t stream) {
  const int64_t nb = mx_blocks(k);
  const bool fused = x && fuses(m, nb);
  if (x && !fused) {
    uint8_t* codes = (uint8_t*)scratch;
    uint8_t* scales = codes + m * nb * kMxBytes;
    launch_mx_quantize(T, x, stride, codes, scales, m, k, stream);
    xc = codes;
    xs = scales;
  }
  if (m <= kFewTokens) {
    auto go = [&](auto mt, auto packed) {
      constexpr int MT = decltype(mt)::value;
      constexpr int NT = 1;
      constexpr bool P = decltype(packed)::value;
      int64_t lds = std::max<int64_t>(P ? 0 : few_lds(m, nb),
                                      (int64_t)8 * NT * MT * 64 * 16);
      few_kernel<T, MT, NT, P>
          <<<dim3((unsigned)((n + 16 * NT - 1) / (16 * NT))), 512, lds,
             stream>>>(x, stride, xc, xs, wc, ws, bias, y, (int)m, n, k,
                       (int)nb);
      HIP_CHECK(hipGetLastError());
    };
    auto by_mt = [&](auto packed) {
      switch ((m + 15) / 16) {
        case 1:
          return go(std::integral_constant<int, 1>{}, packed);
        case 2:
          return go(std::integral_constant<int, 2>{}, packed);
        case 3:
          return go(std::integral_constant<int, 3>{}, packed);
        default:
          return go(std::integral_constant<int, 4>{}, packed);
      }
    };
    fused ? by_mt(std::false_type{}) : by_mt(std::true_type{});
    return;
  }
  if (((m + 255) / 256) * ((n + 255) / 256) >= 256)
    run_tile<T, 2, 4, 4, 2>(xc, xs, wc, ws, bias, y, m, n, (int)nb, stream);
  else if (((m + 127) / 128) * ((n + 127) / 128) >= 256)
    run_tile<T, 2, 2, 2, 2>(xc, xs, wc, ws, bias, y, m, n, (int)nb, stream);
  else
    run_tile<T, 2, 2, 1, 1>(xc, xs, wc, ws, bias, y, m, n, (int)nb, stream);
}

}  // namespace

int64_t mx_linear_workspace(int64_t m, int64_t, int64_t k, bool packed) {
  const int64_t nb = mx_blocks(k);
  return packed || fuses(m, nb) ? 0 : m * nb * (kMxBytes + 1);
}

void launch_mx_linear(LmType t, const void* x, int64_t stride,
                      const uint8_t* xcodes, const uint8_t* xscales,
                      const uint8_t* wcodes, const uint8_t* wscales,
                      const void* bias, void* y, int64_t m, int64_t n,
                      int64_t k, void* ws, hipStream_t stream) {
  switch (t) {
    case LmType::F32:
      return run_linear<LmType::F32>(x, stride, xcodes, xscales, wcodes,
                                     wscales, bias, y, m, n, k, ws, stream);
    case LmType::BF16:
      return run_linear<LmType::BF16>(x, stride, xcodes, xscales, wcodes,
                                      wscales, bias, y, m, n, k, ws, stream);
    case LmType::F16:
      return run_linear<LmType::F16>(x, stride, xcodes, xscales, wcodes,
                                     wscales, bias, y, m, n, k, ws, stream);
  }
}
