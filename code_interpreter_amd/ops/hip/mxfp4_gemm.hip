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

template <LmType T>
struct Out {
  using type = typename std::conditional<
      T == LmType::F32, float,
      typename std::conditional<T == LmType::BF16, __bf16, _Float16>::type>::
      type;
};

// outputs n .. n + 3 of a row
template <LmType T>
__device__ __forceinline__ void store4(void* y, int64_t at, const float* f,
                                       int valid) {
  using E = typename Out<T>::type;
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
// Before the product, one launch quantises the tokens and lays out both
// operands' scales by steps of 256 elements of k: [step][row][8], 1 behind a
// row's end. Rows' scales for a step are then neighbours in memory, where in
// a row's own order a wave would touch a cache line for every row.
constexpr int kPrepareThreads = 256;

// A block that quantises takes kPrepareSteps steps of kPrepareRows rows: 8192
// x 8192 bf16 in 42 us, 46 with 1 step, 45 with 4.
constexpr int kPrepareSteps = 2, kPrepareRows = 32 / kPrepareSteps;
// of one that does not
constexpr int kLayRows = kPrepareThreads, kLaySteps = 4;

__device__ __forceinline__ void lay_out_scales(const uint8_t* from,
                                               uint2* to, int64_t rows,
                                               int nb, int steps, int blk) {
  // a row's parts share its cache lines: by blocks of one chiplet, which gets
  // every eighth
  const int parts = (steps + kLaySteps - 1) / kLaySteps, eight = 8 * parts;
  const int64_t row =
      ((int64_t)(blk / eight) * 8 + blk % 8) * kLayRows + threadIdx.x;
  const int t0 = blk % eight / 8 * kLaySteps;
  if (row >= rows) return;
  const uint8_t* p = from + row * nb;
  struct __attribute__((packed)) raw8 {
    uint32_t x, y;
    __device__ operator uint2() const { return {x, y}; }
  };
  uint2 v[kLaySteps];
#pragma unroll
  for (int i = 0; i < kLaySteps; i++)
    if (t0 + i < steps)
      v[i] = (t0 + i) * 8 + 8 <= nb
                 ? *(const raw8*)(p + (t0 + i) * 8)
                 : uint2{load_scales(p, (t0 + i) * 8, nb),
                         load_scales(p, (t0 + i) * 8 + 4, nb)};
#pragma unroll
  for (int i = 0; i < kLaySteps; i++)
    if (t0 + i < steps) to[(t0 + i) * rows + row] = v[i];
}

// blocks [0, x_blocks): x to codes and laid out scales, or (packed) its
// scales laid out; the others: the weight's scales laid out. The scales of a
// quantising block's rows are neighbours, 128 bytes for each of its two steps.
template <LmType T, bool kPacked>
__global__ __launch_bounds__(kPrepareThreads) void prepare_kernel(
    const char* __restrict__ x, int64_t stride,
    const uint8_t* __restrict__ xs, uint32_t* __restrict__ codes,
    uint8_t* __restrict__ xst, int64_t m, int64_t k, int x_blocks,
    const uint8_t* __restrict__ ws, uint2* __restrict__ wst, int64_t n,
    int nb, int steps) {
  if ((int)blockIdx.x >= x_blocks) {
    lay_out_scales(ws, wst, n, nb, steps, blockIdx.x - x_blocks);
    return;
  }
  if constexpr (kPacked) {
    lay_out_scales(xs, (uint2*)xst, m, nb, steps, blockIdx.x);
  } else {
    constexpr int kRowGroups = kPrepareSteps * 32;
    constexpr int kGroups = kPrepareRows * kRowGroups / kPrepareThreads;
    const int parts = (steps + kPrepareSteps - 1) / kPrepareSteps;
    const int64_t row0 = (int64_t)(blockIdx.x / parts) * kPrepareRows +
                         threadIdx.x / kRowGroups;
    // of a row's groups of 8 elements, and the block it belongs to
    const int col = blockIdx.x % parts * kRowGroups + threadIdx.x % kRowGroups;
    const int blk = col >> 2;
    if (blk >= steps * 8) return;  // whole waves or halves: of 32 groups
    u32x4 w[kGroups], w2[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; i++) {
      const int64_t row = row0 + i * (kPrepareThreads / kRowGroups);
      if (row < m)
        load8<T>(x + row * stride * Size<T>::value, (int64_t)col * kPer, k,
                 w[i], w2[i]);
    }
#pragma unroll
    for (int i = 0; i < kGroups; i++) {
      const int64_t row = row0 + i * (kPrepareThreads / kRowGroups);
      if (row >= m) break;
      uint32_t byte = block_scale<T>(w[i], w2[i]);
      if (blk < nb)
        codes[row * nb * 4 + col] =
            byte == 255 ? 0u : encode<T>(w[i], w2[i], scale_value(byte));
      if ((col & 3) == 0)
        xst[((blk >> 3) * m + row) * 8 + (blk & 7)] =
            blk < nb ? (uint8_t)byte : 0x7F;
    }
  }
}

// A block of WM x WN waves makes BM tokens x BN outputs; a wave FM x FN
// tiles of 32 x 32. A step takes 256 elements of k, 128 bytes of a row, into
// one of two buffers of shared memory by asynchronous loads of 16 bytes a
// lane. In shared memory the 8 units of 16 bytes of row r stand at their
// index ^ (r / 2 & 7), so that 16 lanes that read the same unit of 16 rows
// touch all of the 64 banks once.
//
// 8192^3 in 260 us on random codes at the best clock, 4.2 PFLOP/s, and up to
// 315 after long work; the instructions alone reach 5.2 there, since the power
// limit lowers the clock (on zeros 8.7, and this kernel 4.8). The matrix units
// are busy half of the cycles: a wave's 128 x 128 results take all of the
// accumulators, so that a tile's results go out while no products run, and a
// block's loads start anew. Without the stores the kernel takes 10 us less.
//
// A step is 4 instructions deep in k. While the matrix units work on one of
// them the next one's operands are read; the last one's time covers the
// barrier, the first reads of the next step's buffer and the start of the
// loads of the one after.
template <LmType T, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM* WN * 64, 1) void tile_kernel(
    const uint8_t* __restrict__ xc, const uint2* __restrict__ xs,
    const uint8_t* __restrict__ wc, const uint2* __restrict__ ws,
    const void* __restrict__ bias, void* __restrict__ y, int64_t m, int64_t n,
    int nb, int tiles_m, int tiles_n) {
#ifdef __HIP_DEVICE_COMPILE__  // buffer descriptors are no type on the host
  constexpr int kWaves = WM * WN;
  constexpr int BM = WM * FM * 32, BN = WN * FN * 32;
  constexpr int kRow = 128;
  constexpr int kBuf = (BM + BN) * kRow;
  constexpr int kLoadsX = BM / 8 / kWaves, kLoadsW = BN / 8 / kWaves;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0, "");
  static_assert(kWaves % 2 == 0, "");
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

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int l31 = lane & 31, h = lane >> 5;
  const int64_t row_bytes = (int64_t)nb * kMxBytes;

  // this lane's rows of each load, clamped to the last one: what is made of
  // a row behind it is not stored
  const uint8_t* xb = xc + m0 * row_bytes;
  const uint8_t* wb = wc + n0 * row_bytes;
  const int unit = (lane & 7) ^ (((wave & 1) * 4 + (lane >> 4)) & 7);
  uint32_t xo[kLoadsX], wo[kLoadsW];
#pragma unroll
  for (int i = 0; i < kLoadsX; i++) {
    int64_t r = (i * kWaves + wave) * 8 + (lane >> 3);
    xo[i] = (uint32_t)(min(r, m - 1 - m0) * row_bytes) + unit * 16;
  }
#pragma unroll
  for (int i = 0; i < kLoadsW; i++) {
    int64_t r = (i * kWaves + wave) * 8 + (lane >> 3);
    wo[i] = (uint32_t)(min(r, n - 1 - n0) * row_bytes) + unit * 16;
  }
  const int full = nb / 8, rest = nb % 8;  // steps; blocks behind them
  const int steps = full + (rest != 0);
  // in the last, short step a unit behind the row's end is read as its last
  const int back = rest && unit >= rest ? (unit - rest + 1) * 16 : 0;

  // The tile's rows as buffers: an asynchronous load is then one instruction,
  // with the row in a register of the lane and the step in a scalar one.
  auto buffer = [](const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(
        (void*)p, 0, (int)min(bytes, (int64_t)0xFFFFFFFF), 0x00020000);
  };
  const auto xr = buffer(xb, min(m - m0, (int64_t)BM) * row_bytes);
  const auto wr = buffer(wb, min(n - n0, (int64_t)BN) * row_bytes);
  // step t into buffer `into`
  auto load = [&](int t, int into, auto rsrc, uint32_t at, int to) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rsrc, (lds_void*)(smem + into * kBuf + to + wave * 1024), 16,
        (int)at - (t == full ? back : 0), t * kRow, 0, 0);
  };
  auto load_w = [&](int t, int into, int i) {
    load(t, into, wr, wo[i], i * kWaves * 1024);
  };
  auto load_x = [&](int t, int into, int i) {
    load(t, into, xr, xo[i], BN * kRow + i * kWaves * 1024);
  };

  // scales: the lower lanes take a step's blocks 0 to 3, the upper 4 to 7
  uint32_t xso[FM], wso[FN];
#pragma unroll
  for (int i = 0; i < FM; i++)
    xso[i] = (uint32_t)(min((int64_t)(wm * FM + i) * 32 + l31, m - 1 - m0) * 8) +
             4 * h;
#pragma unroll
  for (int i = 0; i < FN; i++)
    wso[i] = (uint32_t)(min((int64_t)(wn * FN + i) * 32 + l31, n - 1 - n0) * 8) +
             4 * h;
  uint32_t sx[FM], sw[FN];
  auto scale_x = [&](int t, int i) {
    return *(const uint32_t*)((const char*)(xs + (int64_t)t * m + m0) +
                              xso[i]);
  };
  auto scale_w = [&](int t, int i) {
    return *(const uint32_t*)((const char*)(ws + (int64_t)t * n + n0) +
                              wso[i]);
  };

  v16f acc[FN][FM] = {};
  struct Operands {
    u32x4 w[FN], x[FM];
  };
  // what instruction s of a step takes: blocks s (lower lanes) and 4 + s
  const int at0 = (wn * FN * 32 + l31) * kRow;
  const int at1 = (BN + wm * FM * 32 + l31) * kRow;
  // operand i of them: FN of the weights, then FM of the tokens
  auto read = [&](int t, int s, int i, Operands& o) {
    const char* from = smem + (t & 1) * kBuf;
    const int u = ((s + 4 * h) ^ (lane >> 1 & 7)) * 16;
    if (i < FN)
      o.w[i] = *(const u32x4*)(from + at0 + i * 32 * kRow + u);
    else
      o.x[i - FN] = *(const u32x4*)(from + at1 + (i - FN) * 32 * kRow + u);
  };
  auto product = [&](auto step, const Operands& o, int i, int j) {
    constexpr int s = decltype(step)::value;
    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
        operand(o.w[i]), operand(o.x[j]), acc[i][j], 4, 4, s, (int)sw[i], s,
        (int)sx[j]);
  };

  // all of this wave's loads have landed, and its reads are done
  auto settle = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  std::integral_constant<int, 0> s0;
  std::integral_constant<int, 1> s1;
  std::integral_constant<int, 2> s2;
  std::integral_constant<int, 3> s3;

  // The products of one instruction's depth, with `between(slot)` behind
  // each: what is read and loaded for later then goes out piece by piece
  // while the matrix units work, instead of holding up the products. The
  // compiler would gather it; the barriers for its scheduler keep the order.
  constexpr int kSlots = FN * FM;
  auto multiply = [&](auto step, const Operands& o, auto between) {
#pragma unroll
    for (int slot = 0; slot < kSlots; slot++) {
      product(step, o, slot / FM, slot % FM);
      __builtin_amdgcn_sched_barrier(0);
      between(slot);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // piece by piece: those of `count` that fall to this of the slots
  auto spread = [](int slot, int count, auto piece) {
#pragma unroll
    for (int i = 0; i < count; i++)
      if (i * kSlots / count == slot) piece(i);
  };
  // operands are read early in a part, one a slot
  constexpr int kReads = FN + FM;
  auto read_early = [&](int slot, int t, int s, Operands& o) {
#pragma unroll
    for (int i = 0; i < kReads; i++)
      if (i * kSlots / (2 * kReads) == slot) read(t, s, i, o);
  };

  // Step t's tokens and step t + 1's weights are under way while step t - 1
  // is worked on.
#pragma unroll
  for (int i = 0; i < kLoadsW; i++) load_w(0, 0, i);
#pragma unroll
  for (int i = 0; i < kLoadsX; i++) load_x(0, 0, i);
#pragma unroll
  for (int i = 0; i < FM; i++) sx[i] = scale_x(0, i);
#pragma unroll
  for (int i = 0; i < FN; i++) sw[i] = scale_w(0, i);
  settle();
#pragma unroll
  for (int i = 0; i < kLoadsW; i++) load_w(min(1, steps - 1), 1, i);
  Operands a, b;
#pragma unroll
  for (int i = 0; i < kReads; i++) read(0, 0, i, a);
  for (int t = 0; t < full; t++) {
    // No branches in here, which the compiler would gather the products
    // behind: where there is no next step, or none after it, the last one is
    // read and loaded again, into a buffer that is free.
    const int ahead = min(t + 1, steps - 1), next = min(t + 2, steps - 1);
    uint32_t nx[FM], nw[FN];
    multiply(s0, a, [&](int slot) {
      read_early(slot, t, 1, b);
      spread(slot, kLoadsX, [&](int i) { load_x(ahead, (t + 1) & 1, i); });
    });
    multiply(s1, b, [&](int slot) {
      read_early(slot, t, 2, a);
      spread(slot, FM, [&](int i) { nx[i] = scale_x(ahead, i); });
      spread(slot, FN, [&](int i) { nw[i] = scale_w(ahead, i); });
    });
    multiply(s2, a, [&](int slot) { read_early(slot, t, 3, b); });
    settle();  // every wave's part of step t + 1 is there, step t is read
    multiply(s3, b, [&](int slot) {
      read_early(slot, t + 1, 0, a);
      spread(slot, kLoadsW, [&](int i) { load_w(next, t & 1, i); });
    });
#pragma unroll
    for (int i = 0; i < FM; i++) sx[i] = nx[i];
#pragma unroll
    for (int i = 0; i < FN; i++) sw[i] = nw[i];
  }
  if (rest) {  // codes behind the row's end are made 0; their scales are 1
    // where there was no whole step, the tokens' part has landed in settle()
    auto last = [&](auto step) {
      constexpr int s = decltype(step)::value;
      if (s >= rest) return;
      const bool in = s + 4 * h < rest;
#pragma unroll
      for (int i = 0; i < kReads; i++) {
        read(full, s, i, a);
        u32x4& w = i < FN ? a.w[i] : a.x[i - FN];
        w = in ? w : u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++) product(step, a, i, j);
    };
    last(s0);
    last(s1);
    last(s2);
    last(s3);
  }

  // A lane holds 4 neighbouring outputs of one token at a time: stored from
  // there, rows would go out in pieces of 8 or 16 bytes. They pass through
  // shared memory, 32 tokens of a wave at a time, and go out 16 bytes a lane
  // along the rows.
  using E = typename Out<T>::type;
  using E4 = E __attribute__((ext_vector_type(4)));
  constexpr int kOutRow = FN * 32 * (int)sizeof(E);
  constexpr int kPad = kOutRow + 16;
  constexpr int kLanes = kOutRow / 16;  // of a row
  constexpr int kPer16 = 16 / (int)sizeof(E);
  static_assert(kWaves * 32 * kPad + BN * 4 <= 2 * kBuf, "");
  float* sb = (float*)smem;
  char* out = smem + BN * 4 + wave * 32 * kPad;
  settle();
  for (int i = threadIdx.x; i < BN; i += kWaves * 64)
    sb[i] = bias && n0 + i < n ? bias_at<T>(bias, n0 + i) : 0.f;
  __syncthreads();
  const int col = (lane % kLanes) * kPer16;
  const int64_t c0 = n0 + wn * FN * 32 + col;
#pragma unroll
  for (int j = 0; j < FM; j++) {
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int at = i * 32 + 8 * g + 4 * h;
        const v4f add = *(const v4f*)(sb + wn * FN * 32 + at);
        E4 v;
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = (E)(acc[i][j][4 * g + r] + add[r]);
        *(E4*)(out + l31 * kPad + at * (int)sizeof(E)) = v;
      }
    const int64_t row0 = m0 + (wm * FM + j) * 32;
#pragma unroll
    for (int p = 0; p < 32; p += 64 / kLanes) {
      const int r = p + lane / kLanes;
      const u32x4 v = *(const u32x4*)(out + r * kPad + col * (int)sizeof(E));
      if (row0 + r >= m) continue;
      E* to = (E*)y + (row0 + r) * n + c0;
      if (c0 + kPer16 <= n) {
        *(raw16*)to = v;
      } else {
        const E* e = (const E*)(out + r * kPad) + col;
        for (int q = 0; q < kPer16 && c0 + q < n; q++) to[q] = e[q];
      }
    }
  }
#endif
}

// ---------------------------------------------------------------------------
// small tiles: where there are too few large ones to fill the chip
// ---------------------------------------------------------------------------
// The time is the memory's answer, not the products': so a block keeps the
// loads of kStages - 1 steps under way, in a ring of buffers, and small tiles
// make many blocks. WM x WN x WK waves make a tile of 32 WM tokens x 32 WN
// outputs; of the 4 instructions of a step WK waves take a share each, and
// their sums are added in a fixed order at the end. Rows stand in shared
// memory as for the large tiles; the scales of a step come the same way, 4
// bytes a lane. 333 x 5001 x 2056 takes 9.5 us, 37 x 4096 x 4096 6.1 us, more
// than half of it waiting; buffers beyond these 3 to 6 gave nothing.
template <LmType T, int WM, int WN, int WK, int kStages>
__global__ __launch_bounds__(WM* WN* WK * 64) void small_kernel(
    const uint8_t* __restrict__ xc, const uint2* __restrict__ xs,
    const uint8_t* __restrict__ wc, const uint2* __restrict__ ws,
    const void* __restrict__ bias, void* __restrict__ y, int64_t m, int64_t n,
    int nb, int tiles_m, int tiles_n) {
#ifdef __HIP_DEVICE_COMPILE__  // buffer descriptors are no type on the host
  constexpr int kWaves = WM * WN * WK;
  constexpr int BM = WM * 32, BN = WN * 32;
  constexpr int kRow = 128;
  constexpr int kScales = (BM + BN) * kRow;  // behind the rows
  constexpr int kBuf = kScales + kWaves * 256;
  constexpr int kLoads = (BM + BN) / 8 / kWaves;  // of a wave, 8 rows each
  constexpr int kPerStep = kLoads + 1;            // with one of scales
  constexpr int kWait = (kStages - 2) * kPerStep;
  static_assert(kWaves % 2 == 0 && BM % (8 * kWaves) == 0 &&
                    BN % (8 * kWaves) == 0 && kWait < 64, "");
  constexpr int kOut = BN + 4;  // floats between tokens in the epilogue
  static_assert(WK * BM * kOut * 4 <= kStages * kBuf, "");
  extern __shared__ __attribute__((aligned(16))) char smem[];

  int id = blockIdx.x;
  {  // neighbouring tiles to one chiplet, columns of 8 tiles of tokens
    const int all = tiles_m * tiles_n, q = all / 8, r = all % 8;
    const int xcd = id % 8, idx = id / 8;
    id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  }
  const int per = 8 * tiles_n, group = id / per;
  const int high = min(8, tiles_m - group * 8);
  const int64_t m0 = (int64_t)(group * 8 + (id % per) % high) * BM;
  const int64_t n0 = (int64_t)((id % per) / high) * BN;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave % WK, wn = wave / WK % WN, wm = wave / (WK * WN);
  const int l31 = lane & 31, h = lane >> 5;
  const int64_t row_bytes = (int64_t)nb * kMxBytes;
  const int full = nb / 8, rest = nb % 8;
  const int steps = full + (rest != 0);

  auto buffer = [](const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(
        (void*)p, 0, (int)min(bytes, (int64_t)0xFFFFFFFF), 0x00020000);
  };
  const auto wr = buffer(wc + n0 * row_bytes,
                         min(n - n0, (int64_t)BN) * row_bytes);
  const auto xr = buffer(xc + m0 * row_bytes,
                         min(m - m0, (int64_t)BM) * row_bytes);
  // rows of the weight first, then of the tokens; 8 of one operand a load
  const int unit = (lane & 7) ^ (((wave & 1) * 4 + (lane >> 4)) & 7);
  const int back = rest && unit >= rest ? (unit - rest + 1) * 16 : 0;
  uint32_t off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; i++) {
    const int64_t r = (i * kWaves + wave) * 8 + (lane >> 3);
    const int64_t at = i * kWaves * 8 < BN ? min(r, n - 1 - n0)
                                           : min(r - BN, m - 1 - m0);
    off[i] = (uint32_t)(at * row_bytes) + unit * 16;
  }
  // scales: words 2 r, 2 r + 1 of row r. A wave behind the last word loads
  // the first ones once more, to a place that is not read.
  constexpr int kScaleWaves = (BM + BN) * 2 / 64;
  static_assert(kScaleWaves <= kWaves, "");
  const int word0 = (wave % kScaleWaves) * 64;
  const bool of_x = word0 >= BN * 2;
  const auto sr = of_x ? buffer(xs, m * steps * 8) : buffer(ws, n * steps * 8);
  const int sstep = (int)(of_x ? m : n) * 8;
  const int64_t r0 = of_x ? m0 : n0, last = (of_x ? m : n) - 1;
  const int64_t srow = min(r0 + (word0 + lane - (of_x ? BN * 2 : 0)) / 2, last);
  const int soff = (int)srow * 8 + (lane & 1) * 4;

  auto stage = [&](int t, int into) {
    char* to = smem + into * kBuf;
    const int less = t == full ? back : 0;
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      lds_void* at = (lds_void*)(to + (i * kWaves + wave) * 1024);
      if (i * kWaves * 8 < BN)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            wr, at, 16, (int)off[i] - less, t * kRow, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            xr, at, 16, (int)off[i] - less, t * kRow, 0, 0);
    }
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        sr, (lds_void*)(to + kScales + wave * 256), 4, soff, t * sstep, 0, 0);
  };

  v16f acc = {};
  const int aw = (wn * 32 + l31) * kRow, ax = (BN + wm * 32 + l31) * kRow;
  const int sw = kScales + (wn * 32 + l31) * 8 + 4 * h;
  const int sx = kScales + (BN + wm * 32 + l31) * 8 + 4 * h;
  auto multiply = [&](int at, auto last) {
    const char* from = smem + at * kBuf;
    // a wave's instructions are wk * 4 / WK and those behind it: their scales
    // are shifted to the front of the word
    const uint32_t s0 = *(const uint32_t*)(from + sw) >> (wk * 4 / WK * 8);
    const uint32_t s1 = *(const uint32_t*)(from + sx) >> (wk * 4 / WK * 8);
    auto one = [&](auto step) {
      constexpr int s = decltype(step)::value;
      const int blk = wk * 4 / WK + s;
      if (decltype(last)::value && blk >= rest) return;
      const int u = ((blk + 4 * h) ^ (lane >> 1 & 7)) * 16;
      u32x4 w = *(const u32x4*)(from + aw + u);
      u32x4 x = *(const u32x4*)(from + ax + u);
      if (decltype(last)::value && blk + 4 * h >= rest)
        w = x = u32x4{0, 0, 0, 0};
      acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
          operand(w), operand(x), acc, 4, 4, s, (int)s0, s, (int)s1);
    };
    one(std::integral_constant<int, 0>{});
    if constexpr (WK < 4) one(std::integral_constant<int, 1>{});
    if constexpr (WK < 2) {
      one(std::integral_constant<int, 2>{});
      one(std::integral_constant<int, 3>{});
    }
  };

  // Behind the last step the last one is loaded again, into buffers that are
  // free, so that the number of loads under way is always the same.
#pragma unroll
  for (int t = 0; t < kStages - 1; t++) stage(min(t, steps - 1), t);
  auto arrive = [] {
    // this wave's loads of a step have landed, and its reads of the step
    // before are done; behind the barrier every wave's
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((kWait & 15) | 7 << 4 |
                               (kWait >> 4) << 14);  // and lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  int now = 0, into = kStages - 1;
  for (int t = 0; t < full; t++) {
    arrive();
    stage(min(t + kStages - 1, steps - 1), into);
    multiply(now, std::false_type{});
    now = now + 1 == kStages ? 0 : now + 1;
    into = into + 1 == kStages ? 0 : into + 1;
  }
  if (rest) {
    arrive();
    multiply(now, std::true_type{});
  }

  // the waves' sums as [wk][token][output]
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  float* sums = (float*)smem;
  float* mine = sums + (wk * BM + wm * 32 + l31) * kOut + wn * 32 + 4 * h;
#pragma unroll
  for (int g = 0; g < 4; g++)
    *(v4f*)(mine + 8 * g) = v4f{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2],
                                acc[4 * g + 3]};
  __syncthreads();
#pragma unroll
  for (int i = 0; i < BM * BN / (kWaves * 256); i++) {
    const int e = (i * kWaves * 64 + threadIdx.x) * 4;
    const int64_t row = m0 + e / BN, col = n0 + e % BN;
    const int valid = (int)min((int64_t)4, n - col);
    if (row >= m || valid <= 0) continue;
    v4f sum = *(const v4f*)(sums + e / BN * kOut + e % BN);
#pragma unroll
    for (int k = 1; k < WK; k++)
      sum += *(const v4f*)(sums + (k * BM + e / BN) * kOut + e % BN);
    float f[4];
    for (int r = 0; r < 4; r++)
      f[r] = sum[r] + (bias && r < valid ? bias_at<T>(bias, col + r) : 0.f);
    store4<T>(y, row * n + col, f, valid);
  }
#endif
}

// ---------------------------------------------------------------------------
// few tokens
// ---------------------------------------------------------------------------
// The weights are read once, from memory into registers, and bound the time; G
// groups of 16 tokens are held against them. A block makes 16 outputs of all
// tokens: its 8 waves take turns along k, 512 elements a turn, and add up
// through shared memory at the end, in a fixed order. The loads of two turns
// are under way before the first is worked on. The tokens come from memory
// as codes (packed), or are quantised by each block into its shared memory,
// which saves a launch and costs the more the more tokens there are. One
// token, 8192 x 8192: 35.7 MB in 9.3 to 10.7 us.
//
// Instruction j of a turn takes blocks 4 j + q from the lanes 16 q .. 16 q +
// 15, so that 4 lanes load 64 bytes in a row. A lane holds the 16 scales of
// its row's turn, and shifts the one for instruction j to the word's front.
using raw16b = uint32_t __attribute__((ext_vector_type(4), aligned(1)));

// bytes of a token's codes and scales in shared memory
__host__ __device__ constexpr int few_codes(int nb) { return (nb | 1) * 16; }
__host__ __device__ constexpr int few_scales(int nb) {
  return ((nb + 15) / 16 | 1) * 16;
}

struct Turn {
  u32x4 c[4], s;
};

// blocks [at, at + 16) of a row of nb, from memory or shared memory; behind
// its end codes of 0 and scales of 1
template <bool kScales>
__device__ __forceinline__ void load_turn(const uint8_t* codes,
                                          const uint8_t* scales, int at,
                                          int nb, int q, Turn& to) {
  if (at + 16 <= nb) {
#pragma unroll
    for (int j = 0; j < 4; j++)
      to.c[j] = *(const u32x4*)(codes + (int64_t)(at + 4 * j + q) * 16);
    if constexpr (kScales) to.s = *(const raw16b*)(scales + at);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int blk = at + 4 * j + q;
    to.c[j] = blk < nb ? *(const u32x4*)(codes + (int64_t)blk * 16)
                       : u32x4{0, 0, 0, 0};
    if constexpr (kScales)
      to.s[j] = (blk < nb ? (uint32_t)scales[blk] : 0x7Fu) << (8 * q);
  }
}

template <LmType T, bool kPacked, int G>
__global__ __launch_bounds__(512, G > 1 ? 2 : 4) void few_kernel(
    const void* __restrict__ x, int64_t stride,
    const uint8_t* __restrict__ xc, const uint8_t* __restrict__ xs,
    const uint8_t* __restrict__ wc, const uint8_t* __restrict__ ws,
    const void* __restrict__ bias, void* __restrict__ y, int m, int64_t n,
    int64_t k, int nb) {
  constexpr int kWaves = 8;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l15 = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int turns = (nb + 15) / 16;

  const int64_t r = min(n0 + l15, n - 1);
  const uint8_t* wrow = wc + r * nb * kMxBytes;
  const uint8_t* srow = ws + r * nb;
  Turn next, after;
  if (wave < turns) load_turn<true>(wrow, srow, wave * 16, nb, q, next);
  if (wave + kWaves < turns)
    load_turn<true>(wrow, srow, (wave + kWaves) * 16, nb, q, after);

  // In shared memory tokens stand an odd number of 16-byte units apart: 16
  // lanes that read the same unit of 16 tokens touch all banks once.
  const int crow = few_codes(nb), sstride = few_scales(nb);
  uint8_t* lds_s = (uint8_t*)smem + m * crow;
  if constexpr (!kPacked) {
    const uint32_t per_row = (uint32_t)nb * 4, groups = per_row * m;
    constexpr int kGroups = 4;  // loads under way
    for (uint32_t g0 = threadIdx.x; g0 < groups; g0 += 512 * kGroups) {
      u32x4 w[kGroups], w2[kGroups];
      uint32_t row[kGroups], col[kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; i++) {
        const uint32_t g = g0 + i * 512;
        row[i] = g / per_row;
        col[i] = g - row[i] * per_row;
        if (g < groups)
          load8<T>((const char*)x + row[i] * stride * Size<T>::value,
                   (int64_t)col[i] * kPer, k, w[i], w2[i]);
      }
#pragma unroll
      for (int i = 0; i < kGroups; i++) {
        if (g0 + i * 512 >= groups) break;  // whole blocks: a multiple of 4
        const uint32_t byte = block_scale<T>(w[i], w2[i]);
        *(uint32_t*)(smem + row[i] * crow + col[i] * 4) =
            byte == 255 ? 0u : encode<T>(w[i], w2[i], scale_value(byte));
        if ((col[i] & 3) == 0)
          lds_s[row[i] * sstride + (col[i] >> 2)] = (uint8_t)byte;
      }
    }
    // scales of 1 up to the end of a row's last turn
    for (uint32_t g = threadIdx.x; g < 16u * m; g += 512) {
      const int col = nb + (int)(g & 15);
      if (col < turns * 16) lds_s[(g >> 4) * sstride + col] = 0x7F;
    }
    __syncthreads();
  }

  v4f acc[G] = {};
  int token[G];
#pragma unroll
  for (int g = 0; g < G; g++) token[g] = min(g * 16 + l15, m - 1);
  for (int turn = wave; turn < turns; turn += kWaves) {
    Turn now = next;
    next = after;
    if (turn + 2 * kWaves < turns)
      load_turn<true>(wrow, srow, (turn + 2 * kWaves) * 16, nb, q, after);
#pragma unroll
    for (int g = 0; g < G; g++) {
      Turn tok;
      if constexpr (kPacked) {
        load_turn<true>(xc + (int64_t)token[g] * nb * 16,
                        xs + (int64_t)token[g] * nb, turn * 16, nb, q, tok);
      } else {
        load_turn<false>((const uint8_t*)smem + token[g] * crow, nullptr,
                         turn * 16, nb, q, tok);
        tok.s = *(const u32x4*)(lds_s + token[g] * sstride + turn * 16);
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
        acc[g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            operand(now.c[j]), operand(tok.c[j]), acc[g], 4, 4, 0,
            (int)(now.s[j] >> (8 * q)), 0, (int)(tok.s[j] >> (8 * q)));
    }
  }

  __syncthreads();  // the tokens' place is taken by the partial sums
  v4f* part = (v4f*)smem;  // [group][wave][64]
#pragma unroll
  for (int g = 0; g < G; g++) part[g * 512 + threadIdx.x] = acc[g];
  __syncthreads();
  if (wave >= G) return;  // a wave adds up a group
  const int64_t col = n0 + 4 * q;
  const int valid = (int)min((int64_t)4, n - col);
  const int row = wave * 16 + l15;
  if (row >= m || valid <= 0) return;
  v4f sum = part[wave * 512 + lane];
#pragma unroll
  for (int w = 1; w < kWaves; w++) sum += part[wave * 512 + w * 64 + lane];
  float f[4];
  for (int r = 0; r < 4; r++)
    f[r] = sum[r] + (bias && r < valid ? bias_at<T>(bias, col + r) : 0.f);
  store4<T>(y, (int64_t)row * n + col, f, valid);
}

// ---------------------------------------------------------------------------
// launching
// ---------------------------------------------------------------------------
// Few tokens are up to 16, or 64 where one block a compute unit makes all
// outputs: two do not fit, of more than 16.
constexpr int64_t kFewTokens = 16, kFewTokensAtOnce = 64;
constexpr int64_t kFill = 512 * 16;  // outputs, of two blocks a unit
// Quantised by each block for itself they take 0.1 ns an element for each of
// the chip's fills with blocks, and save a launch of 3 us, as much of the
// host's time again. In us, so and with a launch:
// 4096 x  512, m = 17: 4.2,  5.9; m = 48:   6.0, 6.1
// 4096 x 1024, m = 32: 6.1,  6.3
// 8192 x 1024, m = 16: 4.9,  6.5; m = 32:  10.3, 6.4
// 4096 x 4096, m =  4: 5.0,  6.2; m =  8:   6.5, 6.4
// 8192 x 8192, m =  1: 10.3, 12.2; m = 4:  13.0, 13.0
// 131072 x 4096, m = 1: 68.6, 71; m =  8: 121.5, 72
constexpr int64_t kFusedElements = 1 << 15;
// From codes a block reads all tokens' along the whole of k, which weighs more
// the longer it is. Against small tiles, m = 1, 8, 16:
//   8192 x  4096  6.0,  6.8,  7.6
//   8192 x  8192  9.2, 10.8, 12.2  tiles 12.3, 12.7, 12.9
//  16384 x  8192 16.7, 18.5, 21.0        18.5, 18.5, 18.6
//   8192 x 16384 15.7, 18.3, 21.1        18.7, 19.3, 19.2
//  32768 x  4096 17.7, 18.7, 21.1        22.4, 24.2, 25.1
// 131072 x  4096 68.7, 68.3, 76.9        95.5, 95.1, 96.4
// and m = 17, 32, 33, 64:
//   4096 x  4096  4.9,  5.7,  6.4,  8.1         8.5,  8.4,  8.7,  8.8
//   4096 x  8192  8.5, 10.0, 11.3, 14.7        11.5, 11.4, 11.6, 11.6
//   4096 x 16384 14.3, 16.8, 19.3, 25.7        16.9, 17.0, 17.3, 17.3
// Tokens that are quantised first cost the tiles nothing more, and this 3 us:
//   4096 x  2048  6.4,  6.8,  7.3,  8.2         6.9,  7.0,  7.1,  7.1
//   4096 x  4096  7.6,  8.7,  9.2, 11.3         9.3,  9.3,  9.4,  9.5
//   4096 x  8192 11.6, 13.3, 14.6, 18.0        12.1, 12.2, 12.4, 12.4
constexpr int64_t kFewK = 4096;
constexpr int64_t kFewWeights = 1 << 25;

int64_t few_lds(int64_t m, int64_t nb) {
  return m * (few_codes((int)nb) + few_scales((int)nb));
}

bool fuses(int64_t m, int64_t n, int64_t nb) {
  const int64_t elements = m * nb * kMxBlock;
  if (m > kFewTokens)
    return m <= kFewTokensAtOnce && n <= kFill / 2 &&
           elements <= kFusedElements;
  return elements * ((n + kFill - 1) / kFill) <= kFusedElements;
}

bool few(int64_t m, int64_t n, int64_t nb, bool packed) {
  const int64_t k = nb * kMxBlock;
  if (!packed && fuses(m, n, nb)) return true;
  if (m > kFewTokens) {
    const int64_t most = packed ? kFewTokensAtOnce : kFewTokensAtOnce / 2;
    return m <= most && n <= kFill / 2 && m * k <= most * kFewK;
  }
  if (k <= kFewK || n * k <= kFewWeights) return true;
  return packed && (m <= kFewTokens / 2 || n * k <= 2 * kFewWeights);
}

template <LmType T, int WM, int WN, int FM, int FN>
void run_tile(const uint8_t* xc, const uint2* xs, const uint8_t* wc,
              const uint2* ws, const void* bias, void* y, int64_t m,
              int64_t n, int nb, hipStream_t stream) {
  constexpr int BM = WM * FM * 32, BN = WN * FN * 32;
  int64_t tm = (m + BM - 1) / BM, tn = (n + BN - 1) / BN;
  tile_kernel<T, WM, WN, FM, FN>
      <<<lm_grid(tm * tn, WM * WN * 64), WM * WN * 64, 2 * (BM + BN) * 128,
         stream>>>(xc, xs, wc, ws, bias, y, m, n, nb, (int)tm, (int)tn);
  HIP_CHECK(hipGetLastError());
}

template <LmType T, int WM, int WN, int WK, int kStages>
void run_small(const uint8_t* xc, const uint2* xs, const uint8_t* wc,
               const uint2* ws, const void* bias, void* y, int64_t m,
               int64_t n, int nb, hipStream_t stream) {
  constexpr int BM = WM * 32, BN = WN * 32;
  int64_t tm = (m + BM - 1) / BM, tn = (n + BN - 1) / BN;
  small_kernel<T, WM, WN, WK, kStages>
      <<<lm_grid(tm * tn, WM * WN * WK * 64), WM * WN * WK * 64,
         kStages * ((BM + BN) * 128 + WM * WN * WK * 256), stream>>>(
          xc, xs, wc, ws, bias, y, m, n, nb, (int)tm, (int)tn);
  HIP_CHECK(hipGetLastError());
}

// what the tiles' workspace holds: x's codes, its scales by steps, the
// weight's
struct TileSpace {
  int64_t codes, xs, ws;
};

int64_t round16(int64_t v) { return (v + 15) & ~(int64_t)15; }

TileSpace tile_space(int64_t m, int64_t n, int64_t nb, bool packed) {
  int64_t steps = (nb + 7) / 8;
  return {packed ? 0 : m * nb * kMxBytes, round16(m * steps * 8),
          n * steps * 8};
}

template <LmType T>
void run_tiles(const void* x, int64_t stride, const uint8_t* xc,
               const uint8_t* xs, const uint8_t* wc, const uint8_t* ws,
               const void* bias, void* y, int64_t m, int64_t n, int64_t k,
               void* scratch, hipStream_t stream) {
  const int64_t nb = mx_blocks(k), steps = (nb + 7) / 8;
  TileSpace space = tile_space(m, n, nb, x == nullptr);
  uint8_t* codes = (uint8_t*)scratch;
  uint8_t* xst = codes + space.codes;
  uint2* wst = (uint2*)(xst + space.xs);
  auto lay_blocks = [&](int64_t rows) {
    return (rows + 8 * kLayRows - 1) / (8 * kLayRows) * 8 *
           ((steps + kLaySteps - 1) / kLaySteps);
  };
  const int64_t w_blocks = lay_blocks(n);
  const int64_t x_blocks =
      x ? (m + kPrepareRows - 1) / kPrepareRows *
              ((steps + kPrepareSteps - 1) / kPrepareSteps)
        : lay_blocks(m);
  // a token tile's offsets into the codes are 32 bits
  if (nb * kMxBytes >= 1 << 23)
    throw std::runtime_error("rows too long for one launch");
  const dim3 grid = lm_grid(x_blocks + w_blocks, kPrepareThreads);
  if (x)
    prepare_kernel<T, false><<<grid, kPrepareThreads, 0, stream>>>(
        (const char*)x, stride, nullptr, (uint32_t*)codes, xst, m, k,
        (int)x_blocks, ws, wst, n, (int)nb, (int)steps);
  else
    prepare_kernel<T, true><<<grid, kPrepareThreads, 0, stream>>>(
        nullptr, 0, xs, nullptr, xst, m, k, (int)x_blocks, ws, wst, n,
        (int)nb, (int)steps);
  HIP_CHECK(hipGetLastError());
  if (x) xc = codes;
  auto* xs2 = (const uint2*)xst;
  // The largest tiles of which there are enough to fill the chip, and of which
  // the tokens fill more than half of one. In us, of m x n x k with tiles of
  // 256 x 256, 128 x 128 (2 buffers), 64 x 128, 64 x 64 (3), 32 x 64 (4), 32 x
  // 32 (6):
  // 2000 x 5001 x 2056 30.6, 33.0,    -,    -, 49.0, 74.0
  // 2000 x 4096 x 4096 38.8, 33.5, 40.5,    -, 56.8, 86.9
  // 1200 x 8192 x 8192 60.6, 74.8, 78.2,    -,    -,    -
  //  800 x 8192 x 8192 56.1, 48.3, 58.5,    -,    -,    -
  //  800 x 4096 x 4096 34.0, 22.5, 22.1, 25.5, 28.7, 40.1
  //  333 x 8192 x 8192 52.1, 34.1, 32.4,    -,    -,    -
  //  500 x 4096 x 4096    -, 21.2, 16.4, 16.7, 21.5,    -
  //  333 x 5001 x 2056 25.7, 15.2, 12.0, 13.4, 16.4, 20.2
  //  200 x 4096 x 4096    -, 19.5, 14.2, 13.0, 12.5,    -
  //  100 x 4096 x 4096 30.8, 19.3, 13.5, 12.2, 10.8, 11.1
  //  333 x 700 x 700   20.9, 11.6,    -,  9.1,  8.2,  7.6
  //  160 x 131072 x 4096 107, 124,  126,  137,  160,    -
  //  128 x 131072 x 4096 106,  91,  104,  113,  138,    -
  //   64 x 131072 x 4096 100,  86,   79,   86,   95,    -
  //   32 x 32768 x 4096 33.4, 25.8, 19.2, 19.7, 19.1,   -
  auto tiles = [&](int64_t bm, int64_t bn) {
    return ((m + bm - 1) / bm) * ((n + bn - 1) / bn);
  };
  const int b = (int)nb;
  // the small tiles' scales are addressed in 31 bits
  const bool far = std::max(m, n) * steps * 8 >= (int64_t)1 << 31;
  // A tile of 256 x 256 is a compute unit's alone, so that its start and end
  // are not hidden: it wants a long k, and not a second round for a few. The
  // rule goes by k and the tiles' number alone, and near its borders takes up
  // to a fifth more than 128 x 128 would: most for tokens that fill little
  // more than half of a tile, as 164. 256 x 256 and 128 x 128:
  // 8192 x 8192 x  512 56.1, 54.6, x 1024 77.1, 75.3, x 1536 91.5, 93.5
  // 4096 x 4096 x  512 21.0, 20.7, x 1024 24.8, 25.2, x 1536 29.9, 30.8
  //  164 x 43710 x 512 21.9, 17.2, x 1024 25.3, 21.3, x 1536 28.3, 24.9
  // 7055 x 3310 x 1536 50.2, 41.9, x 3100 78.8, 75.9 (364 of them)
  const int64_t large = tiles(256, 256);
  if (m > 128 && k >= 1024 && large >= 144 && !(large > 256 && large <= 384))
    run_tile<T, 2, 2, 4, 4>(xc, xs2, wc, wst, bias, y, m, n, b, stream);
  else if ((m > 64 && tiles(128, 128) >= 240) || far)
    run_tile<T, 2, 2, 2, 2>(xc, xs2, wc, wst, bias, y, m, n, b, stream);
  else if (tiles(64, 128) >= 160)
    run_small<T, 2, 4, 1, 3>(xc, xs2, wc, wst, bias, y, m, n, b, stream);
  else if (tiles(64, 64) >= 256)
    run_small<T, 2, 2, 1, 3>(xc, xs2, wc, wst, bias, y, m, n, b, stream);
  else if (tiles(32, 64) >= 256)
    run_small<T, 1, 2, 2, 4>(xc, xs2, wc, wst, bias, y, m, n, b, stream);
  else
    run_small<T, 1, 1, 4, 6>(xc, xs2, wc, wst, bias, y, m, n, b, stream);
}

template <class F>
void by_groups(int64_t m, F f) {
  if (m <= 16)
    f(std::integral_constant<int, 1>{});
  else if (m <= 32)
    f(std::integral_constant<int, 2>{});
  else
    f(std::integral_constant<int, 4>{});
}

template <LmType T>
void run_linear(const void* x, int64_t stride, const uint8_t* xc,
                const uint8_t* xs, const uint8_t* wc, const uint8_t* ws,
                const void* bias, void* y, int64_t m, int64_t n, int64_t k,
                void* scratch, hipStream_t stream) {
  const int64_t nb = mx_blocks(k);
  if (!few(m, n, nb, x == nullptr))
    return run_tiles<T>(x, stride, xc, xs, wc, ws, bias, y, m, n, k, scratch,
                        stream);
  const dim3 grid = lm_grid((n + 15) / 16, 512);
  const int64_t sums = 512 * sizeof(v4f);  // of 16 tokens
  if (x && fuses(m, n, nb)) {
    by_groups(m, [&](auto groups) {
      constexpr int G = decltype(groups)::value;
      few_kernel<T, false, G>
          <<<grid, 512, std::max(few_lds(m, nb), G * sums), stream>>>(
              x, stride, nullptr, nullptr, wc, ws, bias, y, (int)m, n, k,
              (int)nb);
    });
  } else {
    if (x) {
      uint8_t* codes = (uint8_t*)scratch;
      uint8_t* scales = codes + m * nb * kMxBytes;
      launch_mx_quantize(T, x, stride, codes, scales, m, k, stream);
      xc = codes;
      xs = scales;
    }
    by_groups(m, [&](auto groups) {
      constexpr int G = decltype(groups)::value;
      few_kernel<T, true, G><<<grid, 512, G * sums, stream>>>(
          nullptr, 0, xc, xs, wc, ws, bias, y, (int)m, n, k, (int)nb);
    });
  }
  HIP_CHECK(hipGetLastError());
}

}  // namespace

int64_t mx_linear_workspace(int64_t m, int64_t n, int64_t k, bool packed) {
  const int64_t nb = mx_blocks(k);
  if (few(m, n, nb, packed))
    return packed || fuses(m, n, nb) ? 0 : m * nb * (kMxBytes + 1);
  TileSpace space = tile_space(m, n, nb, packed);
  return space.codes + space.xs + space.ws;
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
