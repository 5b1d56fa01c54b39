// Rows of logits: log probabilities of given tokens, entropies, the most
// likely alternatives, and distillation from recorded teacher logits, with
// their backward passes.
//
// Mathematics. With c = log2(e) / T, m = max x, e_j = 2^(c (x_j - m)):
//   S = sum e_j, U = sum e_j c (x_j - m)
//   ln p_j = (x_j - m) / T - ln S,  H = ln S - ln 2 * U / S
// A thread keeps (m, S, U) of what it has seen; a new maximum m' scales
//   S by r = 2^(c (m - m')), and U becomes r (U + S c (m - m'))
// which also joins two threads', waves' or blocks' triples. So a row is
// read once. The difference x - m is taken before the product with c: of a
// mask of the type's lowest value, c x alone would be an infinity.
//
// An element of -inf has no share: e is 0, and the exponent that U takes is
// held at kLow, since 0 * -inf is no number. A row with nothing but -inf
// has m = -inf and S = 0 and is reported as empty. A NaN or +inf makes S
// NaN, and with it all of the row's numbers.
//
// Memory bounds all of it, with the vector units close behind for 16-bit
// logits: 9 instructions an element forward, an exponential among them. 4096
// x 131072 bf16: 217 us forward, 4.9 TB/s; backward 340 us, 6.3 TB/s (part
// of what is read again comes from the chip's cache). Distillation backward,
// 4096 x 65536: 183 us, 5.9 TB/s. A large copy: 4.8 TB/s.
//
// All sums are 32-bit, over a fixed split of the row and in a fixed order:
// the same input gives the same bits.

#include <algorithm>
#include <type_traits>

#include "lm.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLow = -16384.f;  // 2^kLow is 0
constexpr int kThreads = 256;
constexpr int kMaxKeys = 4096;  // of a row's parts together, 32 KB
constexpr int kWaves = kThreads / 64;

// 16 bytes at any element's address: the hardware takes vector loads and
// stores at 2-byte alignment, so rows of odd length need no path of their own
using raw16 = uint32_t __attribute__((ext_vector_type(4), aligned(2)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

template <LmType T>
struct Elem;
template <>
struct Elem<LmType::F32> {
  using type = float;
  static constexpr int kVec = 4;
  static constexpr uint32_t kNegInf = 0xFF800000u;  // in every lane of a word
  static __device__ float get(const u32x4& w, int i) {
    return __uint_as_float(w[i]);
  }
  static __device__ void put(u32x4& w, int i, uint32_t bits) { w[i] = bits; }
  static __device__ float load(const type* p) { return *p; }
  static __device__ uint32_t bits(const type* p) { return __float_as_uint(*p); }
  static __device__ void store(type* p, float f) { *p = f; }
};
template <>
struct Elem<LmType::BF16> {
  using type = uint16_t;
  static constexpr int kVec = 8;
  static constexpr uint32_t kNegInf = 0xFF80FF80u;
  static __device__ float get(const u32x4& w, int i) {
    return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
  }
  static __device__ void put(u32x4& w, int i, uint32_t b) {
    w[i >> 1] = i & 1 ? (w[i >> 1] & 0xFFFFu) | b << 16
                      : (w[i >> 1] & 0xFFFF0000u) | b;
  }
  static __device__ float load(const type* p) {
    return __uint_as_float((uint32_t)*p << 16);
  }
  static __device__ uint32_t bits(const type* p) { return *p; }
  static __device__ void store(type* p, float f) {
    __bf16 h = (__bf16)f;
    __builtin_memcpy(p, &h, 2);
  }
};
template <>
struct Elem<LmType::F16> {
  using type = uint16_t;
  static constexpr int kVec = 8;
  static constexpr uint32_t kNegInf = 0xFC00FC00u;
  static __device__ float half(uint32_t b) {
    uint16_t u = (uint16_t)b;
    _Float16 h;
    __builtin_memcpy(&h, &u, 2);
    return (float)h;
  }
  static __device__ float get(const u32x4& w, int i) {
    return half(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu);
  }
  static __device__ void put(u32x4& w, int i, uint32_t b) {
    Elem<LmType::BF16>::put(w, i, b);
  }
  static __device__ float load(const type* p) { return half(*p); }
  static __device__ uint32_t bits(const type* p) { return *p; }
  static __device__ void store(type* p, float f) {
    _Float16 h = (_Float16)f;
    __builtin_memcpy(p, &h, 2);
  }
};

// f32 values rounded to the type, into a 16-byte word
template <LmType T>
__device__ u32x4 pack(const float* f) {
  u32x4 w;
  if constexpr (T == LmType::F32) {
    for (int i = 0; i < 4; i++) w[i] = __float_as_uint(f[i]);
  } else if constexpr (T == LmType::BF16) {
    using b2 = __bf16 __attribute__((ext_vector_type(2)));
    using f2 = float __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; i++) {
      b2 h = __builtin_convertvector((f2{f[2 * i], f[2 * i + 1]}), b2);
      uint32_t u;
      __builtin_memcpy(&u, &h, 4);
      w[i] = u;
    }
  } else {
    using h2 = _Float16 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; i++) {
      h2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]};
      uint32_t u;
      __builtin_memcpy(&u, &h, 4);
      w[i] = u;
    }
  }
  return w;
}

// elements [at, at + kVec) of a row of `end` elements; -inf behind its end
template <LmType T>
__device__ u32x4 load_vec(const typename Elem<T>::type* row, int64_t at,
                          int64_t end) {
  using E = Elem<T>;
  if (at + E::kVec <= end) return *(const raw16*)(row + at);
  u32x4 w = {E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf};
#pragma unroll
  for (int i = 0; i < E::kVec; i++)
    if (at + i < end) E::put(w, i, E::bits(row + at + i));
  return w;
}

__device__ __forceinline__ float exp2_raw(float x) {
  return __builtin_amdgcn_exp2f(x);
}

struct Triple {
  float m, s, u;
};

__device__ __forceinline__ float or_zero(float m) {
  return m == -INFINITY ? 0.f : m;
}

// a's sums under the maximum m >= a.m
__device__ __forceinline__ Triple under(Triple a, float m, float c) {
  float y = (a.m - or_zero(m)) * c;
  float r = exp2_raw(y);
  return {m, a.s * r, (a.u + a.s * fmaxf(y, kLow)) * r};
}

__device__ __forceinline__ Triple join(Triple a, Triple b, float c) {
  float m = fmaxf(a.m, b.m);
  Triple x = under(a, m, c), y = under(b, m, c);
  return {m, x.s + y.s, x.u + y.u};
}

__device__ __forceinline__ float wave_sum(float a) {
#pragma unroll
  for (int d = 32; d; d >>= 1) a += __shfl_xor(a, d);
  return a;
}
__device__ __forceinline__ float wave_max(float a) {
#pragma unroll
  for (int d = 32; d; d >>= 1) a = fmaxf(a, __shfl_xor(a, d));
  return a;
}

__device__ __forceinline__ Triple join_wave(Triple a, float c) {
  a = under(a, wave_max(a.m), c);
  return {a.m, wave_sum(a.s), wave_sum(a.u)};
}

// bits that order as the values do. Both zeros are one value.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

// a value's order above, the complement of its index below: a larger key is a
// better alternative, of equal values the earlier. 0 stands for none.
__device__ __forceinline__ uint64_t make_key(float x, uint32_t index) {
  return (uint64_t)order_of(x) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  return value_of((uint32_t)(key >> 32));
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) {
  return ~(uint32_t)key;
}

// The r-th largest of the kMany numbers that each lane of a wave holds, 0 if
// there are not so many, from the top kBits of them (a lower bound of it, for
// numbers that have more): each bit is set where r of them stay at or above.
template <int kBits, int kMany>
__device__ __forceinline__ uint32_t rth_of_wave(const uint32_t (&x)[kMany],
                                                int r) {
  uint32_t found = 0;
#pragma unroll
  for (int bit = 31; bit > 31 - kBits; bit--) {
    const uint32_t with = found | 1u << bit;
    int there = 0;
#pragma unroll
    for (int i = 0; i < kMany; i++) there += __popcll(__ballot(x[i] >= with));
    if (there >= r) found = with;
  }
  return found;
}

// ---------------------------------------------------------------------------
// alternatives
// ---------------------------------------------------------------------------
// candidates that are held at a time: the best so far and those of a word a
// thread, at least
constexpr int kCap = kMaxTop + kThreads * 8;
constexpr int kFew = 256;  // that are ranked as they are
constexpr int kPending = 4;  // chunks between two looks at their number

struct TopShared {
  // the best so far, then candidates; a pair more than there can be
  alignas(16) uint64_t keys[kCap + 2];
  uint64_t best[kMaxTop];
  uint64_t most[kThreads];  // the threads' largest
  float least;    // a candidate is larger than this
  int count;      // entries of keys
  int flag[3];    // whether a chunk has candidates, by its number mod 3
};

// The k best of keys[0 .. n), which are all different, to best, sorted: each
// key's place is the number of larger ones. keys[n] is written, and keys are
// 16-byte aligned.
__device__ void rank_keys(uint64_t* keys, int n, int k, uint64_t* best) {
  using Pair = uint64_t __attribute__((ext_vector_type(2)));
  if (threadIdx.x == 0) keys[n] = 0;  // the last pair's other half
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t key = keys[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 2) {
      const Pair o = *(const Pair*)&keys[j];
      rank += (o[0] > key) + (o[1] > key);
    }
    if (rank < k) best[rank] = key;
  }
}

// keys[0 .. n) -> the k best, sorted, at keys[0 ..). Returns their number.
__device__ int keep_best(TopShared& sh, int n, int k) {
  rank_keys(sh.keys, n, k, sh.best);
  __syncthreads();
  const int have = min(n, k);
  for (int i = threadIdx.x; i < have; i += kThreads) sh.keys[i] = sh.best[i];
  if (threadIdx.x == 0) {
    sh.count = have;
    if (have == k) sh.least = key_value(sh.best[k - 1]);
  }
  __syncthreads();
  return have;
}

// The k best of a row's elements, from chunks that the block holds in
// registers: words w[0 .. U) of each thread, thread t's word i at element
// base + (i * 256 + t) * kVec. Chunks come in the order of their indexes, so
// that an element must be larger than the last of the k best so far to
// displace it; few of a later chunk are. Candidates are gathered, for kPending
// chunks without a barrier, and ranked when there are 2 k + 32 or more, or at
// the end: ranking raises the bar for what follows, and costs the square of
// their number (2048 x 131072 bf16 with 64: 152 us, 161 from 3 k + 32 on).
//
// For the first chunk, and where candidates are many: k threads hold an
// element that is not below the k-th largest of the threads' own maxima, which
// so is a lower bound of the chunk's k-th largest element. Not many elements
// pass it but where many are equal, or few threads have one at all. Candidates
// that still are many are spread over all threads, whose largest give a bound
// once more, by index among equal ones. Those that do not fit come word by
// word: 64 rows of 131072 equal bf16 logits with 20 alternatives take 32 us, 18
// where they differ.
template <LmType T, int U>
struct Top {
  using E = Elem<T>;
  TopShared& sh;
  const int k;
  const typename E::type* const src;  // the row, and where its part ends
  const int64_t end;
  int have = 0, count = 0, chunk = 0;  // equal in all threads
  int64_t since;  // what stands before it is settled, or in count
  float least = -INFINITY;

  __device__ Top(TopShared& sh, int k, const typename E::type* src,
                 int64_t begin, int64_t end)
      : sh(sh), k(k), src(src), end(end), since(begin) {
    if (threadIdx.x == 0) {
      sh.count = 0;
      sh.least = least;
      sh.flag[0] = sh.flag[1] = sh.flag[2] = 0;
    }
    __syncthreads();
  }

  // Elements larger than `least` and not less than `bound` to the keys. Words
  // in which no lane has one, most of them, are passed over as a whole.
  __device__ void append(const u32x4& w, float word_max, int64_t at,
                         float bound) {
    if (!__any((word_max > least) & (word_max >= bound))) return;
#pragma unroll
    for (int j = 0; j < E::kVec; j++) {
      const float x = E::get(w, j);
      if (!((x > least) & (x >= bound))) continue;
      const int place = atomicAdd(&sh.count, 1);
      if (place < kCap) sh.keys[place] = make_key(x, (uint32_t)(at + j));
    }
  }

  __device__ int64_t place_of(int64_t base, int i) const {
    return base + (int64_t)(i * kThreads + threadIdx.x) * E::kVec;
  }

  __device__ void append_all(const u32x4* w, const float* word_max,
                             int64_t base, float bound) {
#pragma unroll
    for (int i = 0; i < U; i++)
      append(w[i], word_max[i], place_of(base, i), bound);
  }

  __device__ void merge(int n) {
    have = count = keep_best(sh, n, k);
    least = sh.least;
  }

  // The k-th largest of the threads' numbers, from the top bits of them.
  __device__ uint32_t kth_of_block(uint32_t mine) {
    uint32_t* const order = (uint32_t*)sh.most;
    order[threadIdx.x] = mine;
    __syncthreads();
    uint32_t all[kWaves];
#pragma unroll
    for (int i = 0; i < kWaves; i++)
      all[i] = order[i * 64 + (threadIdx.x & 63)];
    return rth_of_wave<20>(all, k);
  }

  // n > kFew keys to those that are not below the k-th largest of the threads'
  // largest keys
  __device__ int thin(int n) {
    constexpr int kMine = (kCap + kThreads - 1) / kThreads;
    const int tid = threadIdx.x;
    uint64_t mine[kMine], most = 0;
#pragma unroll
    for (int i = 0; i < kMine; i++) {
      mine[i] = tid + i * kThreads < n ? sh.keys[tid + i * kThreads] : 0;
      most = max(most, mine[i]);
    }
    sh.most[tid] = most;
    __syncthreads();
    if (tid == 0) sh.count = 0;
    uint32_t all[kWaves], low[kWaves];
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      const uint64_t key = sh.most[i * 64 + (tid & 63)];
      all[i] = (uint32_t)(key >> 32);
      low[i] = (uint32_t)key;
    }
    const uint32_t found = rth_of_wave<32>(all, k);
    int more = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      more += __popcll(__ballot(all[i] > found));
      if (all[i] != found) low[i] = 0;
    }
    const uint64_t bound =
        (uint64_t)found << 32 | rth_of_wave<32>(low, k - more);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; i++)
      if (mine[i] >= max(bound, (uint64_t)1))
        sh.keys[atomicAdd(&sh.count, 1)] = mine[i];
    __syncthreads();
    return sh.count;
  }

  // n keys to the best
  __device__ void settle(int n) {
    if (n > kFew) n = thin(n);
    merge(n);
  }

  // What the chunks before `upto` have left. Where candidates did not fit,
  // what is not settled comes once more, from memory: held in registers until
  // here the chunks would cost all rows theirs.
  __device__ void review(int64_t upto, float bound, bool always) {
    __syncthreads();
    const int n = sh.count;
    __syncthreads();
    if (n > kCap) {
      if (threadIdx.x == 0) sh.count = count;
      __syncthreads();
      if (count > have) merge(count);
#pragma unroll 1
      for (; since < upto; since += kThreads * E::kVec) {
        const int64_t at = since + threadIdx.x * E::kVec;
        const u32x4 word = load_vec<T>(src, at, end);
        append(word, INFINITY, at, bound);
        __syncthreads();
        settle(sh.count);
      }
    } else if (n >= 2 * k + 32 || (always && n > have)) {
      settle(n);
    } else {
      count = n;
    }
    since = upto;
  }

  __device__ void take(const u32x4* w, const float* word_max, int64_t base,
                       float thread_max, bool last) {
    const int64_t upto = base + kThreads * E::kVec * U;
    const int now = chunk % 3;
    float bound = -INFINITY;
    chunk++;
    if (have < k) {
      if (now || chunk > 3) {
        if (__any(thread_max > least) && (threadIdx.x & 63) == 0)
          sh.flag[now] = 1;
        __syncthreads();
        // of the chunk after the next: it is set behind another barrier
        if (threadIdx.x == 0) sh.flag[(now + 2) % 3] = 0;
        if (!sh.flag[now]) {
          since = upto;
          return;
        }
      }
      // NaN's order would be the largest of all; no number's is below -inf's
      const uint32_t none = order_of(-INFINITY);
      bound = value_of(max(
          kth_of_block(thread_max == thread_max ? order_of(thread_max) : none),
          none));
      append_all(w, word_max, base, bound);
      last = true;
    } else {
      append_all(w, word_max, base, bound);
    }
    if (last || chunk < 4 || chunk % kPending == 0) review(upto, bound, last);
  }
};

// ---------------------------------------------------------------------------
// what is made of a row's sums
// ---------------------------------------------------------------------------
struct LogprobsEnd {
  const int64_t* tokens;
  int64_t ignore;
  float inv_t;
  int top;
  float *logprobs, *entropy, *top_lp;
  int64_t* top_ids;
  RowStats* stats;
};

struct DistillEnd {
  LmType type;  // of the teacher's record
  const void* teacher;
  const int64_t* ids;
  int k;
  float inv_t;
  float *row_loss, *q;
  RowStats* stats;
};

// A row's token, and its logit: read before the row's sums are joined, so
// that the two loads, one upon the other, are over by then.
struct Token {
  float x;
  bool ignored, outside;
};

template <LmType T>
__device__ Token token_of(int64_t id, const typename Elem<T>::type* src,
                          int64_t v, const LogprobsEnd& e) {
  const bool ignored = id == e.ignore;
  const bool outside = !ignored && (id < 0 || id >= v);
  return {ignored || outside ? 0.f : Elem<T>::load(src + id), ignored,
          outside};
}

// a row's log probability, entropy and what its backward needs, by one
// thread
__device__ void write_row(int64_t row, const Triple& t, const Token& token,
                          const LogprobsEnd& e) {
  const float log2_sum = log2f(t.s);
  const bool ignored = token.ignored, outside = token.outside;
  const bool empty = t.m == -INFINITY && t.s == 0.f;
  float lp, h;
  if (ignored) {
    lp = h = 0.f;
  } else if (outside) {
    lp = h = NAN;
  } else if (empty) {
    lp = -INFINITY;
    h = 0.f;
  } else {
    lp = (token.x - t.m) * e.inv_t - log2_sum * kLn2;
    h = (log2_sum - t.u / t.s) * kLn2;
    if (!(t.s == t.s)) lp = NAN;
  }
  e.logprobs[row] = lp;
  e.entropy[row] = h;
  if (e.stats)
    e.stats[row] = {outside ? NAN : t.m, log2_sum, h,
                  ignored || (empty && !outside) ? 0.f : 1.f};
}

// an alternative of a row; key 0 stands for none
__device__ void write_top(int64_t row, int place, uint64_t key,
                          const Triple& t, const Token& token,
                          const LogprobsEnd& e) {
  if (token.ignored) key = 0;
  const int64_t at = row * e.top + place;
  e.top_lp[at] =
      key ? (key_value(key) - t.m) * e.inv_t - log2f(t.s) * kLn2 : -INFINITY;
  e.top_ids[at] = key ? (int64_t)key_index(key) : -1;
}

__device__ float load_any(LmType t, const void* p, int64_t i) {
  switch (t) {
    case LmType::F32:
      return ((const float*)p)[i];
    case LmType::BF16:
      return Elem<LmType::BF16>::load((const uint16_t*)p + i);
    default:
      return Elem<LmType::F16>::load((const uint16_t*)p + i);
  }
}

// A wave's part of a row's record: 4 entries a lane. Read in two steps, the
// logits at the entries' tokens upon the entries.
template <LmType T>
struct Record {
  static constexpr int kMine = kMaxRecord / 64;
  float z[kMine], x[kMine];
  int64_t id[kMine];  // -1: none

  __device__ void load_entries(int64_t row, const DistillEnd& e) {
#pragma unroll
    for (int i = 0; i < kMine; i++) {
      const int at = (threadIdx.x & 63) + 64 * i;
      id[i] = at < e.k ? e.ids[row * e.k + at] : -1;
      z[i] = at < e.k ? load_any(e.type, e.teacher, row * e.k + at) : 0.f;
    }
  }

  __device__ void load_logits(const typename Elem<T>::type* src, int64_t v) {
#pragma unroll
    for (int i = 0; i < kMine; i++)
      x[i] = id[i] >= 0 && id[i] < v ? Elem<T>::load(src + id[i]) : 0.f;
  }
};

// a row by a wave: the teacher's softmax over its record, and
// T^2 sum q (ln q - ln p). The logarithms are kept in units of 1 / T, and their
// sum in quarters, so that recorded logits of the type's lowest value overflow
// only where the loss does. Returns (in every lane) the loss, and whether the
// row has a record.
struct RowLoss {
  float loss;
  bool there;
};

template <LmType T>
__device__ RowLoss distill_row(int64_t row, Record<T> rec, int64_t v,
                               const DistillEnd& e, float c, const Triple& t) {
  constexpr int kMine = Record<T>::kMine;
  const int lane = threadIdx.x & 63;
  auto& z = rec.z;
  auto& id = rec.id;
  float top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kMine; i++) {
    if (id[i] == -1) z[i] = -INFINITY;
    if (z[i] == -INFINITY) id[i] = -1;
    bad |= z[i] != z[i] || z[i] == INFINITY ||
           (id[i] != -1 && (id[i] < 0 || id[i] >= v));
    top = fmaxf(top, z[i]);
  }
  bad = __any(bad);
  const bool empty = t.m == -INFINITY && t.s == 0.f;
  const float log2_sum = log2f(t.s);
  top = wave_max(top);
  const bool absent = top == -INFINITY && !bad;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMine; i++)
    sum += id[i] != -1 ? exp2_raw((z[i] - top) * c) : 0.f;
  sum = wave_sum(sum);
  const float log2_q = log2f(sum);
  const float temp = 1.f / e.inv_t;
  const float log_q = log2_q * kLn2 * temp, log_p = log2_sum * kLn2 * temp;
  float loss = 0.f;
#pragma unroll
  for (int i = 0; i < kMine; i++) {
    int at = lane + 64 * i;
    float share = 0.f;
    if (id[i] != -1 && !bad) {
      share = exp2_raw((z[i] - top) * c - log2_q);
      float lq = z[i] - top - log_q;
      float lp = empty ? -INFINITY : rec.x[i] - t.m - log_p;
      if (share > 0.f) loss = fmaf(share, (lq - lp) * 0.25f, loss);
    }
    if (at < e.k) e.q[row * e.k + at] = share;
  }
  loss = wave_sum(loss) * (4.f * temp);
  loss = absent ? 0.f : bad ? NAN : loss;
  if (lane == 0) {
    e.row_loss[row] = loss;
    // in the entropy's place: whether the row counts in the mean
    e.stats[row] = {bad ? NAN : t.m, log2_sum, absent ? 0.f : 1.f,
                  absent || (empty && !bad) ? 0.f : 1.f};
  }
  return {loss, !absent};
}

// ---------------------------------------------------------------------------
// one pass over a row, or over one of `splits` parts of it
// ---------------------------------------------------------------------------
struct NoTop {
  __device__ NoTop(int&, int, const void*, int64_t, int64_t) {}
};

struct Part {
  Triple t;
  float pad;
};

// `direct`: a row is one block's, which also makes the results of its sums;
// else they are left in parts and part_keys, for a kernel that joins them.
template <LmType T, int U, bool kTop, class End>
__global__ __launch_bounds__(kThreads, 4) void score_kernel(
    const typename Elem<T>::type* __restrict__ x, int64_t stride, int64_t v,
    int splits, int64_t part_len, float c, bool direct, End end_of_row,
    Part* __restrict__ parts, uint64_t* __restrict__ part_keys) {
  using E = Elem<T>;
  constexpr bool kDistill = std::is_same<End, DistillEnd>::value;
  constexpr int kChunk = kThreads * E::kVec * U;
  __shared__ typename std::conditional<kTop, TopShared, int>::type sh;
  __shared__ Triple wave_t[kWaves];

  const int64_t row = blockIdx.x / (unsigned)splits;
  const int64_t begin = (blockIdx.x % (unsigned)splits) * part_len;
  const int64_t end = min(v, begin + part_len);
  const typename E::type* src = x + row * stride;
  const int tid = threadIdx.x;
  int k = 0;
  if constexpr (kTop) k = end_of_row.top;

  typename std::conditional<kTop, Top<T, U>, NoTop>::type best(
      sh, k, src, begin, end);

  Triple t = {-INFINITY, 0.f, 0.f};
  u32x4 next[U];
#pragma unroll
  for (int i = 0; i < U; i++)
    next[i] = load_vec<T>(src, begin + (int64_t)(i * kThreads + tid) * E::kVec,
                          end);
  for (int64_t base = begin; base < end; base += kChunk) {
    u32x4 w[U];
#pragma unroll
    for (int i = 0; i < U; i++) w[i] = next[i];
    if (base + kChunk < end) {
#pragma unroll
      for (int i = 0; i < U; i++)
        next[i] = load_vec<T>(
            src, base + kChunk + (int64_t)(i * kThreads + tid) * E::kVec, end);
    }
    float word_max[U], chunk_max = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; i++) {
      word_max[i] = E::get(w[i], 0);
#pragma unroll
      for (int j = 1; j < E::kVec; j++)
        word_max[i] = fmaxf(word_max[i], E::get(w[i], j));
      chunk_max = fmaxf(chunk_max, word_max[i]);
    }
    if (chunk_max > t.m) t = under(t, chunk_max, c);
    const float m = or_zero(t.m);
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int i = 0; i < U; i++)
#pragma unroll
      for (int j = 0; j < E::kVec; j++) {
        float y = (E::get(w[i], j) - m) * c;
        float e = exp2_raw(y);
        s += e;
        if constexpr (!kDistill) u = fmaf(e, fmaxf(y, kLow), u);
      }
    t.s += s;
    t.u += u;
    if constexpr (kTop)
      best.take(w, word_max, base, chunk_max, base + kChunk >= end);
  }

  t = join_wave(t, c);
  if ((tid & 63) == 0) wave_t[tid >> 6] = t;
  __syncthreads();
  t = wave_t[0];
  for (int i = 1; i < kWaves; i++) t = join(t, wave_t[i], c);
  if (!direct) {
    if (tid == 0) parts[blockIdx.x].t = t;
    if constexpr (kTop) {
      if (tid < k)
        part_keys[(int64_t)blockIdx.x * k + tid] =
            tid < best.have ? sh.keys[tid] : 0;
    }
  } else if constexpr (kDistill) {
    if (tid < 64) {
      Record<T> rec;
      rec.load_entries(row, end_of_row);
      rec.load_logits(src, v);
      distill_row<T>(row, rec, v, end_of_row, c, t);
    }
  } else {
    const Token token =
        token_of<T>(end_of_row.tokens[row], src, v, end_of_row);
    if (tid == 0) write_row(row, t, token, end_of_row);
    if constexpr (kTop) {
      if (tid < k)
        write_top(row, tid, tid < best.have ? sh.keys[tid] : 0, t, token,
                  end_of_row);
    }
  }
}

// the parts of a row, by one wave
__device__ Triple join_parts(const Part* parts, int splits, float c) {
  Triple t = {-INFINITY, 0.f, 0.f};
  for (int i = threadIdx.x & 63; i < splits; i += 64)
    t = join(t, parts[i].t, c);
  return join_wave(t, c);
}

// ---------------------------------------------------------------------------
// token log probabilities
// ---------------------------------------------------------------------------
// a wave a row, without alternatives
template <LmType T>
__global__ __launch_bounds__(kThreads) void logprobs_rows_kernel(
    const typename Elem<T>::type* __restrict__ x, int64_t stride,
    int64_t rows, int64_t v, float c, const Part* __restrict__ parts,
    int splits, LogprobsEnd e) {
  int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= rows) return;
  const Token token = token_of<T>(e.tokens[row], x + row * stride, v, e);
  const Triple t = join_parts(parts + row * splits, splits, c);
  if ((threadIdx.x & 63) == 0) write_row(row, t, token, e);
}

// The r-th largest of the lanes' keys, or a lower bound of it, 0 counting as
// none. Keys of equal values are told apart by their indexes only from kTies
// too many on: a few equal ones are common in 16 bits, and cost less than this.
constexpr int kTies = 8;

template <LmType T>
__device__ uint64_t rth_key(uint64_t key, int r) {
  // the bits of a 16-bit type's order behind those are all 0, or 1 where the
  // value is negative
  constexpr int kBits = T == LmType::F32 ? 32 : 20;
  constexpr uint32_t kRest = T == LmType::F32 ? 0 : 0xFFFu;
  const uint32_t order = (uint32_t)(key >> 32) & ~kRest;
  const uint32_t found = rth_of_wave<kBits>({order}, r);
  if (!found) return 0;
  uint32_t below = 0;
  if (__popcll(__ballot(order >= found)) >= r + kTies) {
    const int more = __popcll(__ballot(order > found));
    below = rth_of_wave<32>({order == found ? (uint32_t)key : 0u}, r - more);
  }
  const uint32_t rest = found & 0x80000000u ? 0 : kRest;
  return (uint64_t)(found | rest) << 32 | below;
}

// A block a row, with alternatives: joins the parts' sorted lists. Where r
// lists have a key of at least b in place p, there are r p such keys: so the
// ceil(k / p)-th largest of the lists' keys in place p is a lower bound of
// the k-th best key of all. Each wave finds the bound of another p; few keys
// pass the largest of them, and these are ranked.
template <LmType T>
__global__ __launch_bounds__(kThreads) void top_rows_kernel(
    const typename Elem<T>::type* __restrict__ x, int64_t stride, int64_t v,
    float c, const Part* __restrict__ parts,
    const uint64_t* __restrict__ part_keys, int splits, LogprobsEnd e) {
  constexpr int kMine = kMaxKeys / kThreads;
  __shared__ alignas(16) uint64_t keys[kMaxKeys + 2];
  __shared__ uint64_t best[kMaxTop], bounds[kWaves];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, k = e.top;
  const uint64_t* src = part_keys + row * splits * k;
  const int all = splits * k;
  const int64_t id = e.tokens[row];
  // splits is 64 at most: a list a lane
  const int place = min(k, (k + splits - 1) / splits << (tid >> 6));
  const uint64_t listed = lane < splits ? src[lane * k + place - 1] : 0;
  uint64_t mine[kMine];
#pragma unroll
  for (int i = 0; i < kMine; i++)
    mine[i] = tid + i * kThreads < all ? src[tid + i * kThreads] : 0;
  const uint64_t bound_of_wave = rth_key<T>(listed, (k + place - 1) / place);
  const Token token = token_of<T>(id, x + row * stride, v, e);
  const Triple t = join_parts(parts + row * splits, splits, c);
  if (lane == 0) bounds[tid >> 6] = bound_of_wave;
  if (tid == 0) count = 0;
  if (tid < k) best[tid] = 0;
  __syncthreads();
  uint64_t bound = 1;  // none is no alternative
#pragma unroll
  for (int i = 0; i < kWaves; i++) bound = max(bound, bounds[i]);
#pragma unroll
  for (int i = 0; i < kMine; i++)
    if (mine[i] >= bound) keys[atomicAdd(&count, 1)] = mine[i];
  __syncthreads();
  const int n = count;
  rank_keys(keys, n, k, best);
  if (tid == 0) write_row(row, t, token, e);
  __syncthreads();
  if (tid < k) write_top(row, tid, best[tid], t, token, e);
}

// dx_j = -p_j (a + b ln p_j) at every j, and g_lp / T more at the token,
// with a = (g_lp + g_H H) / T, b = g_H / T
template <LmType T, int U>
__global__ __launch_bounds__(kThreads) void logprobs_bwd_kernel(
    const typename Elem<T>::type* __restrict__ x, int64_t stride, int64_t v,
    int chunks, const int64_t* __restrict__ tokens, float inv_t, float c,
    const RowStats* __restrict__ stats, const float* __restrict__ g_lp,
    const float* __restrict__ g_h, typename Elem<T>::type* __restrict__ dx) {
  using E = Elem<T>;
  const int64_t row = blockIdx.x / (unsigned)chunks;
  const int64_t base =
      (int64_t)(blockIdx.x % (unsigned)chunks) * (kThreads * E::kVec * U);
  const RowStats st = stats[row];
  const float g = g_lp ? g_lp[row] : 0.f, gh = g_h ? g_h[row] : 0.f;
  const float a = (g + gh * st.entropy) * inv_t, b = gh * inv_t * kLn2;
  const bool live = st.live != 0.f;
  const int64_t token = live ? tokens[row] : -1;
  const typename E::type* src = x + row * stride;
  typename E::type* dst = dx + row * v;
  u32x4 w[U];
  if (live) {
#pragma unroll
    for (int i = 0; i < U; i++)
      w[i] = load_vec<T>(
          src, base + (int64_t)(i * kThreads + threadIdx.x) * E::kVec, v);
  }
#pragma unroll
  for (int i = 0; i < U; i++) {
    const int64_t at = base + (int64_t)(i * kThreads + threadIdx.x) * E::kVec;
    if (at >= v) continue;
    float d[E::kVec];
    if (live) {
#pragma unroll
      for (int j = 0; j < E::kVec; j++) {
        float y = (E::get(w[i], j) - st.max) * c - st.log2_sum;
        d[j] = -exp2_raw(y) * fmaf(b, fmaxf(y, kLow), a);
      }
      if ((uint64_t)(token - at) < (uint64_t)E::kVec) {
#pragma unroll
        for (int j = 0; j < E::kVec; j++)
          if (token - at == j) d[j] += g * inv_t;
      }
    } else {
#pragma unroll
      for (int j = 0; j < E::kVec; j++) d[j] = 0.f;
    }
    if (at + E::kVec <= v) {
      *(raw16*)(dst + at) = pack<T>(d);
    } else {
#pragma unroll
      for (int j = 0; j < E::kVec; j++)
        if (at + j < v) E::store(dst + at + j, d[j]);
    }
  }
}

// ---------------------------------------------------------------------------
// distillation
// ---------------------------------------------------------------------------
// The waves' sums, in their order, by the block's first thread.
__device__ void write_total(double s, double n, int mean, float* total,
                            float* count) {
  __shared__ double wave_s[16], wave_n[16];
  const int waves = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    wave_s[threadIdx.x >> 6] = s;
    wave_n[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < waves; i++) {
    s += wave_s[i];
    n += wave_n[i];
  }
  const double by = mean && n > 1 ? n : 1;
  *total = (float)(s / by);
  *count = (float)by;
}

// rows of distillation whose parts one block joins, a wave a row, and adds up:
// a launch less. In us, so and with that launch: 3 x 70000 f16 7.0, 8.5; by
// four rows a wave, 61 x 131072 17.3, 11.0.
constexpr int kOneBlock = 16;

// kWhole: one block for all rows, which also adds them up
template <LmType T, bool kWhole>
__global__ __launch_bounds__(kWhole ? kOneBlock * 64 : kThreads) void
distill_rows_kernel(const typename Elem<T>::type* __restrict__ x,
                    int64_t stride, int64_t rows, int64_t v, float c,
                    const Part* __restrict__ parts, int splits, DistillEnd e,
                    int mean, float* __restrict__ total,
                    float* __restrict__ count) {
  const int64_t row =
      (int64_t)blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
  double s = 0, n = 0;
  if (row < rows) {
    Record<T> rec;
    rec.load_entries(row, e);
    rec.load_logits(x + row * stride, v);
    const Triple t = join_parts(parts + row * splits, splits, c);
    const RowLoss r = distill_row<T>(row, rec, v, e, c, t);
    s = r.loss;
    n = r.there;
  }
  if constexpr (kWhole) write_total(s, n, mean, total, count);
}

// sum or mean of the rows' losses, in a fixed order, in 64 bits; one block
__global__ __launch_bounds__(1024) void distill_total_kernel(
    const float* __restrict__ row_loss, const RowStats* __restrict__ stats,
    int64_t rows, int mean, float* __restrict__ total,
    float* __restrict__ count) {
  double s = 0, n = 0;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    s += row_loss[i];
    n += stats[i].entropy;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    s += __shfl_xor(s, d);
    n += __shfl_xor(n, d);
  }
  write_total(s, n, mean, total, count);
}

// dx_j = g T (p_j - sum of q at j). The block writes p_j of its chunk, and
// then the few elements that the record names once more: whole values, from
// the logit itself, so that each is rounded once.
template <LmType T, int U>
__global__ __launch_bounds__(kThreads) void distill_bwd_kernel(
    const typename Elem<T>::type* __restrict__ x, int64_t stride, int64_t v,
    int chunks, const int64_t* __restrict__ ids, const float* __restrict__ q,
    int k, float inv_t, float c, const RowStats* __restrict__ stats,
    const float* __restrict__ grad, int64_t grad_stride,
    const float* __restrict__ count, typename Elem<T>::type* __restrict__ dx) {
  using E = Elem<T>;
  constexpr int kChunk = kThreads * E::kVec * U;
  static_assert(kMaxRecord == kThreads, "");
  __shared__ alignas(16) int s_id[kMaxRecord];
  __shared__ alignas(16) float s_q[kMaxRecord];
  const int64_t row = blockIdx.x / (unsigned)chunks;
  const int64_t base = (int64_t)(blockIdx.x % (unsigned)chunks) * kChunk;
  const int tid = threadIdx.x;
  const RowStats st = stats[row];
  const bool live = st.live != 0.f;
  const float g = live ? grad[row * grad_stride] /
                             ((count ? *count : 1.f) * inv_t)
                       : 0.f;
  const typename E::type* src = x + row * stride;
  typename E::type* dst = dx + row * v;
  u32x4 w[U];
  if (live) {
#pragma unroll
    for (int i = 0; i < U; i++)
      w[i] = load_vec<T>(src, base + (int64_t)(i * kThreads + tid) * E::kVec,
                         v);
    const int64_t id = tid < k ? ids[row * k + tid] : -1;
    s_id[tid] = id >= 0 && id < v ? (int)id : -1;
    s_q[tid] = tid < k ? q[row * k + tid] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < U; i++) {
    const int64_t at = base + (int64_t)(i * kThreads + tid) * E::kVec;
    if (at >= v) continue;
    float d[E::kVec];
#pragma unroll
    for (int j = 0; j < E::kVec; j++)
      d[j] = live ? g * exp2_raw((E::get(w[i], j) - st.max) * c - st.log2_sum)
                  : 0.f;
    if (at + E::kVec <= v) {
      *(raw16*)(dst + at) = pack<T>(d);
    } else {
#pragma unroll
      for (int j = 0; j < E::kVec; j++)
        if (at + j < v) E::store(dst + at + j, d[j]);
    }
  }
  if (!live) return;
  __syncthreads();  // also orders the block's stores
  const int id = s_id[tid];
  if (id < 0 || id < base || id >= base + kChunk) return;
  // the first of equal ids writes; four a read, or the search would take as
  // long as the chunk
  float share = 0.f;
  bool first = true;
#pragma unroll 2
  for (int j = 0; j < k; j += 4) {
    const int4 a = *(const int4*)&s_id[j];
    const float4 b = *(const float4*)&s_q[j];
    share += a.x == id ? b.x : 0.f;
    share += a.y == id ? b.y : 0.f;
    share += a.z == id ? b.z : 0.f;
    share += a.w == id ? b.w : 0.f;
    first &= !((a.x == id & j < tid) | (a.y == id & j + 1 < tid) |
               (a.z == id & j + 2 < tid) | (a.w == id & j + 3 < tid));
  }
  if (!first) return;
  float p = exp2_raw((E::load(src + id) - st.max) * c - st.log2_sum);
  E::store(dst + id, g * (p - share));
}

// ---------------------------------------------------------------------------
// launching
// ---------------------------------------------------------------------------
// Parts of a row. Rows are split into parts of whole chunks until there are
// kWant blocks (kWantPlain without alternatives, which leave less to do
// between the loads). From kWhole rows on they are not, nor are short rows: a
// row by one block saves the launch that joins the parts, 2 us of it, 4 with
// alternatives. In us, of rows x row, split and whole:
//                     no alternatives    1            20            64
//    1 x  8000 f32     5.1,  3.8     9.2,  6.9   10.4,  9.6   11.9, 12.7
//    1 x 16000 f32     5.1,  4.7     9.5,  9.0   10.2, 13.3   12.5, 19.4
//  200 x 16000 f32     8.0,  5.7    15.4, 10.8   18.9, 15.2   25.0, 21.1
//  200 x 32000 bf16    9.4,  7.0    16.3, 13.2   20.5, 18.2   27.6, 24.8
//  256 x 131072 bf16  17.2, 16.9    25.0, 29.9   32.4, 41.7   46.4, 61.1
//  400 x 50001 bf16      -, 14.3       -, 22.1      -, 29.9      -, 42.2
// (of the last, split: 24.5, 32.3, 45.8 with alternatives)
constexpr int64_t kWant = 1024;
constexpr int64_t kWantPlain = 512;
constexpr int64_t kWhole = 384;
constexpr int64_t kSome = 128;  // rows from which twice as long ones are short
constexpr int64_t kMaxSplits = 64;

struct Plan {
  int unroll;        // words of 16 bytes a thread holds at a time
  int64_t splits, part_len;
};

int vec_of(LmType t) { return t == LmType::F32 ? 4 : 8; }

Plan plan_of(LmType t, int64_t rows, int64_t v, int top) {
  Plan p;
  int64_t word = (int64_t)kThreads * vec_of(t);
  const int64_t want = top ? kWant : kWantPlain;
  const bool alone =
      rows >= kWhole || v <= (top && rows < kSome ? 8 : 16) * word;
  p.unroll =
      v > word && (alone || rows * ((v + 4 * word - 1) / (4 * word)) >= want)
          ? 4
          : 1;
  int64_t chunk = word * p.unroll;
  int64_t chunks = (v + chunk - 1) / chunk;
  int64_t splits = std::min(std::min(chunks, kMaxSplits),
                            std::max<int64_t>(1, want / rows));
  if (alone) splits = 1;
  if (top) splits = std::min<int64_t>(splits, kMaxKeys / top);
  p.part_len = (chunks + splits - 1) / splits * chunk;
  p.splits = (v + p.part_len - 1) / p.part_len;
  return p;
}

template <class F>
void by_type(LmType t, F f) {
  switch (t) {
    case LmType::F32:
      f(std::integral_constant<LmType, LmType::F32>{});
      break;
    case LmType::BF16:
      f(std::integral_constant<LmType, LmType::BF16>{});
      break;
    case LmType::F16:
      f(std::integral_constant<LmType, LmType::F16>{});
      break;
  }
  HIP_CHECK(hipGetLastError());
}

template <class End>
void run_score(LmType t, const void* x, int64_t stride, int64_t rows,
               int64_t v, const Plan& p, float c, bool top, bool direct,
               const End& end, Part* parts, uint64_t* keys,
               hipStream_t stream) {
  const dim3 grid = lm_grid(rows * p.splits, kThreads);
  auto go = [&](auto type, auto unroll, auto with_top) {
    constexpr LmType T = decltype(type)::value;
    score_kernel<T, decltype(unroll)::value, decltype(with_top)::value, End>
        <<<grid, kThreads, 0, stream>>>(
            (const typename Elem<T>::type*)x, stride, v, (int)p.splits,
            p.part_len, c, direct, end, parts, keys);
  };
  auto by_top = [&](auto type, auto unroll) {
    if constexpr (std::is_same<End, LogprobsEnd>::value) {
      if (top) return go(type, unroll, std::true_type{});
    }
    go(type, unroll, std::false_type{});
  };
  auto by_unroll = [&](auto type) {
    if (p.unroll == 4)
      by_top(type, std::integral_constant<int, 4>{});
    else
      by_top(type, std::integral_constant<int, 1>{});
  };
  by_type(t, by_unroll);
}

}  // namespace

int64_t score_workspace(LmType t, int64_t rows, int64_t v, int top) {
  Plan p = plan_of(t, rows, v, top);
  if (p.splits == 1) return 0;  // one block makes a row
  return rows * p.splits * (int64_t)(sizeof(Part) + 8 * (int64_t)top);
}

void launch_token_logprobs(LmType t, const void* x, int64_t stride,
                           int64_t rows, int64_t v, const int64_t* tokens,
                           int64_t ignore, float inv_t, int top,
                           float* logprobs, float* entropy, float* top_lp,
                           int64_t* top_ids, RowStats* stats, void* ws,
                           hipStream_t stream) {
  Plan p = plan_of(t, rows, v, top);
  const float c = inv_t * kLog2e;
  Part* parts = (Part*)ws;
  uint64_t* keys = (uint64_t*)(parts + rows * p.splits);
  const LogprobsEnd e = {tokens,  ignore, inv_t,   top,  logprobs,
                         entropy, top_lp, top_ids, stats};
  const bool direct = p.splits == 1;
  run_score(t, x, stride, rows, v, p, c, top > 0, direct, e, parts, keys,
            stream);
  if (direct) return;
  by_type(t, [&](auto type) {
    constexpr LmType T = decltype(type)::value;
    auto* xt = (const typename Elem<T>::type*)x;
    if (top)
      top_rows_kernel<T><<<lm_grid(rows, kThreads), kThreads, 0, stream>>>(
          xt, stride, v, c, parts, keys, (int)p.splits, e);
    else
      logprobs_rows_kernel<T>
          <<<lm_grid((rows + kWaves - 1) / kWaves, kThreads), kThreads, 0,
             stream>>>(xt, stride, rows, v, c, parts, (int)p.splits, e);
  });
}

void launch_token_logprobs_bwd(LmType t, const void* x, int64_t stride,
                               int64_t rows, int64_t v,
                               const int64_t* tokens, float inv_t,
                               const RowStats* stats, const float* g_lp,
                               const float* g_h, void* dx,
                               hipStream_t stream) {
  by_type(t, [&](auto type) {
    constexpr LmType T = decltype(type)::value;
    constexpr int U = 4;
    constexpr int64_t chunk = (int64_t)kThreads * Elem<T>::kVec * U;
    int64_t chunks = (v + chunk - 1) / chunk;
    logprobs_bwd_kernel<T, U>
        <<<lm_grid(rows * chunks, kThreads), kThreads, 0, stream>>>(
            (const typename Elem<T>::type*)x, stride, v, (int)chunks, tokens,
            inv_t, inv_t * kLog2e, stats, g_lp, g_h,
            (typename Elem<T>::type*)dx);
  });
}

void launch_distill(LmType t, const void* x, int64_t stride, int64_t rows,
                    int64_t v, LmType tt, const void* teacher,
                    const int64_t* ids, int k, float inv_t, float* row_loss,
                    float* q, RowStats* stats, float* total, float* count,
                    bool mean, void* ws, hipStream_t stream) {
  Plan p = plan_of(t, rows, v, 0);
  const float c = inv_t * kLog2e;
  Part* parts = (Part*)ws;
  const DistillEnd e = {tt, teacher, ids, k, inv_t, row_loss, q, stats};
  const bool direct = p.splits == 1;
  const bool whole = !direct && total && rows <= kOneBlock;
  run_score(t, x, stride, rows, v, p, c, false, direct, e, parts, nullptr,
            stream);
  if (!direct)
    by_type(t, [&](auto type) {
      constexpr LmType T = decltype(type)::value;
      auto go = [&](auto w) {
        constexpr bool W = decltype(w)::value;
        distill_rows_kernel<T, W>
            <<<lm_grid(W ? 1 : (rows + kWaves - 1) / kWaves, kThreads),
               W ? kOneBlock * 64 : kThreads, 0, stream>>>(
                (const typename Elem<T>::type*)x, stride, rows, v, c, parts,
                (int)p.splits, e, mean, total, count);
      };
      whole ? go(std::true_type{}) : go(std::false_type{});
    });
  if (total && !whole) {
    distill_total_kernel<<<1, 1024, 0, stream>>>(row_loss, stats, rows, mean,
                                                 total, count);
    HIP_CHECK(hipGetLastError());
  }
}

void launch_distill_bwd(LmType t, const void* x, int64_t stride,
                        int64_t rows, int64_t v, const int64_t* ids,
                        const float* q, int k, float inv_t,
                        const RowStats* stats, const float* grad,
                        int64_t grad_stride, const float* count, void* dx,
                        hipStream_t stream) {
  by_type(t, [&](auto type) {
    constexpr LmType T = decltype(type)::value;
    constexpr int U = 4;
    constexpr int64_t chunk = (int64_t)kThreads * Elem<T>::kVec * U;
    int64_t chunks = (v + chunk - 1) / chunk;
    distill_bwd_kernel<T, U>
        <<<lm_grid(rows * chunks, kThreads), kThreads, 0, stream>>>(
            (const typename Elem<T>::type*)x, stride, v, (int)chunks, ids, q,
            k, inv_t, inv_t * kLog2e, stats, grad, grad_stride, count,
            (typename Elem<T>::type*)dx);
  });
}
