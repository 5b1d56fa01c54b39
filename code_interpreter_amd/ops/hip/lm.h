// Declarations of the language-model kernels (_hiplm): microscaled 4-bit
// quantisation and product, and scoring of rows of logits.
#pragma once

#include "common.h"

// types of activations and logits
enum class LmType : int { F32 = 0, BF16 = 1, F16 = 2 };

constexpr int kMxBlock = 32;   // elements that share a scale
constexpr int kMxBytes = 16;   // bytes of codes of a block

// a grid of one axis: its threads are counted in 32 bits
inline dim3 lm_grid(int64_t blocks, int threads) {
  if (blocks > (int64_t)0xFFFFFFFF / threads)
    throw std::runtime_error("too many rows for one launch");
  return dim3((unsigned)blocks);
}

inline int64_t mx_blocks(int64_t k) { return (k + kMxBlock - 1) / kMxBlock; }

// x: [rows][k], row stride in elements. codes: [rows][blocks][16],
// scales: [rows][blocks]
void launch_mx_quantize(LmType t, const void* x, int64_t stride,
                        uint8_t* codes, uint8_t* scales, int64_t rows,
                        int64_t k, hipStream_t stream);
void launch_mx_dequantize(LmType t, const uint8_t* codes,
                          const uint8_t* scales, void* out, int64_t rows,
                          int64_t k, hipStream_t stream);

// y[m][n] = sum over k of x[m][k] w[n][k] + bias[n]; x in 16 or 32 bits is
// quantised on the way in (into `ws` where the chosen kernel wants it
// there), or comes as codes and scales (x null)
int64_t mx_linear_workspace(int64_t m, int64_t n, int64_t k, bool packed);
void launch_mx_linear(LmType t, const void* x, int64_t stride,
                      const uint8_t* xcodes, const uint8_t* xscales,
                      const uint8_t* wcodes, const uint8_t* wscales,
                      const void* bias, void* y, int64_t m, int64_t n,
                      int64_t k, void* ws, hipStream_t stream);

// ---- rows of logits -------------------------------------------------------
constexpr int kMaxTop = 128;      // alternatives of a row
constexpr int kMaxRecord = 256;   // recorded teacher entries of a row

// bytes of scratch of one forward call
int64_t score_workspace(LmType t, int64_t rows, int64_t v, int top);

// what a row leaves for its backward: its largest logit, log2 of the sum of
// 2^(c (x - max)), its entropy, and 1 where its gradient is not zero as a
// whole
struct RowStats {
  float max, log2_sum, entropy, live;
};

void launch_token_logprobs(LmType t, const void* x, int64_t stride,
                           int64_t rows, int64_t v, const int64_t* tokens,
                           int64_t ignore, float inv_t, int top,
                           float* logprobs, float* entropy, float* top_lp,
                           int64_t* top_ids, RowStats* stats, void* ws,
                           hipStream_t stream);
void launch_token_logprobs_bwd(LmType t, const void* x, int64_t stride,
                               int64_t rows, int64_t v,
                               const int64_t* tokens, float inv_t,
                               const RowStats* stats, const float* g_lp,
                               const float* g_h, void* dx,
                               hipStream_t stream);

// teacher: [rows][k] recorded logits and ids, an id of -1 or a logit of
// -inf where a row has fewer. row_loss [rows], q [rows][k]. total (may be
// null): the sum, or the mean over rows with a record; count: what the sum
// was divided by
void launch_distill(LmType t, const void* x, int64_t stride, int64_t rows,
                    int64_t v, LmType tt, const void* teacher,
                    const int64_t* ids, int k, float inv_t, float* row_loss,
                    float* q, RowStats* stats, float* total, float* count,
                    bool mean, void* ws, hipStream_t stream);
void launch_distill_bwd(LmType t, const void* x, int64_t stride,
                        int64_t rows, int64_t v, const int64_t* ids,
                        const float* q, int k, float inv_t,
                        const RowStats* stats, const float* grad,
                        int64_t grad_stride, const float* count, void* dx,
                        hipStream_t stream);
