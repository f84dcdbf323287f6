// log_prob_common.cuh -- what the losses over rows of class scores share between
// the row kernels (one source file for each type of score) and the entries.
#pragma once

#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "b2_internal.cuh"

namespace b2 {

enum Mode { kLogProb = 0, kDistill = 1, kPolicy = 2 };

struct PolicyToken {
  float old_lp, advantage, ref_lp;
  bool has_ref;
};
struct PolicyClip {
  double low, high;  // the ratio's range
  double kl_coef;
};
struct RowArgs {
  const void* x;
  int64_t rows, inner, outer_stride, inner_stride;
  int classes;
  int slice;          // values of a row that each CTA of a cluster has, a multiple of 8
  int filter_words;   // of each of a teacher's two bit filters, a power of two
  int teacher_bytes;  // shared memory of a row's teacher
  float c;  // log2(e) / temperature
  float temperature;
  double inv_t;
  float2* stats;   // [rows] (m, s): written by pass 1 unless null, read by pass 2 alone
  void* grad;      // [rows, classes] dense; null: no pass 2
  // the chosen classes
  const void* ids;
  int ids_bytes, top;
  const void* teacher;
  int teacher_dtype;
  // what multiplies a row
  const void* weights;  // null: 1; float, or one byte a row (0 / not 0)
  int weight_bytes;
  const double* total;     // sum of the weights; null: rows
  const float* upstream;   // per row (log-probability gradient)
  const float* grad_loss;  // scalar; null: 1
  // policy
  const float *old_lp, *ref_lp, *advantages;
  PolicyClip clip;
  // results per row
  float* log_probs;
  double* row_out;  // [1 or 3][rows], multiplied by the row's weight
};

// The passes over the rows: pass 1 (statistics, and the loss of each row) when
// `stats`, pass 2 (the gradient) when `grad`.
int launch_rows_f32(cudaStream_t s, const RowArgs& a, Mode mode, bool stats, bool grad, const DeviceInfo* d,
                    const char* what);
int launch_rows_f16(cudaStream_t s, const RowArgs& a, Mode mode, bool stats, bool grad, const DeviceInfo* d,
                    const char* what);
int launch_rows_bf16(cudaStream_t s, const RowArgs& a, Mode mode, bool stats, bool grad, const DeviceInfo* d,
                     const char* what);

constexpr int kMaxTop = 1024;  // teacher entries of a row

__device__ __forceinline__ int64_t class_at(const void* ids, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(ids)[i] : (int64_t) static_cast<const int32_t*>(ids)[i];
}

__device__ __forceinline__ float weight_at(const void* w, int bytes, int64_t i) {
  if (w == nullptr) return 1.0f;
  return bytes == 4 ? static_cast<const float*>(w)[i] : (static_cast<const uint8_t*>(w)[i] != 0 ? 1.0f : 0.0f);
}

// One token of the clipped policy loss with a KL term, in 64 bits: advantages of both
// signs cancel in the mean, and a border or coefficient rounded to 32 bits would move
// all cut tokens' terms the same way; the ratio may pass 32 bits' range, and times an
// advantage of 0 is 0 all the same.  The log-probability lp is the fp32 number that
// b2_token_log_probs gives, in the loss from the scores too: where the old one is that
// number, the ratio is exactly 1.
struct PolicyKl {
  double kl, rise;  // exp(d) - d - 1 and exp(d) - 1
};
__device__ __forceinline__ PolicyKl policy_kl(float lp, const PolicyToken& t) {
  if (!t.has_ref) return PolicyKl{0.0, 0.0};
  const double d = (double)t.ref_lp - (double)lp;
  if (fabs(d) <= 1.0) {
    // kl's series, where the subtraction would cancel: the sum of d^(k - 2) / k!,
    // k = 2 .. 11, leaves out less than 1e-8 of it
    double s = 1.0 / 39916800.0;
    s = fma(s, d, 1.0 / 3628800.0);
    s = fma(s, d, 1.0 / 362880.0);
    s = fma(s, d, 1.0 / 40320.0);
    s = fma(s, d, 1.0 / 5040.0);
    s = fma(s, d, 1.0 / 720.0);
    s = fma(s, d, 1.0 / 120.0);
    s = fma(s, d, 1.0 / 24.0);
    s = fma(s, d, 1.0 / 6.0);
    s = fma(s, d, 0.5);
    const double kl = s * d * d;
    return PolicyKl{kl, d + kl};
  }
  const double e = exp(d);
  return PolicyKl{isinf(e) ? e : e - d - 1.0, e - 1.0};  // d itself may be infinite
}

struct PolicyTerm {
  double slope;  // in the token's log-probability
  double held;   // the ratio, or the border that it is held at
  bool cut;
};
// Where the KL term's coefficient is 0 it is only reported: an infinite one touches
// neither slope nor value.
__device__ __forceinline__ PolicyTerm policy_term(const PolicyToken& t, const PolicyClip& c, double ratio, double rise) {
  const bool above = ratio > c.high, below = ratio < c.low;
  PolicyTerm p;
  p.cut = (t.advantage > 0.0f && above) || (t.advantage < 0.0f && below);
  p.held = p.cut ? (above ? c.high : c.low) : ratio;
  p.slope = p.cut ? 0.0 : -ratio * (double)t.advantage;
  if (c.kl_coef != 0.0) p.slope -= c.kl_coef * rise;
  return p;
}
// Where the ratio is not cut, the unclipped term is the larger one.
__device__ __forceinline__ double policy_value(const PolicyTerm& p, const PolicyToken& t, const PolicyClip& c,
                                               double kl) {
  const double value = -p.held * (double)t.advantage;
  return c.kl_coef != 0.0 ? value + c.kl_coef * kl : value;
}

}  // namespace b2
