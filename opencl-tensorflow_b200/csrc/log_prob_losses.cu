// log_prob_losses.cu -- losses over the log-softmax of rows of class scores:
// the log-probability of a chosen class, distillation from a teacher's top
// logits, the preference loss over pairs of sequences and the clipped policy
// loss with a KL term; each forward and backward.  The passes over the scores are
// in log_prob_rows.cuh; here are the sums over rows and tokens and the entries.
#include <cooperative_groups.h>

#include <cmath>

#include "log_prob_common.cuh"

namespace cg = cooperative_groups;

namespace b2 {
namespace {

template <class F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---------------------------------------------------------- sums over rows

constexpr int kSumCtas = 8;  // one portable cluster
constexpr int kSumThreads = 512;

// Adds up to four doubles per thread over the cluster, in a fixed order; the
// sums are valid in thread 0 of CTA 0.
template <int kN>
__device__ __forceinline__ void cluster_sum(double* v) {
  __shared__ double warp_part[kN][kSumThreads / 32];
  __shared__ double cta_part[kN];
  cg::cluster_group cluster = cg::this_cluster();
#pragma unroll
  for (int k = 0; k < kN; ++k) {
    v[k] = warp_sum(v[k]);
    if ((threadIdx.x & 31) == 0) warp_part[k][threadIdx.x >> 5] = v[k];
  }
  __syncthreads();
  if (threadIdx.x < kN) {
    double c = 0.0;
    for (int i = 0; i < kSumThreads / 32; ++i) c += warp_part[threadIdx.x][i];
    cta_part[threadIdx.x] = c;
  }
  cluster.sync();
  if (cluster.block_rank() == 0 && threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      v[k] = 0.0;
      for (int i = 0; i < kSumCtas; ++i) v[k] += *cluster.map_shared_rank(&cta_part[k], i);
    }
  }
  cluster.sync();
}

// *total = sum of the weights.
__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    weight_sum_kernel(const void* __restrict__ weights, int bytes, int64_t rows, double* __restrict__ total) {
  double v[1] = {0.0};
  for (int64_t i = (int64_t)blockIdx.x * kSumThreads + threadIdx.x; i < rows; i += kSumCtas * kSumThreads)
    v[0] += (double)weight_at(weights, bytes, i);
  cluster_sum<1>(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) *total = v[0];
}

// *loss and stats[k - 1] = sum_r values[k][r] / total, 0 when the total is 0.  The total is
// *total_in, or the sum of the weights (rows without any); total_out: null, or where it goes.
template <int kN>
__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    mean_kernel(const double* __restrict__ values, const void* __restrict__ weights, int weight_bytes,
                const double* __restrict__ total_in, double* __restrict__ total_out, int64_t rows,
                float* __restrict__ loss, float* __restrict__ stats) {
  const bool add = total_in == nullptr && weights != nullptr;
  double v[kN + 1] = {};
  for (int64_t i = (int64_t)blockIdx.x * kSumThreads + threadIdx.x; i < rows; i += kSumCtas * kSumThreads) {
#pragma unroll
    for (int k = 0; k < kN; ++k) v[k] += values[k * rows + i];
    if (add) v[kN] += (double)weight_at(weights, weight_bytes, i);
  }
  cluster_sum<kN + 1>(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const double t = total_in != nullptr ? *total_in : add ? v[kN] : (double)rows;
#pragma unroll
    for (int k = 0; k < kN; ++k) (k == 0 ? loss : stats + k - 1)[0] = t != 0.0 ? (float)(v[k] / t) : 0.0f;
    if (total_out != nullptr) *total_out = t;
  }
}

// ------------------------------------------------------------- preferences

constexpr int kTokenThreads = 256;

__device__ __forceinline__ int64_t offset_at(const void* o, int bytes, int64_t i, int64_t tokens) {
  const int64_t v = class_at(o, bytes, i);
  return v < 0 ? 0 : v > tokens ? tokens : v;  // never outside the tokens, whatever the caller's offsets hold
}

struct PreferenceArgs {
  const float *lp, *ref;
  const void* mask;
  int mask_bytes;
  int64_t tokens;
  const void* offsets;
  int offset_bytes;
  int64_t pairs;
  double beta, smoothing;
};

// The sum of a sequence's w (lp - ref) by `threads` threads, t among them.
__device__ __forceinline__ double sequence_part(const PreferenceArgs& A, int64_t i, int t, int threads) {
  const int64_t a = offset_at(A.offsets, A.offset_bytes, i, A.tokens);
  const int64_t b = offset_at(A.offsets, A.offset_bytes, i + 1, A.tokens);
  double v = 0.0;
  for (int64_t n = a + t; n < b; n += threads) {
    const float w = weight_at(A.mask, A.mask_bytes, n);
    if (w != 0.0f) v += (double)w * ((double)A.lp[n] - (A.ref != nullptr ? (double)A.ref[n] : 0.0));
  }
  return v;
}

// One CTA per sequence: rewards[i] = beta sum_n w_n (lp_n - ref_n).
__global__ void __launch_bounds__(kTokenThreads)
    sequence_sum_kernel(const PreferenceArgs A, double* __restrict__ sums) {
  __shared__ double part[kTokenThreads / 32];
  const int64_t i = blockIdx.x;
  const double v = warp_sum(sequence_part(A, i, threadIdx.x, kTokenThreads));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    double c = 0.0;
    for (int k = 0; k < kTokenThreads / 32; ++k) c += part[k];
    sums[i] = A.beta * c;
  }
}

__device__ __forceinline__ double softplus(double z) { return fmax(z, 0.0) + log1p(exp(-fabs(z))); }

// One pair's loss; its rewards and its sequences' slopes are written.
__device__ __forceinline__ double pair_loss(const PreferenceArgs& A, int64_t p, double chosen, double rejected,
                                            float* __restrict__ rewards, float* __restrict__ slopes) {
  const double eps = A.smoothing, h = chosen - rejected;
  // sigma(h) and sigma(-h), each without cancellation
  const double z = exp(-fabs(h)), small = z / (1.0 + z), large = 1.0 / (1.0 + z);
  const double up = h >= 0.0 ? large : small, down = h >= 0.0 ? small : large;
  const double slope = (eps * up - (1.0 - eps) * down) * A.beta / (double)A.pairs;
  rewards[p] = (float)chosen;
  rewards[A.pairs + p] = (float)rejected;
  slopes[p] = (float)slope;
  slopes[A.pairs + p] = (float)-slope;
  // without smoothing -log sigma(-h), infinite where the rejected answer is impossible, has no part
  return (1.0 - eps) * softplus(-h) + (eps != 0.0 ? eps * softplus(h) : 0.0);
}

__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    pair_kernel(const PreferenceArgs A, const double* __restrict__ sums, float* __restrict__ loss,
                float* __restrict__ rewards, float* __restrict__ slopes) {
  double v[1] = {0.0};
  for (int64_t p = (int64_t)blockIdx.x * kSumThreads + threadIdx.x; p < A.pairs; p += kSumCtas * kSumThreads)
    v[0] += pair_loss(A, p, sums[p], sums[A.pairs + p], rewards, slopes);
  cluster_sum<1>(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) *loss = (float)(v[0] / (double)A.pairs);
}

// A few pairs of short sequences in one launch: each CTA of the cluster takes
// pairs in turn, half of its warps a sequence.
constexpr int kFewPairs = 4 * kSumCtas;
constexpr int kFewTokens = 32768;

__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    few_pairs_kernel(const PreferenceArgs A, float* __restrict__ loss, float* __restrict__ rewards,
                     float* __restrict__ slopes) {
  constexpr int kHalf = kSumThreads / 2, kWarps = kSumThreads / 32;
  __shared__ double part[2][kWarps];
  double v[1] = {0.0};
  int turn = 0;
  for (int64_t p = blockIdx.x; p < A.pairs; p += kSumCtas, turn ^= 1) {
    const int half = threadIdx.x / kHalf;
    const double sum = warp_sum(sequence_part(A, p + half * A.pairs, threadIdx.x % kHalf, kHalf));
    if ((threadIdx.x & 31) == 0) part[turn][threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      double chosen = 0.0, rejected = 0.0;
      for (int k = 0; k < kWarps / 2; ++k) chosen += part[turn][k], rejected += part[turn][kWarps / 2 + k];
      v[0] += pair_loss(A, p, A.beta * chosen, A.beta * rejected, rewards, slopes);
    }
  }
  cluster_sum<1>(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) *loss = (float)(v[0] / (double)A.pairs);
}

// grad[n] = grad_loss * slope of n's sequence * w_n; 0 outside the sequences.
// A token belongs to the last sequence that starts at or before it.
__global__ void __launch_bounds__(kTokenThreads)
    preference_grad_kernel(const PreferenceArgs A, const float* __restrict__ grad_loss,
                           const float* __restrict__ slopes, float* __restrict__ grad) {
  const float gl = *grad_loss;
  for (int64_t n = (int64_t)blockIdx.x * kTokenThreads + threadIdx.x; n < A.tokens;
       n += (int64_t)gridDim.x * kTokenThreads) {
    int64_t lo = 0, hi = 2 * A.pairs + 1;  // first offset > n
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (class_at(A.offsets, A.offset_bytes, mid) > n)
        hi = mid;
      else
        lo = mid + 1;
    }
    const int64_t seq = lo - 1;
    const float w = weight_at(A.mask, A.mask_bytes, n);
    const bool inside = seq >= 0 && seq < 2 * A.pairs && w != 0.0f;
    grad[n] = inside ? gl * slopes[seq] * w : 0.0f;
  }
}

// ------------------------------------------------------------------- policy

struct PolicyArgs {
  const float *lp, *old_lp, *ref_lp, *advantages;
  const void* mask;
  int mask_bytes;
  int64_t tokens;
  PolicyClip clip;
};

constexpr int kPolicySums = 4;  // loss, kl, clipped, weights

// What thread `first` of every `step` adds up (loss, kl, clipped, weights); the
// tokens' slopes are written, rounded once.  The ratio in 64 bits costs 0.7 us, at 64
// tokens and at a million, the KL term nothing beside it (14.4 us, two launches); there
// a mean of terms that cancel to 1e-3 was 7e-7 off with ratios in 32.  Loads that do not
// wait for the token's weight, and four tokens a turn, are no faster at a million.
__device__ __forceinline__ void policy_part(const PolicyArgs& A, int64_t first, int64_t step,
                                            float* __restrict__ slopes, double* v) {
  const bool has_ref = A.ref_lp != nullptr;
  for (int64_t n = first; n < A.tokens; n += step) {
    const float w = weight_at(A.mask, A.mask_bytes, n);
    float slope = 0.0f;
    if (w != 0.0f) {
      const PolicyToken token{A.old_lp[n], A.advantages[n], has_ref ? A.ref_lp[n] : 0.0f, has_ref};
      const float lp = A.lp[n];
      const PolicyKl k = policy_kl(lp, token);
      const PolicyTerm t = policy_term(token, A.clip, exp((double)lp - (double)token.old_lp), k.rise);
      v[0] += (double)w * policy_value(t, token, A.clip, k.kl);
      v[1] += (double)w * k.kl;
      slope = (float)((double)w * t.slope);
      v[2] += t.cut ? (double)w : 0.0;
      v[3] += (double)w;
    }
    if (slopes != nullptr) slopes[n] = slope;
  }
}

// *loss, stats = {mean KL, clipped share, 1 / sum of the weights}, all 0 when the weights sum to 0.
__device__ __forceinline__ void store_means(const double* v, float* __restrict__ loss, float* __restrict__ stats) {
  const double inv = v[3] != 0.0 ? 1.0 / v[3] : 0.0;
  *loss = v[3] != 0.0 ? (float)(v[0] / v[3]) : 0.0f;
  stats[0] = v[3] != 0.0 ? (float)(v[1] / v[3]) : 0.0f;
  stats[1] = v[3] != 0.0 ? (float)(v[2] / v[3]) : 0.0f;
  stats[2] = (float)inv;
}

// Few tokens in one launch, by one cluster.
constexpr int kFewPolicyTokens = 8 * kSumCtas * kSumThreads;

__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    few_policy_kernel(const PolicyArgs A, float* __restrict__ slopes, float* __restrict__ loss,
                      float* __restrict__ stats) {
  double v[kPolicySums] = {};
  policy_part(A, (int64_t)blockIdx.x * kSumThreads + threadIdx.x, kSumCtas * kSumThreads, slopes, v);
  cluster_sum<kPolicySums>(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) store_means(v, loss, stats);
}

__global__ void __launch_bounds__(kTokenThreads)
    policy_kernel(const PolicyArgs A, float* __restrict__ slopes, double* __restrict__ partial) {
  __shared__ double part[kPolicySums][kTokenThreads / 32];
  double v[kPolicySums] = {};
  policy_part(A, (int64_t)blockIdx.x * kTokenThreads + threadIdx.x, (int64_t)gridDim.x * kTokenThreads, slopes, v);
#pragma unroll
  for (int k = 0; k < kPolicySums; ++k) {
    v[k] = warp_sum(v[k]);
    if ((threadIdx.x & 31) == 0) part[k][threadIdx.x >> 5] = v[k];
  }
  __syncthreads();
  if (threadIdx.x < kPolicySums) {
    double c = 0.0;
    for (int i = 0; i < kTokenThreads / 32; ++i) c += part[threadIdx.x][i];
    partial[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = c;
  }
}

__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    policy_mean_kernel(const double* __restrict__ partial, int64_t parts, float* __restrict__ loss,
                       float* __restrict__ stats) {
  double v[kPolicySums] = {};
  for (int64_t i = (int64_t)blockIdx.x * kSumThreads + threadIdx.x; i < parts; i += kSumCtas * kSumThreads)
#pragma unroll
    for (int k = 0; k < kPolicySums; ++k) v[k] += partial[k * parts + i];
  cluster_sum<kPolicySums>(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) store_means(v, loss, stats);
}

__global__ void __launch_bounds__(kTokenThreads)
    policy_grad_kernel(const float* __restrict__ grad_loss, const float* __restrict__ inv_total,
                       const float* __restrict__ slopes, int64_t tokens, float* __restrict__ grad) {
  // In 32 bits: slope, 1 / sum, their factor and the product each add half a step at most.
  // In 64 they would be one less where grad_loss is no power of two; a million tokens,
  // forward and backward, take 20.5 us then and not 18.5.
  const float f = *grad_loss * *inv_total;
  for (int64_t n = (int64_t)blockIdx.x * kTokenThreads + threadIdx.x; n < tokens;
       n += (int64_t)gridDim.x * kTokenThreads)
    grad[n] = slopes[n] == 0.0f ? 0.0f : f * slopes[n];
}

// ----------------------------------------------------------------- entries

int launch_rows(cudaStream_t s, const RowArgs& a, int dtype, Mode mode, bool stats, bool grad, const DeviceInfo* d,
                const char* what) {
  if (dtype == B2_FLOAT32) return launch_rows_f32(s, a, mode, stats, grad, d, what);
  if (dtype == B2_FLOAT16) return launch_rows_f16(s, a, mode, stats, grad, d, what);
  return launch_rows_bf16(s, a, mode, stats, grad, d, what);
}

// Checks a row view and starts the kernel's arguments with it.
int row_args(const b2_logits_t* x, const char* what, RowArgs* a) {
  B2_REQUIRE(x != nullptr, "%s: null logits", what);
  B2_REQUIRE(x->dtype == B2_FLOAT32 || x->dtype == B2_FLOAT16 || x->dtype == B2_BFLOAT16,
             "%s: logits must be float32, float16 or bfloat16", what);
  B2_REQUIRE(x->outer >= 0 && x->inner >= 0, "%s: negative number of rows", what);
  B2_REQUIRE(x->classes >= 1 && x->classes <= (1 << 30), "%s: classes must be in [1, 2^30], got %lld", what,
             (long long)x->classes);
  B2_REQUIRE(x->inner == 0 || x->outer <= kMaxInt32 / x->inner, "%s: too many rows", what);
  B2_REQUIRE(x->outer * x->inner == 0 || x->data != nullptr, "%s: null logits", what);
  *a = RowArgs{};
  a->x = x->data;
  a->rows = x->outer * x->inner;
  a->inner = x->inner > 0 ? x->inner : 1;
  a->outer_stride = x->outer_stride;
  a->inner_stride = x->inner_stride;
  a->classes = (int)x->classes;
  a->temperature = 1.0f;
  a->inv_t = 1.0;
  a->c = (float)M_LOG2E;
  return B2_OK;
}

int index_ok(int bytes, const char* what, const char* name) {
  B2_REQUIRE(bytes == 4 || bytes == 8, "%s: %s must be 32- or 64-bit integers", what, name);
  return B2_OK;
}

int weight_ok(const void* w, int bytes, const char* what) {
  B2_REQUIRE(w == nullptr || bytes == 1 || bytes == 4, "%s: weights must be float32, or one byte each", what);
  return B2_OK;
}

// Statistics are read and written as pairs of floats, and the sum behind them in 64 bits.
int stats_ok(const float* row_stats, const char* what) {
  B2_REQUIRE((reinterpret_cast<uintptr_t>(row_stats) & 7) == 0, "%s: row_stats must be 8-byte aligned", what);
  return B2_OK;
}

int sum_weights(cudaStream_t s, const void* w, int bytes, int64_t rows, double* total, const char* what) {
  weight_sum_kernel<<<kSumCtas, kSumThreads, 0, s>>>(w, bytes, rows, total);
  return check_launch(s, what);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_token_log_probs(b2_stream_t stream, const b2_logits_t* logits, const void* targets, int target_bytes,
                       float* log_probs, float* row_stats) {
  clear_error();
  RowArgs a;
  B2_RETURN_IF_ERROR(row_args(logits, "token_log_probs", &a));
  B2_RETURN_IF_ERROR(index_ok(target_bytes, "token_log_probs", "targets"));
  B2_RETURN_IF_ERROR(stats_ok(row_stats, "token_log_probs"));
  if (a.rows == 0) return B2_OK;
  B2_REQUIRE(targets != nullptr && log_probs != nullptr, "token_log_probs: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  a.ids = targets;
  a.ids_bytes = target_bytes;
  a.log_probs = log_probs;
  a.stats = reinterpret_cast<float2*>(row_stats);
  return launch_rows(static_cast<cudaStream_t>(stream), a, logits->dtype, kLogProb, true, false, d, "token_log_probs");
}

int b2_token_log_probs_grad(b2_stream_t stream, const b2_logits_t* logits, const void* targets, int target_bytes,
                            const float* row_stats, const float* grad_log_probs, void* grad_logits) {
  clear_error();
  RowArgs a;
  B2_RETURN_IF_ERROR(row_args(logits, "token_log_probs_grad", &a));
  B2_RETURN_IF_ERROR(index_ok(target_bytes, "token_log_probs_grad", "targets"));
  B2_RETURN_IF_ERROR(stats_ok(row_stats, "token_log_probs_grad"));
  if (a.rows == 0) return B2_OK;
  B2_REQUIRE(targets != nullptr && row_stats != nullptr && grad_log_probs != nullptr && grad_logits != nullptr,
             "token_log_probs_grad: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  a.ids = targets;
  a.ids_bytes = target_bytes;
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(row_stats));
  a.upstream = grad_log_probs;
  a.grad = grad_logits;
  return launch_rows(static_cast<cudaStream_t>(stream), a, logits->dtype, kLogProb, false, true, d,
                     "token_log_probs_grad");
}

static int distill_args(const b2_logits_t* logits, const void* teacher_ids, int id_bytes, const void* teacher_logits,
                        int teacher_dtype, int64_t top, const void* weights, int weight_bytes, double temperature,
                        const char* what, RowArgs* a) {
  B2_RETURN_IF_ERROR(row_args(logits, what, a));
  B2_RETURN_IF_ERROR(index_ok(id_bytes, what, "teacher_ids"));
  B2_RETURN_IF_ERROR(weight_ok(weights, weight_bytes, what));
  B2_REQUIRE(a->rows > 0, "%s: the mean over no rows is undefined", what);
  B2_REQUIRE(top >= 1 && top <= kMaxTop, "%s: the teacher's entries per row must be in [1, %d], got %lld", what,
             kMaxTop, (long long)top);
  B2_REQUIRE(teacher_dtype == B2_FLOAT32 || teacher_dtype == B2_FLOAT16 || teacher_dtype == B2_BFLOAT16,
             "%s: teacher_logits must be float32, float16 or bfloat16", what);
  B2_REQUIRE(temperature >= 1e-30 && temperature <= 1e30, "%s: temperature must be in [1e-30, 1e30]", what);
  B2_REQUIRE(teacher_ids != nullptr && teacher_logits != nullptr, "%s: null pointer", what);
  a->ids = teacher_ids;
  a->ids_bytes = id_bytes;
  a->teacher = teacher_logits;
  a->teacher_dtype = teacher_dtype;
  a->top = (int)top;
  a->weights = weights;
  a->weight_bytes = weight_bytes;
  a->temperature = (float)temperature;
  a->inv_t = 1.0 / temperature;
  a->c = (float)(M_LOG2E / temperature);
  return B2_OK;
}

int b2_distillation_loss(b2_stream_t stream, const b2_logits_t* logits, const void* teacher_ids, int id_bytes,
                         const void* teacher_logits, int teacher_dtype, int64_t top, const void* weights,
                         int weight_bytes, double temperature, float* loss, float* row_stats,
                         const float* grad_loss, void* grad_logits) {
  clear_error();
  RowArgs a;
  B2_RETURN_IF_ERROR(distill_args(logits, teacher_ids, id_bytes, teacher_logits, teacher_dtype, top, weights,
                                  weight_bytes, temperature, "distillation_loss", &a));
  B2_REQUIRE(loss != nullptr, "distillation_loss: null pointer");
  B2_RETURN_IF_ERROR(stats_ok(row_stats, "distillation_loss"));
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // row_stats: statistics [rows][2], the sum of the weights (64 bits), the rows' losses (64 bits)
  Scratch scratch;
  double* total = reinterpret_cast<double*>(row_stats + 2 * a.rows);
  if (row_stats == nullptr) {
    B2_RETURN_IF_ERROR(scratch.alloc((a.rows + 1) * sizeof(double), s));
    total = scratch.as<double>();
  }
  a.row_out = total + 1;
  const bool early = grad_logits != nullptr && weights != nullptr;  // the gradient divides by the sum
  if (early) B2_RETURN_IF_ERROR(sum_weights(s, weights, weight_bytes, a.rows, total, "distillation_loss"));
  a.total = early ? total : nullptr;
  a.stats = reinterpret_cast<float2*>(row_stats);
  a.grad_loss = grad_loss;
  a.grad = grad_logits;
  B2_RETURN_IF_ERROR(
      launch_rows(s, a, logits->dtype, kDistill, true, grad_logits != nullptr, d, "distillation_loss"));
  mean_kernel<1><<<kSumCtas, kSumThreads, 0, s>>>(a.row_out, weights, weight_bytes, a.total, total, a.rows, loss,
                                                  nullptr);
  return check_launch(s, "distillation_loss");
}

int b2_distillation_loss_grad(b2_stream_t stream, const b2_logits_t* logits, const void* teacher_ids, int id_bytes,
                              const void* teacher_logits, int teacher_dtype, int64_t top, const void* weights,
                              int weight_bytes, double temperature, const float* row_stats, const float* grad_loss,
                              void* grad_logits) {
  clear_error();
  RowArgs a;
  B2_RETURN_IF_ERROR(distill_args(logits, teacher_ids, id_bytes, teacher_logits, teacher_dtype, top, weights,
                                  weight_bytes, temperature, "distillation_loss_grad", &a));
  B2_REQUIRE(row_stats != nullptr && grad_loss != nullptr && grad_logits != nullptr,
             "distillation_loss_grad: null pointer");
  B2_RETURN_IF_ERROR(stats_ok(row_stats, "distillation_loss_grad"));
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  a.total = reinterpret_cast<const double*>(row_stats + 2 * a.rows);
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(row_stats));
  a.grad_loss = grad_loss;
  a.grad = grad_logits;
  return launch_rows(s, a, logits->dtype, kDistill, false, true, d, "distillation_loss_grad");
}

int b2_preference_loss(b2_stream_t stream, const float* log_probs, const float* ref_log_probs, const void* mask,
                       int mask_bytes, int64_t tokens, const void* offsets, int offset_bytes, int64_t pairs,
                       double beta, double label_smoothing, float* loss, float* rewards, float* slopes) {
  clear_error();
  const char* what = "preference_loss";
  B2_RETURN_IF_ERROR(index_ok(offset_bytes, what, "offsets"));
  B2_RETURN_IF_ERROR(weight_ok(mask, mask_bytes, what));
  B2_REQUIRE(tokens >= 0, "preference_loss: negative number of tokens");
  B2_REQUIRE(pairs >= 1 && pairs <= kMaxInt32 / 2, "preference_loss: the mean over no pairs is undefined");
  B2_REQUIRE(std::isfinite(beta), "preference_loss: beta must be finite");
  B2_REQUIRE(label_smoothing >= 0.0 && label_smoothing <= 0.5, "preference_loss: label_smoothing must be in [0, 0.5]");
  B2_REQUIRE((tokens == 0 || log_probs != nullptr) && offsets != nullptr && loss != nullptr && rewards != nullptr &&
                 slopes != nullptr,
             "preference_loss: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const PreferenceArgs a{log_probs, ref_log_probs, mask, mask_bytes, tokens, offsets, offset_bytes, pairs, beta,
                         label_smoothing};
  if (pairs <= kFewPairs && tokens <= kFewTokens) {
    few_pairs_kernel<<<kSumCtas, kSumThreads, 0, s>>>(a, loss, rewards, slopes);
    return check_launch(s, what);
  }
  Scratch scratch;
  B2_RETURN_IF_ERROR(scratch.alloc(2 * pairs * sizeof(double), s));
  sequence_sum_kernel<<<(unsigned)(2 * pairs), kTokenThreads, 0, s>>>(a, scratch.as<double>());
  B2_RETURN_IF_ERROR(check_launch(s, what));
  pair_kernel<<<kSumCtas, kSumThreads, 0, s>>>(a, scratch.as<double>(), loss, rewards, slopes);
  return check_launch(s, what);
}

int b2_preference_loss_grad(b2_stream_t stream, const float* grad_loss, const float* slopes, const void* mask,
                            int mask_bytes, int64_t tokens, const void* offsets, int offset_bytes, int64_t pairs,
                            float* grad_log_probs) {
  clear_error();
  const char* what = "preference_loss_grad";
  B2_RETURN_IF_ERROR(index_ok(offset_bytes, what, "offsets"));
  B2_RETURN_IF_ERROR(weight_ok(mask, mask_bytes, what));
  B2_REQUIRE(tokens >= 0 && pairs >= 1 && pairs <= kMaxInt32 / 2, "preference_loss_grad: bad sizes");
  if (tokens == 0) return B2_OK;
  B2_REQUIRE(grad_loss != nullptr && slopes != nullptr && offsets != nullptr && grad_log_probs != nullptr,
             "preference_loss_grad: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const PreferenceArgs a{nullptr, nullptr, mask, mask_bytes, tokens, offsets, offset_bytes, pairs, 0.0, 0.0};
  preference_grad_kernel<<<grid_for(tokens, kTokenThreads, 8), kTokenThreads, 0, s>>>(a, grad_loss, slopes,
                                                                                      grad_log_probs);
  return check_launch(s, what);
}

static int policy_ok(int64_t tokens, const void* mask, int mask_bytes, double clip_low, double clip_high,
                     double kl_coef, const char* what) {
  B2_RETURN_IF_ERROR(weight_ok(mask, mask_bytes, what));
  B2_REQUIRE(tokens > 0, "%s: the mean over no tokens is undefined", what);
  B2_REQUIRE(clip_low >= 0.0 && clip_high >= 0.0, "%s: the clip range must not be negative", what);
  B2_REQUIRE(std::isfinite(kl_coef), "%s: kl_coef must be finite", what);
  return B2_OK;
}

int b2_policy_loss(b2_stream_t stream, const float* log_probs, const float* old_log_probs, const float* advantages,
                   const float* ref_log_probs, const void* mask, int mask_bytes, int64_t tokens, double clip_low,
                   double clip_high, double kl_coef, float* loss, float* stats, float* slopes) {
  clear_error();
  const char* what = "policy_loss";
  B2_RETURN_IF_ERROR(policy_ok(tokens, mask, mask_bytes, clip_low, clip_high, kl_coef, what));
  B2_REQUIRE(log_probs != nullptr && old_log_probs != nullptr && advantages != nullptr && loss != nullptr &&
                 stats != nullptr,
             "policy_loss: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const PolicyArgs a{log_probs, old_log_probs, ref_log_probs, advantages, mask, mask_bytes, tokens,
                     PolicyClip{1.0 - clip_low, 1.0 + clip_high, kl_coef}};
  if (tokens <= kFewPolicyTokens) {
    few_policy_kernel<<<kSumCtas, kSumThreads, 0, s>>>(a, slopes, loss, stats);
    return check_launch(s, what);
  }
  const int grid = grid_for(tokens, kTokenThreads, 4);
  Scratch scratch;
  B2_RETURN_IF_ERROR(scratch.alloc((size_t)grid * kPolicySums * sizeof(double), s));
  policy_kernel<<<grid, kTokenThreads, 0, s>>>(a, slopes, scratch.as<double>());
  B2_RETURN_IF_ERROR(check_launch(s, what));
  policy_mean_kernel<<<kSumCtas, kSumThreads, 0, s>>>(scratch.as<double>(), grid, loss, stats);
  return check_launch(s, what);
}

int b2_policy_loss_grad(b2_stream_t stream, const float* grad_loss, const float* stats, const float* slopes,
                        int64_t tokens, float* grad_log_probs) {
  clear_error();
  B2_REQUIRE(tokens > 0, "policy_loss_grad: no tokens");
  B2_REQUIRE(grad_loss != nullptr && stats != nullptr && slopes != nullptr && grad_log_probs != nullptr,
             "policy_loss_grad: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  policy_grad_kernel<<<grid_for(tokens, kTokenThreads, 8), kTokenThreads, 0, s>>>(grad_loss, stats + 2, slopes,
                                                                                  tokens, grad_log_probs);
  return check_launch(s, "policy_loss_grad");
}

int b2_policy_loss_with_grad(b2_stream_t stream, const b2_logits_t* logits, const void* targets, int target_bytes,
                             const float* old_log_probs, const float* advantages, const float* ref_log_probs,
                             const void* mask, int mask_bytes, double clip_low, double clip_high, double kl_coef,
                             const float* grad_loss, float* loss, float* stats, void* grad_logits) {
  clear_error();
  const char* what = "policy_loss_with_grad";
  RowArgs a;
  B2_RETURN_IF_ERROR(row_args(logits, what, &a));
  B2_RETURN_IF_ERROR(index_ok(target_bytes, what, "targets"));
  B2_RETURN_IF_ERROR(policy_ok(a.rows, mask, mask_bytes, clip_low, clip_high, kl_coef, what));
  B2_REQUIRE(targets != nullptr && old_log_probs != nullptr && advantages != nullptr && loss != nullptr &&
                 stats != nullptr && grad_logits != nullptr,
             "policy_loss_with_grad: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Scratch scratch;
  B2_RETURN_IF_ERROR(scratch.alloc((3 * a.rows + 1) * sizeof(double), s));
  double* total = mask != nullptr ? scratch.as<double>() + 3 * a.rows : nullptr;
  if (total != nullptr) B2_RETURN_IF_ERROR(sum_weights(s, mask, mask_bytes, a.rows, total, what));
  a.ids = targets;
  a.ids_bytes = target_bytes;
  a.weights = mask;
  a.weight_bytes = mask_bytes;
  a.total = total;
  a.old_lp = old_log_probs;
  a.ref_lp = ref_log_probs;
  a.advantages = advantages;
  a.clip = PolicyClip{1.0 - clip_low, 1.0 + clip_high, kl_coef};
  a.grad_loss = grad_loss;
  a.row_out = scratch.as<double>();
  a.grad = grad_logits;
  B2_RETURN_IF_ERROR(launch_rows(s, a, logits->dtype, kPolicy, true, true, d, what));
  mean_kernel<3><<<kSumCtas, kSumThreads, 0, s>>>(a.row_out, nullptr, 0, total, nullptr, a.rows, loss, stats);
  return check_launch(s, what);
}

}  // extern "C"
