// log_prob_losses.cu -- losses over the log-softmax of rows of class scores:
// the log-probability of a chosen class, distillation from a teacher's top
// logits, the preference loss over pairs of sequences and the clipped policy
// loss with a KL term; each forward and backward.
//
// For a row x of V scores at temperature T, with m = max x, c = log2(e) / T:
//   e_j = 2^((x_j - m) c),  s = sum_j e_j,  p_j = e_j / s.
// Every gradient with respect to the scores has the form
//   d x_j = a (p_j - q_j)
// with one factor a per row and q non-zero in the row's few chosen classes
// (one for a chosen class, the teacher's top K for distillation), so one row
// kernel serves all of them: pass 1 finds (m, s), the row's end computes its
// loss and a, pass 2 writes a p_j over the row and then the chosen classes
// again with a (p_j - q_j).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "b2_internal.cuh"

namespace cg = cooperative_groups;

namespace b2 {
namespace {

constexpr int kRowThreads = 256;  // of a CTA, whether it has one row or one row a warp
constexpr int kWarps = kRowThreads / 32;
constexpr int kWarpRowClasses = 1024;  // rows up to this long are a warp's
constexpr int kUnroll = 4;             // 16-byte loads in flight per thread in pass 1
constexpr int kMaxTop = 1024;          // teacher entries of a row
constexpr int kFilterWords = 128;      // words of the bit filter that finds repeated classes

enum Mode { kLogProb = 0, kDistill = 1, kPolicy = 2 };

struct RowArgs {
  const void* x;
  int64_t rows, inner, outer_stride, inner_stride;
  int classes;
  float c;  // log2(e) / temperature
  double temperature;
  int has_stats;   // 1: stats are given (backward), 0: pass 1 finds them
  float2* stats;   // [rows] (m, s): written by pass 1 unless null
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
  double clip_low, clip_high, kl_coef;
  // results per row
  float* log_probs;
  double* row_out;  // [1 or 3][rows], multiplied by the row's weight
};

// ------------------------------------------------------------ element types

template <class T>
struct Pack;
template <>
struct Pack<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ float narrow(float v) { return v; }
  static __device__ __forceinline__ void widen(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Pack<__half> {
  static constexpr int n = 8;
  static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void widen(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Pack<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void widen(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ float exp2_fast(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

__device__ __forceinline__ int64_t class_at(const void* ids, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(ids)[i] : (int64_t) static_cast<const int32_t*>(ids)[i];
}

__device__ __forceinline__ float weight_at(const void* w, int bytes, int64_t i) {
  if (w == nullptr) return 1.0f;
  return bytes == 4 ? static_cast<const float*>(w)[i] : (static_cast<const uint8_t*>(w)[i] != 0 ? 1.0f : 0.0f);
}

__device__ __forceinline__ float teacher_at(const void* y, int dtype, int64_t i) {
  if (dtype == B2_FLOAT32) return static_cast<const float*>(y)[i];
  if (dtype == B2_FLOAT16) return __half2float(static_cast<const __half*>(y)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(y)[i]);
}

// ------------------------------------------------------- running softmax

// (m, s) of a part of a row: the largest value seen and the sum of
// 2^((x - m) c).  An empty part, or one of -inf only, is (-inf, 0).
struct Stat {
  float m, s;
};

// Factor that takes a sum relative to `from` to one relative to `to` >= from;
// equal maxima (both may be infinite) need none.
__device__ __forceinline__ float rescale(float from, float to, float c) {
  return from == to ? 1.0f : exp2_fast((from - to) * c);
}

// Written without a fused multiply-add, so that merge(a, b) and merge(b, a), which the two lanes of
// an exchange compute, are the same bits.
__device__ __forceinline__ Stat merge(Stat a, Stat b, float c) {
  const float m = fmaxf(a.m, b.m);
  return Stat{m, __fadd_rn(__fmul_rn(a.s, rescale(a.m, m, c)), __fmul_rn(b.s, rescale(b.m, m, c)))};
}

template <int N>
__device__ __forceinline__ void add_values(Stat& st, const float* f, float c) {
  float mx = f[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mx = fmaxf(mx, f[i]);
  if (mx > st.m) {
    st.s *= exp2_fast((st.m - mx) * c);  // -inf - mx at the first finite value: 0 * 0
    st.m = mx;
  }
  const float base = st.m == -INFINITY ? 0.0f : st.m;  // -inf values only: each adds 2^-inf = 0
  float part = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) part += exp2_fast((f[i] - base) * c);
  st.s += part;
}

// The part of a row that one thread of `kGroup` adds up.
template <class T, int kGroup>
__device__ __forceinline__ Stat row_part(const T* __restrict__ row, int n, int lane, float c) {
  constexpr int N = Pack<T>::n;
  Stat st{-INFINITY, 0.0f};
  const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
  const int nvec = (n - head) / N;
  const int tail = head + nvec * N;
  if (lane < head) {
    const float f = Pack<T>::one(row[lane]);
    add_values<1>(st, &f, c);
  }
  if (tail + lane < n) {
    const float f = Pack<T>::one(row[tail + lane]);
    add_values<1>(st, &f, c);
  }
  const uint4* __restrict__ v = reinterpret_cast<const uint4*>(row + head);
  int i = lane;
  for (; i + (kUnroll - 1) * kGroup < nvec; i += kUnroll * kGroup) {
    uint4 u[kUnroll];
    float f[kUnroll * N];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) u[k] = __ldg(v + i + k * kGroup);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) Pack<T>::widen(u[k], f + k * N);
    add_values<kUnroll * N>(st, f, c);
  }
  for (; i < nvec; i += kGroup) {
    float f[N];
    Pack<T>::widen(__ldg(v + i), f);
    add_values<N>(st, f, c);
  }
  return st;
}

__device__ __forceinline__ Stat warp_merge(Stat st, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stat other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o)};
    st = merge(st, other, c);
  }
  return st;
}

// out[j] = factor * 2^((row[j] - m) c), or zeros.  Vectors where the row and
// its gradient start equally far from a 16-byte border, else one value at a time.
template <class T, int kGroup>
__device__ __forceinline__ void write_row(const T* __restrict__ row, T* __restrict__ out, int n, int lane, float m,
                                          float c, float factor) {
  constexpr int N = Pack<T>::n;
  const uintptr_t a = reinterpret_cast<uintptr_t>(row), b = reinterpret_cast<uintptr_t>(out);
  if (((a ^ b) & 15) != 0) {
    for (int i = lane; i < n; i += kGroup)
      out[i] = Pack<T>::narrow(factor * exp2_fast((Pack<T>::one(row[i]) - m) * c));
    return;
  }
  const int head = min(n, (int)(((16 - (a & 15)) & 15) / sizeof(T)));
  const int nvec = (n - head) / N;
  const int tail = head + nvec * N;
  if (lane < head) out[lane] = Pack<T>::narrow(factor * exp2_fast((Pack<T>::one(row[lane]) - m) * c));
  if (tail + lane < n)
    out[tail + lane] = Pack<T>::narrow(factor * exp2_fast((Pack<T>::one(row[tail + lane]) - m) * c));
  const uint4* __restrict__ v = reinterpret_cast<const uint4*>(row + head);
  uint4* __restrict__ w = reinterpret_cast<uint4*>(out + head);
  for (int i = lane; i < nvec; i += kGroup) {
    float f[N];
    Pack<T>::widen(__ldg(v + i), f);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = factor * exp2_fast((f[k] - m) * c);
    __stcs(w + i, Pack<T>::pack(f));
  }
}

template <class T, int kGroup>
__device__ __forceinline__ void zero_row(T* __restrict__ out, int n, int lane) {
  const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(out) & 15)) & 15) / sizeof(T)));
  constexpr int N = Pack<T>::n;
  const int nvec = (n - head) / N, tail = head + nvec * N;
  if (lane < head) out[lane] = Pack<T>::narrow(0.0f);
  if (tail + lane < n) out[tail + lane] = Pack<T>::narrow(0.0f);
  uint4* w = reinterpret_cast<uint4*>(out + head);
  for (int i = lane; i < nvec; i += kGroup) __stcs(w + i, make_uint4(0, 0, 0, 0));
}

// ------------------------------------------------------------- the teacher

// A row's teacher entries in shared memory, [top] each: the class (-1: none)
// and its probability q, plus two bit filters over the classes, by which an
// entry sees whether its class may be repeated in the row.
struct Teacher {
  int* ids;
  float* q;
  uint32_t *seen, *again;
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <class F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp lays out the row's teacher: softmax over the entries whose class
// lies in the row and whose logit is not -inf.  Returns false when there is none.
__device__ bool load_teacher(const RowArgs& A, int64_t r, int lane, const Teacher& t, float* ymax, float* log_sum) {
  const int64_t base = r * A.top;
  const float inv_t = (float)(1.0 / A.temperature);
  for (int i = lane; i < kFilterWords; i += 32) t.seen[i] = t.again[i] = 0u;
  float mx = -INFINITY;
  bool nan = false;
  for (int k = lane; k < A.top; k += 32) {
    const int64_t id = class_at(A.ids, A.ids_bytes, base + k);
    const bool real = id >= 0 && id < A.classes;
    const float y = real ? teacher_at(A.teacher, A.teacher_dtype, base + k) : -INFINITY;
    t.ids[k] = real && y != -INFINITY ? (int)id : -1;
    t.q[k] = y;
    mx = fmaxf(mx, y);
    nan |= y != y;
  }
  __syncwarp();
  mx = warp_max(mx);
  nan = __any_sync(0xffffffffu, nan);
  if (mx == -INFINITY && !nan) return false;
  float sum = 0.0f;
  for (int k = lane; k < A.top; k += 32) {
    const int id = t.ids[k];
    const float e = id >= 0 ? expf((t.q[k] - mx) * inv_t) : 0.0f;
    t.q[k] = e;
    sum += e;
    if (id >= 0) {
      const uint32_t bit = 1u << (id & 31);
      const int word = (id >> 5) & (kFilterWords - 1);
      if (atomicOr(&t.seen[word], bit) & bit) atomicOr(&t.again[word], bit);
    }
  }
  sum = warp_sum(sum);
  for (int k = lane; k < A.top; k += 32) t.q[k] = t.q[k] / sum;
  __syncwarp();
  *ymax = mx;
  *log_sum = logf(sum);
  return true;
}

// Sum of q over the entries of the class of entry k, added in the entries'
// order (every repeated entry gets the same bits).
__device__ __forceinline__ float class_q(const Teacher& t, int k, int top) {
  const int id = t.ids[k];
  if (!((t.again[(id >> 5) & (kFilterWords - 1)] >> (id & 31)) & 1u)) return t.q[k];
  float sum = 0.0f;
  for (int i = 0; i < top; ++i) sum += t.ids[i] == id ? t.q[i] : 0.0f;
  return sum;
}

// ------------------------------------------------------------- row kernel

// One row per warp (kGroup 32), or per CTA, or per cluster of CTAs that each
// have a slice of it (kGroup kRowThreads).  Each row's values are read from
// HBM once: pass 2 finds them in L2.
template <class T, int kMode, int kGroup>
__global__ void __launch_bounds__(kRowThreads) row_kernel(const RowArgs A) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Stat part[kWarps];
  __shared__ Stat cta_stat;
  __shared__ float factor_s;
  __shared__ int real_s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = kGroup == 32 ? 1 : (int)cluster.num_blocks();
  const int rank = kGroup == 32 ? 0 : (int)cluster.block_rank();
  const int64_t r = kGroup == 32 ? (int64_t)blockIdx.x * kWarps + warp : (int64_t)blockIdx.x / ranks;
  if (kGroup == 32 && r >= A.rows) return;
  const int g = kGroup == 32 ? lane : (int)threadIdx.x;
  const bool leader_warp = kGroup == 32 || warp == 0;

  const T* row = static_cast<const T*>(A.x) + (r / A.inner) * A.outer_stride + (r % A.inner) * A.inner_stride;
  int n = A.classes, begin = 0;
  if (ranks > 1) {
    const int slice = (n + ranks * 8 - 1) / (ranks * 8) * 8;
    begin = min(n, rank * slice);
    n = min(n - begin, slice);
  }
  T* out = static_cast<T*>(A.grad) + r * A.classes + begin;

  Teacher teacher{};
  if (kMode == kDistill) {
    uint32_t* words = reinterpret_cast<uint32_t*>(dyn) + (kGroup == 32 ? warp : 0) * (2 * kFilterWords + 2 * A.top);
    teacher = Teacher{reinterpret_cast<int*>(words + 2 * kFilterWords),
                      reinterpret_cast<float*>(words + 2 * kFilterWords + A.top), words, words + kFilterWords};
  }

  // Rows that do not count: their values are not looked at.
  float w = 1.0f;
  int64_t target = -1;
  if (kMode == kDistill || kMode == kPolicy) w = weight_at(A.weights, A.weight_bytes, r);
  if (kMode != kDistill) {
    target = class_at(A.ids, A.ids_bytes, r);
    if (target >= A.classes) target = -1;
  }
  const bool grad_only = A.has_stats != 0;
  float up = 1.0f;
  if (kMode == kLogProb && grad_only) up = A.upstream[r];
  const bool skip = kMode == kDistill ? w == 0.0f : kMode == kPolicy ? w == 0.0f : target < 0 || up == 0.0f;
  if (skip) {
    if (A.grad != nullptr) zero_row<T, kGroup>(out, n, g);
    if (rank == 0 && g == 0 && !grad_only) {
      if (kMode == kLogProb) A.log_probs[r] = 0.0f;
      if (kMode == kDistill) A.row_out[r] = 0.0;
      if (kMode == kPolicy) A.row_out[r] = A.row_out[A.rows + r] = A.row_out[2 * A.rows + r] = 0.0;
      if (A.stats != nullptr) A.stats[r] = make_float2(0.0f, 1.0f);
    }
    return;  // the whole cluster has the same row
  }

  float ymax = 0.0f, log_sum_q = 0.0f;
  bool real = true;
  if (kMode == kDistill && leader_warp) real = load_teacher(A, r, lane, teacher, &ymax, &log_sum_q);

  // ---- pass 1
  Stat st;
  if (grad_only) {
    const float2 v = A.stats[r];
    st = Stat{v.x, v.y};
  } else {
    st = warp_merge(row_part<T, kGroup>(row + begin, n, g, A.c), A.c);
    if (kGroup != 32) {
      if (lane == 0) part[warp] = st;
      __syncthreads();
      st = warp_merge(lane < kWarps ? part[lane] : Stat{-INFINITY, 0.0f}, A.c);
      if (ranks > 1) {
        if (threadIdx.x == 0) cta_stat = st;
        cluster.sync();
        st = warp_merge(lane < ranks ? *cluster.map_shared_rank(&cta_stat, lane) : Stat{-INFINITY, 0.0f}, A.c);
        cluster.sync();  // every CTA has read the others' shared memory
      }
    }
    if (A.stats != nullptr && rank == 0 && g == 0) A.stats[r] = make_float2(st.m, st.s);
  }

  // ---- the row's end: its loss and the factor of its gradient
  const float log_s = logf(st.s);
  const double gl = A.grad_loss != nullptr ? (double)*A.grad_loss : 1.0;
  const double total = A.total != nullptr ? *A.total : (double)A.rows;
  const double share = total != 0.0 ? (double)w / total : 0.0;
  float factor = 0.0f;
  if (kMode == kLogProb) {
    if (!grad_only && rank == 0 && g == 0)
      A.log_probs[r] = (float)((double)(Pack<T>::one(row[target]) - st.m) - log((double)st.s));
    factor = -up;
  } else if (kMode == kDistill) {
    if (leader_warp) {
      if (!grad_only && real && rank == 0) {
        const double inv_t = 1.0 / A.temperature;
        double sum = 0.0;
        for (int k = lane; k < A.top; k += 32) {
          const int id = teacher.ids[k];
          const float q = teacher.q[k];
          if (id < 0 || q == 0.0f) continue;
          const double log_q =
              (double)(teacher_at(A.teacher, A.teacher_dtype, r * A.top + k) - ymax) * inv_t - (double)log_sum_q;
          const double log_p = (double)(Pack<T>::one(row[id]) - st.m) * inv_t - (double)log_s;
          sum += (double)q * (log_q - log_p);
        }
        sum = warp_sum(sum);
        if (lane == 0) A.row_out[r] = (double)w * sum * A.temperature * A.temperature;
      } else if (!grad_only && rank == 0 && lane == 0) {
        A.row_out[r] = 0.0;
      }
      if (kGroup != 32 && lane == 0) real_s = real;
    }
    factor = (float)(gl * A.temperature * share);
  } else {
    if (g == 0) {
      const double lp = target >= 0 ? (double)(float)((double)(Pack<T>::one(row[target]) - st.m) - log((double)st.s)) : 0.0;
      const double adv = A.advantages[r], ratio = exp(lp - (double)A.old_lp[r]);
      const bool cut = (adv > 0.0 && ratio > 1.0 + A.clip_high) || (adv < 0.0 && ratio < 1.0 - A.clip_low);
      const double held = fmin(fmax(ratio, 1.0 - A.clip_low), 1.0 + A.clip_high);
      double value = fmax(-ratio * adv, -held * adv), slope = cut ? 0.0 : -adv * ratio, kl = 0.0;
      if (A.ref_lp != nullptr) {
        const double d = (double)A.ref_lp[r] - lp, over = expm1(d);
        kl = over - d;
        value += A.kl_coef * kl;
        slope -= A.kl_coef * over;
      }
      if (rank == 0) {
        A.row_out[r] = (double)w * value;
        A.row_out[A.rows + r] = (double)w * kl;
        A.row_out[2 * A.rows + r] = cut ? (double)w : 0.0;
      }
      factor = (float)(-gl * share * slope);
      if (kGroup != 32) factor_s = factor;
    }
    if (kGroup == 32) factor = __shfl_sync(0xffffffffu, factor, 0);
  }
  if (A.grad == nullptr) return;
  if (kGroup != 32) {
    __syncthreads();
    if (kMode == kPolicy) factor = factor_s;
    if (kMode == kDistill) real = real_s != 0;
  }

  // ---- pass 2
  if (kMode == kDistill ? !real : target < 0) {
    zero_row<T, kGroup>(out, n, g);
    return;
  }
  const float inv_s = 1.0f / st.s;
  write_row<T, kGroup>(row + begin, out, n, g, st.m, A.c, factor * inv_s);
  if (kGroup == 32)
    __syncwarp();
  else
    __syncthreads();  // the row's a p is written before the chosen classes are written again
  if (kMode == kDistill) {
    for (int k = g; k < A.top; k += kGroup) {
      const int j = teacher.ids[k] - begin;
      if (teacher.ids[k] < 0 || j < 0 || j >= n) continue;
      const float p = exp2_fast((Pack<T>::one(row[begin + j]) - st.m) * A.c) * inv_s;
      out[j] = Pack<T>::narrow(factor * (p - class_q(teacher, k, A.top)));
    }
  } else if (g == 0) {
    const int64_t j = target - begin;
    if (j >= 0 && j < n) {
      const float p = exp2_fast((Pack<T>::one(row[target]) - st.m) * A.c) * inv_s;
      out[j] = Pack<T>::narrow(factor * (p - 1.0f));
    }
  }
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

// *loss and stats[k - 1] = sum_r values[k][r] / total, 0 when the total is 0.
template <int kN>
__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    mean_kernel(const double* __restrict__ values, const double* __restrict__ total, int64_t rows,
                float* __restrict__ loss, float* __restrict__ stats) {
  double v[kN] = {};
  for (int64_t i = (int64_t)blockIdx.x * kSumThreads + threadIdx.x; i < rows; i += kSumCtas * kSumThreads)
#pragma unroll
    for (int k = 0; k < kN; ++k) v[k] += values[k * rows + i];
  cluster_sum<kN>(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const double t = total != nullptr ? *total : (double)rows;
#pragma unroll
    for (int k = 0; k < kN; ++k) (k == 0 ? loss : stats + k - 1)[0] = t != 0.0 ? (float)(v[k] / t) : 0.0f;
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

// One CTA per sequence: rewards[i] = beta sum_n w_n (lp_n - ref_n).
__global__ void __launch_bounds__(kTokenThreads) sequence_sum_kernel(const PreferenceArgs A, double* __restrict__ sums) {
  __shared__ double part[kTokenThreads / 32];
  const int64_t i = blockIdx.x;
  const int64_t a = offset_at(A.offsets, A.offset_bytes, i, A.tokens);
  const int64_t b = offset_at(A.offsets, A.offset_bytes, i + 1, A.tokens);
  double v = 0.0;
  for (int64_t n = a + threadIdx.x; n < b; n += kTokenThreads) {
    const float w = weight_at(A.mask, A.mask_bytes, n);
    if (w != 0.0f) v += (double)w * ((double)A.lp[n] - (A.ref != nullptr ? (double)A.ref[n] : 0.0));
  }
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    double c = 0.0;
    for (int k = 0; k < kTokenThreads / 32; ++k) c += part[k];
    sums[i] = A.beta * c;
  }
}

__device__ __forceinline__ double softplus(double z) { return fmax(z, 0.0) + log1p(exp(-fabs(z))); }

__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    pair_kernel(const PreferenceArgs A, const double* __restrict__ sums, float* __restrict__ loss,
                float* __restrict__ rewards, float* __restrict__ slopes) {
  double v[1] = {0.0};
  const double eps = A.smoothing;
  for (int64_t p = (int64_t)blockIdx.x * kSumThreads + threadIdx.x; p < A.pairs; p += kSumCtas * kSumThreads) {
    const double chosen = sums[p], rejected = sums[A.pairs + p], h = chosen - rejected;
    v[0] += (1.0 - eps) * softplus(-h) + eps * softplus(h);
    // sigma(h) and sigma(-h), each without cancellation
    const double z = exp(-fabs(h)), small = z / (1.0 + z), large = 1.0 / (1.0 + z);
    const double up = h >= 0.0 ? large : small, down = h >= 0.0 ? small : large;
    const double slope = (eps * up - (1.0 - eps) * down) * A.beta / (double)A.pairs;
    rewards[p] = (float)chosen;
    rewards[A.pairs + p] = (float)rejected;
    slopes[p] = (float)slope;
    slopes[A.pairs + p] = (float)-slope;
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
    grad[n] = seq >= 0 && seq < 2 * A.pairs && w != 0.0f ? gl * slopes[seq] * w : 0.0f;
  }
}

// ------------------------------------------------------------------- policy

struct PolicyArgs {
  const float *lp, *old_lp, *ref_lp, *advantages;
  const void* mask;
  int mask_bytes;
  int64_t tokens;
  double clip_low, clip_high, kl_coef;
};

constexpr int kPolicySums = 4;  // loss, kl, clipped, weights

__global__ void __launch_bounds__(kTokenThreads)
    policy_kernel(const PolicyArgs A, float* __restrict__ slopes, double* __restrict__ partial) {
  __shared__ double part[kPolicySums][kTokenThreads / 32];
  double v[kPolicySums] = {};
  for (int64_t n = (int64_t)blockIdx.x * kTokenThreads + threadIdx.x; n < A.tokens;
       n += (int64_t)gridDim.x * kTokenThreads) {
    const double w = weight_at(A.mask, A.mask_bytes, n);
    double slope = 0.0;
    if (w != 0.0) {
      const double lp = A.lp[n], adv = A.advantages[n], ratio = exp(lp - (double)A.old_lp[n]);
      const bool cut = (adv > 0.0 && ratio > 1.0 + A.clip_high) || (adv < 0.0 && ratio < 1.0 - A.clip_low);
      const double held = fmin(fmax(ratio, 1.0 - A.clip_low), 1.0 + A.clip_high);
      double value = fmax(-ratio * adv, -held * adv), kl = 0.0;
      slope = cut ? 0.0 : -adv * ratio;
      if (A.ref_lp != nullptr) {
        const double d = (double)A.ref_lp[n] - lp, over = expm1(d);
        kl = over - d;
        value += A.kl_coef * kl;
        slope -= A.kl_coef * over;
      }
      v[0] += w * value;
      v[1] += w * kl;
      v[2] += cut ? w : 0.0;
      v[3] += w;
    }
    if (slopes != nullptr) slopes[n] = (float)(w * slope);
  }
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

// *loss, stats = {mean KL, clipped share, 1 / sum of the weights}, all 0 when the weights sum to 0.
__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    policy_mean_kernel(const double* __restrict__ partial, int64_t parts, float* __restrict__ loss,
                       float* __restrict__ stats) {
  double v[kPolicySums] = {};
  for (int64_t i = (int64_t)blockIdx.x * kSumThreads + threadIdx.x; i < parts; i += kSumCtas * kSumThreads)
#pragma unroll
    for (int k = 0; k < kPolicySums; ++k) v[k] += partial[k * parts + i];
  cluster_sum<kPolicySums>(v);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const double inv = v[3] != 0.0 ? 1.0 / v[3] : 0.0;
    *loss = v[3] != 0.0 ? (float)(v[0] / v[3]) : 0.0f;
    stats[0] = v[3] != 0.0 ? (float)(v[1] / v[3]) : 0.0f;
    stats[1] = v[3] != 0.0 ? (float)(v[2] / v[3]) : 0.0f;
    stats[2] = (float)inv;
  }
}

__global__ void __launch_bounds__(kTokenThreads)
    policy_grad_kernel(const float* __restrict__ grad_loss, const float* __restrict__ inv_total,
                       const float* __restrict__ slopes, int64_t tokens, float* __restrict__ grad) {
  const float f = *grad_loss * *inv_total;
  for (int64_t n = (int64_t)blockIdx.x * kTokenThreads + threadIdx.x; n < tokens;
       n += (int64_t)gridDim.x * kTokenThreads)
    grad[n] = slopes[n] == 0.0f ? 0.0f : f * slopes[n];
}

// ------------------------------------------------------------------ launches

template <class T, int kMode, int kGroup>
int launch_rows_as(cudaStream_t s, const RowArgs& a, int cluster, const DeviceInfo* d, const char* what) {
  static SmemOptIn opt;
  auto kernel = row_kernel<T, kMode, kGroup>;
  const int groups = kGroup == 32 ? kWarps : 1;
  const size_t smem = kMode == kDistill ? (size_t)groups * 4 * (2 * kFilterWords + 2 * a.top) : 0;
  if (smem > 32 * 1024) B2_RETURN_IF_ERROR(opt.ensure(reinterpret_cast<const void*>(kernel), d->device, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(kGroup == 32 ? ceil_div(a.rows, kWarps) : a.rows * cluster));
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B2_CUDA_OR_RETURN(cudaLaunchKernelEx(&cfg, kernel, a));
  return check_launch(s, what);
}

template <int kMode>
int launch_rows(cudaStream_t s, const RowArgs& a, int dtype, const DeviceInfo* d, const char* what) {
  // Few rows: each is split over a cluster, so that the GPU's SMs share it.
  int cluster = 1;
  const bool by_warp = a.classes <= kWarpRowClasses;
  while (!by_warp && cluster < 8 && a.rows * cluster * 2 <= 2 * d->sm_count && a.classes / (cluster * 2) >= 2048)
    cluster *= 2;
  if (by_warp) {
    if (dtype == B2_FLOAT32) return launch_rows_as<float, kMode, 32>(s, a, 1, d, what);
    if (dtype == B2_FLOAT16) return launch_rows_as<__half, kMode, 32>(s, a, 1, d, what);
    return launch_rows_as<__nv_bfloat16, kMode, 32>(s, a, 1, d, what);
  }
  if (dtype == B2_FLOAT32) return launch_rows_as<float, kMode, kRowThreads>(s, a, cluster, d, what);
  if (dtype == B2_FLOAT16) return launch_rows_as<__half, kMode, kRowThreads>(s, a, cluster, d, what);
  return launch_rows_as<__nv_bfloat16, kMode, kRowThreads>(s, a, cluster, d, what);
}

// Checks a row view and starts the kernel's arguments with it.
int row_args(const b2_logits_t* x, const char* what, RowArgs* a) {
  B2_REQUIRE(x != nullptr, "%s: null logits", what);
  B2_REQUIRE(x->dtype == B2_FLOAT32 || x->dtype == B2_FLOAT16 || x->dtype == B2_BFLOAT16,
             "%s: logits must be float32, float16 or bfloat16", what);
  B2_REQUIRE(x->outer >= 0 && x->inner >= 0, "%s: negative number of rows", what);
  B2_REQUIRE(x->classes >= 1 && x->classes < kMaxInt32, "%s: classes must be in [1, 2^31 - 2], got %lld", what,
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
  a->temperature = 1.0;
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
  if (a.rows == 0) return B2_OK;
  B2_REQUIRE(targets != nullptr && log_probs != nullptr, "token_log_probs: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  a.ids = targets;
  a.ids_bytes = target_bytes;
  a.log_probs = log_probs;
  a.stats = reinterpret_cast<float2*>(row_stats);
  return launch_rows<kLogProb>(static_cast<cudaStream_t>(stream), a, logits->dtype, d, "token_log_probs");
}

int b2_token_log_probs_grad(b2_stream_t stream, const b2_logits_t* logits, const void* targets, int target_bytes,
                            const float* row_stats, const float* grad_log_probs, void* grad_logits) {
  clear_error();
  RowArgs a;
  B2_RETURN_IF_ERROR(row_args(logits, "token_log_probs_grad", &a));
  B2_RETURN_IF_ERROR(index_ok(target_bytes, "token_log_probs_grad", "targets"));
  if (a.rows == 0) return B2_OK;
  B2_REQUIRE(targets != nullptr && row_stats != nullptr && grad_log_probs != nullptr && grad_logits != nullptr,
             "token_log_probs_grad: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  a.ids = targets;
  a.ids_bytes = target_bytes;
  a.has_stats = 1;
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(row_stats));
  a.upstream = grad_log_probs;
  a.grad = grad_logits;
  return launch_rows<kLogProb>(static_cast<cudaStream_t>(stream), a, logits->dtype, d, "token_log_probs_grad");
}

static int distill_args(const b2_logits_t* logits, const void* teacher_ids, int id_bytes, const void* teacher_logits,
                        int teacher_dtype, int64_t top, const void* weights, int weight_bytes, double temperature,
                        const char* what, RowArgs* a) {
  B2_RETURN_IF_ERROR(row_args(logits, what, a));
  B2_RETURN_IF_ERROR(index_ok(id_bytes, what, "teacher_ids"));
  B2_RETURN_IF_ERROR(weight_ok(weights, weight_bytes, what));
  B2_REQUIRE(a->rows > 0, "%s: the mean over no rows is undefined", what);
  B2_REQUIRE(top >= 1 && top <= kMaxTop, "%s: the teacher's entries per row must be in [1, %d], got %lld", what, kMaxTop,
             (long long)top);
  B2_REQUIRE(teacher_dtype == B2_FLOAT32 || teacher_dtype == B2_FLOAT16 || teacher_dtype == B2_BFLOAT16,
             "%s: teacher_logits must be float32, float16 or bfloat16", what);
  B2_REQUIRE(temperature > 0.0 && std::isfinite(temperature), "%s: temperature must be positive and finite", what);
  B2_REQUIRE(teacher_ids != nullptr && teacher_logits != nullptr, "%s: null pointer", what);
  a->ids = teacher_ids;
  a->ids_bytes = id_bytes;
  a->teacher = teacher_logits;
  a->teacher_dtype = teacher_dtype;
  a->top = (int)top;
  a->weights = weights;
  a->weight_bytes = weight_bytes;
  a->temperature = temperature;
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
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Scratch scratch;
  B2_RETURN_IF_ERROR(scratch.alloc((a.rows + 1) * sizeof(double), s));
  double* total = weights != nullptr ? scratch.as<double>() + a.rows : nullptr;
  if (total != nullptr)
    B2_RETURN_IF_ERROR(sum_weights(s, weights, weight_bytes, a.rows, total, "distillation_loss"));
  a.total = total;
  a.row_out = scratch.as<double>();
  a.stats = reinterpret_cast<float2*>(row_stats);
  a.grad_loss = grad_loss;
  a.grad = grad_logits;
  B2_RETURN_IF_ERROR(launch_rows<kDistill>(s, a, logits->dtype, d, "distillation_loss"));
  mean_kernel<1><<<kSumCtas, kSumThreads, 0, s>>>(a.row_out, total, a.rows, loss, nullptr);
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
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Scratch scratch;
  if (weights != nullptr) {
    B2_RETURN_IF_ERROR(scratch.alloc(sizeof(double), s));
    B2_RETURN_IF_ERROR(
        sum_weights(s, weights, weight_bytes, a.rows, scratch.as<double>(), "distillation_loss_grad"));
    a.total = scratch.as<double>();
  }
  a.has_stats = 1;
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(row_stats));
  a.grad_loss = grad_loss;
  a.grad = grad_logits;
  return launch_rows<kDistill>(s, a, logits->dtype, d, "distillation_loss_grad");
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
  B2_REQUIRE(log_probs != nullptr && old_log_probs != nullptr && advantages != nullptr && loss != nullptr && stats != nullptr,
             "policy_loss: null pointer");
  const DeviceInfo* d = nullptr;
  B2_RETURN_IF_ERROR(device_info(&d));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const PolicyArgs a{log_probs, old_log_probs, ref_log_probs, advantages, mask, mask_bytes, tokens, clip_low,
                     clip_high, kl_coef};
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
  B2_REQUIRE(targets != nullptr && old_log_probs != nullptr && advantages != nullptr && loss != nullptr && stats != nullptr &&
                 grad_logits != nullptr,
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
  a.clip_low = clip_low;
  a.clip_high = clip_high;
  a.kl_coef = kl_coef;
  a.grad_loss = grad_loss;
  a.row_out = scratch.as<double>();
  a.grad = grad_logits;
  B2_RETURN_IF_ERROR(launch_rows<kPolicy>(s, a, logits->dtype, d, what));
  mean_kernel<3><<<kSumCtas, kSumThreads, 0, s>>>(a.row_out, total, a.rows, loss, stats);
  return check_launch(s, what);
}

}  // extern "C"
