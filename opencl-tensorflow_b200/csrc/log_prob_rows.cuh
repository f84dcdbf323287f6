// log_prob_rows.cuh -- the passes over rows of class scores, for one type of
// score; included by one source file a type, so that they compile in parallel.
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
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

#include "log_prob_common.cuh"

namespace cg = cooperative_groups;

namespace b2 {
namespace {

constexpr int kBatch = 4;       // 16-byte vectors that a thread adds up at a time
constexpr int kMaxCluster = 8;  // CTAs of a row, the portable cluster size

// ------------------------------------------------------------ element types

// A 16-byte vector of a type: its values as pairs of fp32, its largest value.
template <class T>
struct Pack;
template <>
struct Pack<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ float narrow(float v) { return v; }
  static __device__ __forceinline__ void widen(const uint4& u, float2* f) {
    f[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2* f) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x),
                      __float_as_uint(f[1].y));
  }
  static __device__ __forceinline__ float largest(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
};
template <>
struct Pack<__half> {
  static constexpr int n = 8;
  static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ __half2 pair(const uint32_t& w) { return *reinterpret_cast<const __half2*>(&w); }
  static __device__ __forceinline__ void widen(const uint4& u, float2* f) {
    f[0] = __half22float2(pair(u.x)), f[1] = __half22float2(pair(u.y));
    f[2] = __half22float2(pair(u.z)), f[3] = __half22float2(pair(u.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __float22half2_rn(f[i]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float largest(const uint4& u) {
    const float2 f = __half22float2(__hmax2(__hmax2(pair(u.x), pair(u.y)), __hmax2(pair(u.z), pair(u.w))));
    return fmaxf(f.x, f.y);
  }
};
template <>
struct Pack<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ __nv_bfloat162 pair(const uint32_t& w) {
    return *reinterpret_cast<const __nv_bfloat162*>(&w);
  }
  static __device__ __forceinline__ float2 split(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void widen(const uint4& u, float2* f) {
    f[0] = split(u.x), f[1] = split(u.y), f[2] = split(u.z), f[3] = split(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float2* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __float22bfloat162_rn(f[i]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float largest(const uint4& u) {
    const __nv_bfloat162 h = __hmax2(__hmax2(pair(u.x), pair(u.y)), __hmax2(pair(u.z), pair(u.w)));
    const float2 f = split(*reinterpret_cast<const uint32_t*>(&h));
    return fmaxf(f.x, f.y);
  }
};

__device__ __forceinline__ float exp2_fast(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

// Two fp32 operations in one instruction (each rounded like its single form).
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return r;
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

__device__ __forceinline__ float raise_max(Stat& st, float mx, float c) {
  if (mx > st.m) {
    st.s *= exp2_fast((st.m - mx) * c);  // at the first finite value: 0 * 2^-inf
    st.m = mx;
  }
  return st.m == -INFINITY ? 0.0f : st.m;  // with -inf values only, each adds 2^-inf = 0
}

__device__ __forceinline__ void add_value(Stat& st, float f, float c) {
  const float base = raise_max(st, f, c);
  st.s += exp2_fast((f - base) * c);
}

// 2^((f - m) c) of a vector's values.
template <class T>
__device__ __forceinline__ void exp_vector(const uint4& u, float m, float c, float2* f) {
  const float2 minus_m = make_float2(-m, -m), c2 = make_float2(c, c);
  Pack<T>::widen(u, f);
#pragma unroll
  for (int i = 0; i < Pack<T>::n / 2; ++i) {
    f[i] = mul2(add2(f[i], minus_m), c2);
    f[i] = make_float2(exp2_fast(f[i].x), exp2_fast(f[i].y));
  }
}

// Adds K vectors: their maximum first, from the packed values, then one
// rescaling of the sum at most, then the exponentials.
template <class T, int K>
__device__ __forceinline__ void add_vectors(Stat& st, const uint4* u, float c) {
  float mx = Pack<T>::largest(u[0]);
#pragma unroll
  for (int k = 1; k < K; ++k) mx = fmaxf(mx, Pack<T>::largest(u[k]));
  const float base = raise_max(st, mx, c);
  float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float2 f[Pack<T>::n / 2];
    exp_vector<T>(u[k], base, c, f);
#pragma unroll
    for (int i = 0; i < Pack<T>::n / 2; ++i) sum = add2(sum, f[i]);
  }
  st.s += sum.x + sum.y;
}

// Where a slice of a row starts against 16-byte borders: `head` values before
// the first vector, `nvec` vectors, the rest from `tail` on.
struct Span {
  int head, nvec, tail;
};
template <class T>
__device__ __forceinline__ Span span_of(const T* p, int n) {
  Span s;
  s.head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
  s.nvec = (n - s.head) / Pack<T>::n;
  s.tail = s.head + s.nvec * Pack<T>::n;
  return s;
}

// A vector of -inf.
template <class T>
__device__ __forceinline__ uint4 empty_vector() {
  const uint32_t w = std::is_same<T, float>::value    ? 0xff800000u
                     : std::is_same<T, __half>::value ? 0xfc00fc00u
                                                      : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}

template <class T>
__device__ __forceinline__ void add_edges(Stat& st, const T* __restrict__ row, const Span& sp, int n, int g, float c) {
  if (g < sp.head) add_value(st, Pack<T>::one(row[g]), c);
  if (sp.tail + g < n) add_value(st, Pack<T>::one(row[sp.tail + g]), c);
}

// A vector of scores.  kAgain: it is read again, so it may stay in L1 (without
// that, loss and gradient of 4096 x 128000 bf16 take 100 us more); else it passes
// L1 by (the forward of 131072 x 2000 then takes 103 us instead of 109).
template <bool kAgain>
__device__ __forceinline__ uint4 load_vector(const uint4* p) {
  if (kAgain) return __ldg(p);
  uint4 u;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
               : "l"(p));
  return u;
}

// The vectors of a slice that thread g of kGroup adds up.
template <class T, int kGroup, bool kAgain>
__device__ __forceinline__ Stat vectors_part(const T* __restrict__ row, const Span& sp, int g, float c) {
  Stat st{-INFINITY, 0.0f};
  const uint4* __restrict__ v = reinterpret_cast<const uint4*>(row + sp.head);
  int i = g;
  for (; i + (kBatch - 1) * kGroup < sp.nvec; i += kBatch * kGroup) {
    uint4 u[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) u[k] = load_vector<kAgain>(v + i + k * kGroup);
    add_vectors<T, kBatch>(st, u, c);
  }
  if (i < sp.nvec) {  // what is left, together
    uint4 u[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      u[k] = i + k * kGroup < sp.nvec ? load_vector<kAgain>(v + i + k * kGroup) : empty_vector<T>();
    add_vectors<T, kBatch>(st, u, c);
  }
  return st;
}

// The part of a slice that thread g of kGroup adds up.
template <class T, int kGroup, bool kAgain>
__device__ __forceinline__ Stat slice_part(const T* __restrict__ row, int n, int g, float c) {
  const Span sp = span_of(row, n);
  Stat st = vectors_part<T, kGroup, kAgain>(row, sp, g, c);
  add_edges(st, row, sp, n, g, c);
  return st;
}

// The lanes of a warp that work on one row: all, or kLanes adjacent ones.
template <int kLanes>
__device__ __forceinline__ unsigned lanes_mask() {
  return kLanes == 32 ? 0xffffffffu : ((1u << (kLanes & 31)) - 1u) << (threadIdx.x & 31 & ~(kLanes - 1));
}
template <int kLanes>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(lanes_mask<kLanes>(), v, o));
  return v;
}
template <int kLanes, class F>
__device__ __forceinline__ F lanes_sum(F v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(lanes_mask<kLanes>(), v, o);
  return v;
}

// The lanes' maximum, then each one's sum relative to it: all lanes get the same bits.
template <int kLanes>
__device__ __forceinline__ Stat lanes_merge(Stat st, float c) {
  const float m = lanes_max<kLanes>(st.m);
  return Stat{m, lanes_sum<kLanes>(st.s * rescale(st.m, m, c))};
}

template <int kGroup>
__device__ __forceinline__ void group_sync() {
  if (kGroup <= 32)
    __syncwarp(lanes_mask<kGroup <= 32 ? kGroup : 32>());
  else
    __syncthreads();
}

template <class T>
__device__ __forceinline__ T scaled_exp(T v, float m, float c, float factor) {
  return Pack<T>::narrow(factor * exp2_fast((Pack<T>::one(v) - m) * c));
}

template <class T>
__device__ __forceinline__ bool same_border(const T* a, const T* b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

template <class T>
__device__ __forceinline__ void write_edges(const T* __restrict__ row, T* __restrict__ out, const Span& sp, int n,
                                            int g, float m, float c, float factor) {
  if (g < sp.head) out[g] = scaled_exp(row[g], m, c, factor);
  if (sp.tail + g < n) out[sp.tail + g] = scaled_exp(row[sp.tail + g], m, c, factor);
}

template <class T>
__device__ __forceinline__ uint4 scaled_vector(const uint4& u, float m, float c, float factor) {
  float2 f[Pack<T>::n / 2];
  exp_vector<T>(u, m, c, f);
#pragma unroll
  for (int k = 0; k < Pack<T>::n / 2; ++k) f[k] = mul2(f[k], make_float2(factor, factor));
  return Pack<T>::pack(f);
}

// A vector's last read.  kAgain: it was read before, in this launch: marked as
// streamed it leaves room for others (131072 x 2000 bf16, loss and gradient: 272 us,
// unmarked 347).  Marked, a gradient alone is slower: 524288 x 500 249 us and not 203,
// distillation's of 8192 x 32000 190 and not 172 (but 16384 x 16000 187 and not 196).
template <bool kAgain>
__device__ __forceinline__ uint4 load_last(const uint4* p) {
  return kAgain ? __ldcs(p) : __ldg(p);
}

// out[j] = factor * 2^((row[j] - m) c) in the row's vectors (of which `sp` tells).
template <class T, int kGroup, bool kAgain>
__device__ __forceinline__ void write_vectors(const T* __restrict__ row, T* __restrict__ out, const Span& sp, int n,
                                              int g, float m, float c, float factor) {
  const uint4* __restrict__ v = reinterpret_cast<const uint4*>(row + sp.head);
  uint4* __restrict__ w = reinterpret_cast<uint4*>(out + sp.head);
  int i = g;
  for (; i + (kBatch - 1) * kGroup < sp.nvec; i += kBatch * kGroup) {
    uint4 u[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) u[k] = load_last<kAgain>(v + i + k * kGroup);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) __stcs(w + i + k * kGroup, scaled_vector<T>(u[k], m, c, factor));
  }
  if (i < sp.nvec) {  // what is left, loaded together
    uint4 u[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (i + k * kGroup < sp.nvec) u[k] = load_last<kAgain>(v + i + k * kGroup);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (i + k * kGroup < sp.nvec) __stcs(w + i + k * kGroup, scaled_vector<T>(u[k], m, c, factor));
  }
}

// A slice's gradient without its chosen classes.  Where row and output do not
// lie equally far from a 16-byte border, the values of an output vector are
// read one by one: all positions but the last of 8 sequences of 193 x 50257 bf16, forward
// and gradient, take 111 us, as a dense tensor 90.
template <class T, int kGroup, bool kAgain>
__device__ __forceinline__ void write_slice(const T* __restrict__ row, T* __restrict__ out, int n, int g, float m,
                                            float c, float factor) {
  constexpr int N = Pack<T>::n;
  const Span sp = span_of(out, n);
  write_edges(row, out, sp, n, g, m, c, factor);
  if (same_border<T>(row, out)) {
    write_vectors<T, kGroup, kAgain>(row, out, sp, n, g, m, c, factor);
    return;
  }
  uint4* __restrict__ w = reinterpret_cast<uint4*>(out + sp.head);
  for (int i = g; i < sp.nvec; i += kGroup) {
    const T* __restrict__ from = row + sp.head + i * N;
    float2 f[N / 2];
#pragma unroll
    for (int k = 0; k < N / 2; ++k)
      f[k] = make_float2(factor * exp2_fast((Pack<T>::one(from[2 * k]) - m) * c),
                         factor * exp2_fast((Pack<T>::one(from[2 * k + 1]) - m) * c));
    __stcs(w + i, Pack<T>::pack(f));
  }
}

template <class T, int kGroup>
__device__ __forceinline__ void zero_slice(T* __restrict__ out, int n, int lane) {
  const Span sp = span_of(out, n);
  if (lane < sp.head) out[lane] = Pack<T>::narrow(0.0f);
  if (sp.tail + lane < n) out[sp.tail + lane] = Pack<T>::narrow(0.0f);
  uint4* w = reinterpret_cast<uint4*>(out + sp.head);
  for (int i = lane; i < sp.nvec; i += kGroup) __stcs(w + i, make_uint4(0, 0, 0, 0));
}

// ------------------------------------------------------------- the teacher

// A row's teacher entries in shared memory, [top] each: the class (-1: none),
// its probability q and the row's score x of it, plus two bit filters over the
// classes, by which an entry sees whether its class may be repeated in the row.
struct Teacher {
  int* ids;
  float *q, *x;
  uint32_t *seen, *again;
};
__device__ __forceinline__ Teacher teacher_in(void* shared, int top, int filter_words) {
  uint32_t* words = static_cast<uint32_t*>(shared);
  float* rest = reinterpret_cast<float*>(words + 2 * filter_words);
  return Teacher{reinterpret_cast<int*>(rest), rest + top, rest + 2 * top, words, words + filter_words};
}
__device__ __forceinline__ int filter_word(int id, int filter_words) { return (id >> 5) & (filter_words - 1); }

// A row's lanes lay out its teacher: softmax over the entries whose class
// lies in the row and whose logit is not -inf.  Returns false when there is none.
// Without kScores the row's scores of the entries are left to load_scores.
template <class T, int kLanes, bool kScores>
__device__ __forceinline__ bool load_teacher(const RowArgs& A, int64_t r, const T* row, int lane, const Teacher& t,
                                             float* ymax, float* sum_q) {
  const int64_t base = r * A.top;
  const float inv_t = (float)A.inv_t;
  for (int i = lane; i < A.filter_words; i += kLanes) t.seen[i] = t.again[i] = 0u;
  float mx = -INFINITY;
  bool nan = false;
  for (int k = lane; k < A.top; k += kLanes) {
    const int64_t id = class_at(A.ids, A.ids_bytes, base + k);
    const float y0 = teacher_at(A.teacher, A.teacher_dtype, base + k);
    const bool real = id >= 0 && id < A.classes && y0 != -INFINITY;
    const float y = real ? y0 : -INFINITY;
    t.ids[k] = real ? (int)id : -1;
    t.q[k] = y;
    if (kScores) t.x[k] = real ? Pack<T>::one(row[id]) : 0.0f;
    mx = fmaxf(mx, y);
    nan |= y != y;
  }
  __syncwarp(lanes_mask<kLanes>());
  mx = lanes_max<kLanes>(mx);
  nan = __any_sync(lanes_mask<kLanes>(), nan);
  if (mx == -INFINITY && !nan) return false;
  float sum = 0.0f;
  for (int k = lane; k < A.top; k += kLanes) {
    const int id = t.ids[k];
    const float e = id >= 0 ? expf((t.q[k] - mx) * inv_t) : 0.0f;
    t.q[k] = e;
    sum += e;
    if (id >= 0) {
      const uint32_t bit = 1u << (id & 31);
      const int word = filter_word(id, A.filter_words);
      if (atomicOr(&t.seen[word], bit) & bit) atomicOr(&t.again[word], bit);
    }
  }
  sum = lanes_sum<kLanes>(sum);
  for (int k = lane; k < A.top; k += kLanes) t.q[k] = t.q[k] / sum;
  __syncwarp(lanes_mask<kLanes>());
  *ymax = mx;
  *sum_q = sum;
  return true;
}

// Where the row has just been added up, they are near: read ahead of it they cost
// 131072 x 2000 bf16, 64 entries, 85 us.
template <class T, int kLanes>
__device__ __forceinline__ void load_scores(const RowArgs& A, const T* row, int lane, const Teacher& t) {
  for (int k = lane; k < A.top; k += kLanes) {
    const int id = t.ids[k];
    t.x[k] = id >= 0 ? Pack<T>::one(row[id]) : 0.0f;
  }
}

// Sum of q over the entries of the class of entry k, added in the entries'
// order (every repeated entry gets the same bits).
__device__ __forceinline__ float class_q(const Teacher& t, int k, int top, int filter_words) {
  const int id = t.ids[k];
  if (!((t.again[filter_word(id, filter_words)] >> (id & 31)) & 1u)) return t.q[k];
  float sum = 0.0f;
  for (int i = 0; i < top; ++i) sum += t.ids[i] == id ? t.q[i] : 0.0f;
  return sum;
}

// ------------------------------------------------------------ a row's end

// log s of a sum of at least 1 that logf would round to 5e-7 (of ten): the exponent's part is added in 64 bits.
__device__ __forceinline__ double log_of(float s) {
  const int e = (__float_as_int(s) >> 23) - 127;
  if (!(s >= 1.0f && e <= 127)) return (double)logf(s);  // NaN, inf, a row without a value
  return fma((double)e, M_LN2, (double)logf(__int_as_float(__float_as_int(s) - (e << 23))));
}

// log of a row's sum.  ex2.approx gives 5.0e-8 too little on average (measured
// on 2^20 arguments in each of [-1, 0], [-4, -2], [-24, -12]) for all but the
// largest value's 2^0, which over the tokens of a sequence would add up; the
// mean is put back.  It is a B200's mean, to be measured again on another chip.  One
// value alone is taken to be the largest: where k values are, the correction is
// 5.0e-8 (k - 1) / s too large, at most the whole 5.0e-8 (all scores equal), which is less
// than half a step of a log-probability below -1.
__device__ __forceinline__ double log_row(float s) {
  return log_of(s) + (double)(5.0e-8f * (1.0f - __frcp_rn(s)));
}

__device__ __forceinline__ float log_prob(float x, const Stat& st) {
  return (float)((double)x - (double)st.m - log_row(st.s));
}

// The lanes' sum over the row's teacher of q (log q - log P), times the weight and T^2.
template <int kLanes>
__device__ __forceinline__ double distill_row(const RowArgs& A, int64_t r, int lane, const Teacher& t, const Stat& st,
                                              float ymax, float sum_q, float w) {
  const double inv_t = A.inv_t, log_s = log_row(st.s), log_q_sum = log_of(sum_q);
  double sum = 0.0;
  for (int k = lane; k < A.top; k += kLanes) {
    const float q = t.q[k];
    if (t.ids[k] < 0 || q == 0.0f) continue;
    const float y = teacher_at(A.teacher, A.teacher_dtype, r * A.top + k);
    const double log_q = ((double)y - (double)ymax) * inv_t - log_q_sum;
    sum += (double)q * (log_q - (((double)t.x[k] - (double)st.m) * inv_t - log_s));
  }
  return (double)w * lanes_sum<kLanes>(sum) * ((double)A.temperature * (double)A.temperature);
}

__device__ __forceinline__ PolicyToken policy_token(const RowArgs& A, int64_t r) {
  return PolicyToken{A.old_lp[r], A.advantages[r], A.ref_lp != nullptr ? A.ref_lp[r] : 0.0f, A.ref_lp != nullptr};
}

__device__ __forceinline__ void store_policy(const RowArgs& A, int64_t r, const PolicyTerm& p, const PolicyToken& t,
                                             double kl, float w) {
  A.row_out[r] = (double)w * policy_value(p, t, A.clip, kl);
  A.row_out[A.rows + r] = (double)w * kl;
  A.row_out[2 * A.rows + r] = p.cut ? (double)w : 0.0;
}

// A row's statistics as a gradient's call finds them; s is inf, which no sum of a
// row is, for a row whose teacher has no entries.
__device__ __forceinline__ float2 saved(const Stat& st, bool real) {
  return make_float2(st.m, real ? st.s : INFINITY);
}

// A row that does not count.
template <int kMode>
__device__ __forceinline__ void store_skipped(const RowArgs& A, int64_t r) {
  if (kMode == kLogProb) A.log_probs[r] = 0.0f;
  if (kMode == kDistill) A.row_out[r] = 0.0;
  if (kMode == kPolicy) A.row_out[r] = A.row_out[A.rows + r] = A.row_out[2 * A.rows + r] = 0.0;
  if (A.stats != nullptr) A.stats[r] = make_float2(0.0f, 1.0f);
}

template <class T>
__device__ __forceinline__ const T* row_at(const RowArgs& A, int64_t r) {
  const T* x = static_cast<const T*>(A.x);
  if (A.inner == A.rows) return x + r * A.inner_stride;  // a 64-bit division takes a hundred instructions
  return x + (r / A.inner) * A.outer_stride + (r % A.inner) * A.inner_stride;
}

__device__ __forceinline__ int target_at(const RowArgs& A, int64_t r) {
  const int64_t t = class_at(A.ids, A.ids_bytes, r);
  return t >= 0 && t < A.classes ? (int)t : -1;
}

// a (p - q) of one chosen class.
template <class T>
__device__ __forceinline__ T chosen_grad(float x, float m, float c, float inv_s, float factor, float q) {
  return Pack<T>::narrow(factor * (exp2_fast((x - m) * c) * inv_s - q));
}

// The gradient of the row's teacher classes in [begin, begin + n), by threads g of `threads`.
template <class T>
__device__ __forceinline__ void write_teacher(const RowArgs& A, const Teacher& t, int g, int threads, float m,
                                              float inv_s, float factor, int begin, int n, T* out) {
  for (int k = g; k < A.top; k += threads) {
    const int id = t.ids[k];
    if (id < begin || id - begin >= n) continue;
    out[id - begin] = chosen_grad<T>(t.x[k], m, A.c, inv_s, factor, class_q(t, k, A.top, A.filter_words));
  }
}

// What a weight of 1 has in the mean, times the upstream gradient.
__device__ __forceinline__ float unit_share(const RowArgs& A) {
  const double total = A.total != nullptr ? *A.total : (double)A.rows;
  return total != 0.0 ? (float)((A.grad_loss != nullptr ? (double)*A.grad_loss : 1.0) / total) : 0.0f;
}

// --------------------------------------------------------------- long rows

// A long row is a CTA's, or in slices a cluster's.  kWarps warps stream it, first
// to add it up and then, from L2, to write its gradient; a warp of its own does
// beside them what the row's end needs: the teacher or the token's scalars, the
// loss, the chosen classes.
//
// What bounds it: HBM, R V values read for a forward, and as many written for a
// gradient; 4.9 instructions and one exponential a value and pass (the units give
// 15 exponentials a clock and SM) stay below that.  Reads alone reach 7.0 TB/s
// here and writes alone 6.2, so it costs nothing that CTAs first read and then
// write.  What costs is the time between the passes, which other CTAs of the SM
// have to fill, and the rows that are between their passes: they have to stay in
// L2 beside the writes.  Measured at 4096 x 128000 bf16 (floors 160 and 320 us):
//   forward, 8 warps x 5 CTAs an SM: 167 us;  8 x 6: 178;  12 x 3: 173;  16 x 2: 186.
//   gradient alone, 12 x 3: 331 us;  8 x 5: 338;  16 x 2: 329.
//   both, slices of 140 KB, 16 x 3: 390 us;  12 x 3: 411;  8 x 5: 453; whole rows
//   of 256 KB, 16 x 3: 443.  Rows of 64 KB (8192 x 32000) 8 x 6: 198;  16 x 3: 213;
//   of 32 KB (16384 x 16000) 8 x 6: 196;  8 x 5: 226;  16 x 3: 264.
// Slower at 4096 x 128000 were: slices held in shared memory between the passes
// (456), persistent CTAs (444), pass 1 of the next row beside pass 2 of this one
// from a ring of bulk copies (408 to 500), both passes as tasks of other CTAs (568).
enum Pass {
  kForward,   // pass 1: statistics and loss
  kBackward,  // pass 2 with statistics from an earlier call
  kStep       // both
};

template <class T, int kMode, int kPass, int kWarps>
__global__ void __launch_bounds__(32 * kWarps + 32, kWarps > 8 ? 3 : kPass == kStep ? 6 : 5)
    long_kernel(const __grid_constant__ RowArgs A) {
  constexpr bool kStats = kPass != kBackward, kGrad = kPass != kForward;
  constexpr int kThreads = 32 * kWarps;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Stat part[kWarps];
  __shared__ Stat rank_stat[kMaxCluster];
  __shared__ float factor_s;
  __shared__ int real_s;
  const int g = threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool helper = warp == kWarps;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t r = (int64_t)blockIdx.x / ranks;
  const T* row = row_at<T>(A, r);
  const int begin = min(A.classes, rank * A.slice), n = min(A.classes - begin, A.slice);
  const T* mine = row + begin;
  T* out = static_cast<T*>(A.grad) + r * A.classes + begin;

  // Rows that do not count: their values are not looked at.
  float w = 1.0f, up = 1.0f;
  int target = -1;
  if (kMode != kLogProb) w = weight_at(A.weights, A.weight_bytes, r);
  if (kMode != kDistill) target = target_at(A, r);
  if (kMode == kLogProb && !kStats) up = A.upstream[r];
  if (kMode != kLogProb ? w == 0.0f : target < 0 || up == 0.0f) {
    if (kGrad && !helper) zero_slice<T, kThreads>(out, n, g);
    if (helper && rank == 0 && lane == 0 && kStats) store_skipped<kMode>(A, r);
    return;  // the whole cluster has the same row
  }
  if (kStats && ranks > 1) cluster.barrier_arrive();  // this CTA has started

  // ---- pass 1; the helper meanwhile fetches what the row's end needs
  const Teacher teacher = kMode == kDistill ? teacher_in(dyn, A.top, A.filter_words) : Teacher{};
  Stat st{-INFINITY, 0.0f};
  float x_target = 0.0f, ymax = 0.0f, sum_q = 0.0f, share = 0.0f;
  PolicyToken token{};
  bool real = true;
  if (kMode == kDistill && !kStats) {
    // The gradient alone is not to wait for the teacher (1021 x 32003 bf16, 64 entries: 37 us, waiting 44).
    if (helper && lane == 0) factor_s = A.temperature * w * unit_share(A);
    __syncthreads();
  }
  if (helper) {
    if (kMode == kDistill) {
      real = load_teacher<T, 32, true>(A, r, row, lane, teacher, &ymax, &sum_q);
      if (kStats && lane == 0) {
        if (kGrad) factor_s = A.temperature * w * unit_share(A);
        real_s = real;
      }
    } else if (target >= 0) {
      x_target = Pack<T>::one(row[target]);
    }
    if (kMode == kPolicy) {
      token = policy_token(A, r);
      share = w * unit_share(A);
    }
  } else if (kStats) {
    st = slice_part<T, kThreads, kGrad>(mine, n, g, A.c);
    st = lanes_merge<32>(st, A.c);
    if (lane == 0) part[warp] = st;
  }
  if (kStats) {
    __syncthreads();
    st = lanes_merge<32>(lane < kWarps ? part[lane] : Stat{-INFINITY, 0.0f}, A.c);
    if (ranks > 1) {
      cluster.barrier_wait();  // every CTA has started: its shared memory may be written
      if (warp == 0 && lane < ranks) *cluster.map_shared_rank(&rank_stat[rank], lane) = st;
      cluster.sync();
      st = lanes_merge<32>(lane < ranks ? rank_stat[lane] : Stat{-INFINITY, 0.0f}, A.c);
    }
  } else {
    const float2 v = A.stats[r];
    st = Stat{v.x, v.y};
  }

  // ---- the row's end
  if (kMode == kPolicy) {
    // The writing warps wait for the slope: its two exponentials take a lane each and the
    // time of one, and the value comes after (4099 x 64000 bf16: 186 us; one after the
    // other by one lane 195).
    PolicyTerm t{};
    float lp = 0.0f;
    if (helper) {
      if (target >= 0) lp = log_prob(x_target, st);
      const double e = exp(lane & 1 ? (double)token.ref_lp - (double)lp : (double)lp - (double)token.old_lp);
      const double exp_d = __shfl_sync(0xffffffffu, e, 1);
      t = policy_term(token, A.clip, __shfl_sync(0xffffffffu, e, 0), token.has_ref ? exp_d - 1.0 : 0.0);
      if (lane == 0) factor_s = (float)(-(double)share * t.slope);
    }
    __syncthreads();
    if (helper && lane == 0 && rank == 0) store_policy(A, r, t, token, policy_kl(lp, token).kl, w);
  }
  if (helper && kStats && rank == 0) {
    if (A.stats != nullptr && lane == 0) A.stats[r] = saved(st, real);
    if (kMode == kLogProb && lane == 0) A.log_probs[r] = log_prob(x_target, st);
    if (kMode == kDistill) {
      const double loss = real ? distill_row<32>(A, r, lane, teacher, st, ymax, sum_q, w) : 0.0;
      if (lane == 0) A.row_out[r] = loss;
    }
  }
  if (!kGrad) return;

  // ---- pass 2
  const float factor = kMode == kLogProb ? -up : factor_s, inv_s = 1.0f / st.s;
  const bool writes = kMode != kDistill ? target >= 0 : kStats ? real_s != 0 : st.s != INFINITY;
  if (!helper) {
    if (writes)
      write_slice<T, kThreads, kStats>(mine, out, n, g, st.m, A.c, factor * inv_s);
    else
      zero_slice<T, kThreads>(out, n, g);
  }
  if (!writes) return;
  __syncthreads();  // the row's a p is written before the chosen classes are written again
  if (!helper) return;
  if (kMode == kDistill)
    write_teacher(A, teacher, lane, 32, st.m, inv_s, factor, begin, n, out);
  else if (lane == 0 && target >= begin && target - begin < n)
    out[target - begin] = chosen_grad<T>(x_target, st.m, A.c, inv_s, factor, 1.0f);
}

// -------------------------------------------------------------- whole rows

// Many rows: each group of kGroup threads has whole rows, one after the other.
// kA: pass 1 (statistics and loss), kB: pass 2 (the gradient).  What a row's end
// needs of memory is loaded while the row before it is worked on.  Short rows
// are bound by the instructions of a row's end (some 300 a warp), so as few
// threads as keep the SMs full share one: with 8 lanes a row instead of 32 the
// forward of 131072 x 2000 bf16 takes 103 us instead of 151 (floor 80).
template <int kGroup>
constexpr int cta_threads() {
  return kGroup <= 32 ? 256 : kGroup;
}
// On an SM.  More writing streams are slower (gradient of 65536 x 4000 bf16: 178 us,
// with 1536 threads some 25 % more), and a teacher's row takes registers (its loss and gradient,
// 64 entries: 318 us, with 1024 threads 378).
template <int kMode, bool kA, bool kB>
constexpr int resident_threads() {
  return !kB ? 1536 : kMode == kDistill && kA ? 768 : 1024;
}

template <class T, int kMode, int kGroup, bool kA, bool kB>
__global__ void __launch_bounds__(cta_threads<kGroup>(), resident_threads<kMode, kA, kB>() / cta_threads<kGroup>())
    rows_kernel(const __grid_constant__ RowArgs A) {
  constexpr int kThreads = cta_threads<kGroup>(), kGroups = kThreads / kGroup, kWarps = kThreads / 32;
  constexpr int kLanes = kGroup < 32 ? kGroup : 32;
  constexpr bool kCta = kGroup > 32;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Stat part[2][kWarps];
  __shared__ float factor_s[2];
  __shared__ int real_s[2];
  const int g = threadIdx.x % kGroup, lane = threadIdx.x % kLanes, group = threadIdx.x / kGroup;
  const bool leader = !kCta || threadIdx.x < 32;  // the lanes that do a row's small work
  const int64_t step = (int64_t)gridDim.x * kGroups;
  int64_t r = (int64_t)blockIdx.x * kGroups + group;
  if (r >= A.rows) return;
  const int n = A.classes;

  // What a row's end needs of memory, loaded while the row before it is worked on.
  struct Ahead {
    float w, up;
    int target;
    bool counts;
  };
  auto look = [&](int64_t i) {
    Ahead h{1.0f, 1.0f, -1, false};
    if (i >= A.rows) return h;
    if (kMode != kLogProb) h.w = weight_at(A.weights, A.weight_bytes, i);
    if (kMode != kDistill) h.target = target_at(A, i);
    if (kMode == kLogProb && !kA) h.up = A.upstream[i];
    h.counts = kMode != kLogProb ? h.w != 0.0f : h.target >= 0 && h.up != 0.0f;
    return h;
  };
  auto teacher_of = [&](int buf) {
    return teacher_in(dyn + (2 * group + buf) * A.teacher_bytes, A.top, A.filter_words);
  };
  struct Begun {  // a row whose end is near
    float x_target, ymax, sum_q;
    bool real;
    Stat st;
  };
  auto begin = [&](int64_t i, const Ahead& h, int buf) {
    Begun b{0.0f, 0.0f, 0.0f, true, Stat{-INFINITY, 0.0f}};
    if (!h.counts) return b;
    const T* row = row_at<T>(A, i);
    if (kMode != kDistill) {
      b.real = h.target >= 0;
      if (leader && b.real) b.x_target = Pack<T>::one(row[h.target]);
    } else if (leader) {
      __syncwarp(lanes_mask<kLanes>());  // the row that had this buffer is done with it
      b.real = load_teacher<T, kLanes, !kA>(A, i, row, lane, teacher_of(buf), &b.ymax, &b.sum_q);
      if (kCta && lane == 0) real_s[buf] = b.real;
    }
    if (!kA) {
      const float2 v = A.stats[i];
      b.st = Stat{v.x, v.y};
    }
    return b;
  };

  const float unit = kB && kMode != kLogProb ? unit_share(A) : 0.0f;
  int buf = 0;
  Ahead now = look(r), next = look(r + step);
  Begun row = begin(r, now, 0);
  if (kA && now.counts) row.st = slice_part<T, kGroup, kB>(row_at<T>(A, r), n, g, A.c);
  if (kA) {
    row.st = lanes_merge<kLanes>(row.st, A.c);
    if (kCta && lane == 0) part[0][threadIdx.x >> 5] = row.st;
  }
  if (kCta) __syncthreads();
  for (;;) {
    // ---- the row's end
    float factor = 0.0f;
    if (now.counts) {
      if (kA && kCta) row.st = lanes_merge<32>(lane < kWarps ? part[buf][lane] : Stat{-INFINITY, 0.0f}, A.c);
      if (kCta && kMode == kDistill) row.real = real_s[buf] != 0;
      if (kA && A.stats != nullptr && g == 0) A.stats[r] = saved(row.st, kMode != kDistill || row.real);
      if (kMode == kLogProb) {
        if (kA && g == 0) A.log_probs[r] = log_prob(row.x_target, row.st);
        factor = -now.up;
      } else if (kMode == kDistill) {
        if (kA && leader) {
          if (row.real) load_scores<T, kLanes>(A, row_at<T>(A, r), lane, teacher_of(buf));
          const double loss =
              row.real ? distill_row<kLanes>(A, r, lane, teacher_of(buf), row.st, row.ymax, row.sum_q, now.w) : 0.0;
          if (lane == 0) A.row_out[r] = loss;
        }
        if (kB) factor = A.temperature * now.w * unit;
      } else {
        if (g == 0) {
          const float lp = row.real ? log_prob(row.x_target, row.st) : 0.0f;
          const PolicyToken token = policy_token(A, r);
          const PolicyKl k = policy_kl(lp, token);
          const PolicyTerm t = policy_term(token, A.clip, exp((double)lp - (double)token.old_lp), k.rise);
          store_policy(A, r, t, token, k.kl, now.w);
          factor = (float)(-(double)(now.w * unit) * t.slope);
          if (kCta) factor_s[buf] = factor;
        }
        if (!kCta) factor = __shfl_sync(lanes_mask<kLanes>(), factor, 0, kLanes);
      }
    } else if (kA && g == 0) {
      store_skipped<kMode>(A, r);
    }
    if (kMode == kPolicy && kCta) {
      __syncthreads();
      factor = factor_s[buf];
    }

    // ---- pass 2 of this row, pass 1 of the next
    const int64_t rn = r + step;
    const Ahead after = look(rn + step);
    Begun begun = begin(rn, next, buf ^ 1);
    const bool writes = kB && now.counts && row.real;
    const float inv_s = 1.0f / row.st.s;
    if (kB) {
      const T* x = row_at<T>(A, r);
      T* out = static_cast<T*>(A.grad) + r * n;
      if (!writes) zero_slice<T, kGroup>(out, n, g);
      if (writes) write_slice<T, kGroup, kA>(x, out, n, g, row.st.m, A.c, factor * inv_s);
      if (kA && next.counts) begun.st = slice_part<T, kGroup, kB>(row_at<T>(A, rn), n, g, A.c);
    } else if (next.counts) {
      begun.st = slice_part<T, kGroup, kB>(row_at<T>(A, rn), n, g, A.c);
    }
    if (kA) {
      begun.st = lanes_merge<kLanes>(begun.st, A.c);
      if (kCta && lane == 0) part[buf ^ 1][threadIdx.x >> 5] = begun.st;
    }
    group_sync<kGroup>();  // the parts; this row's a p, before its chosen classes are written again
    if (writes && leader) {
      T* out = static_cast<T*>(A.grad) + r * n;
      if (kMode == kDistill)
        write_teacher(A, teacher_of(buf), lane, kLanes, row.st.m, inv_s, factor, 0, n, out);
      else if (lane == 0)
        out[now.target] = chosen_grad<T>(row.x_target, row.st.m, A.c, inv_s, factor, 1.0f);
    }
    if (rn >= A.rows) return;
    r = rn;
    now = next;
    next = after;
    row = begun;
    buf ^= 1;
  }
}

// ------------------------------------------------------------------ launches

template <class T, int kMode, int kPass, int kWarps>
int launch_long(cudaStream_t s, const RowArgs& a, int cluster, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(a.rows * cluster));
  cfg.blockDim = dim3(32 * kWarps + 32);
  cfg.dynamicSmemBytes = a.teacher_bytes;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B2_CUDA_OR_RETURN(cudaLaunchKernelEx(&cfg, long_kernel<T, kMode, kPass, kWarps>, a));
  return check_launch(s, what);
}

template <class T, int kMode, int kGroup, bool kA, bool kB>
int launch_groups(cudaStream_t s, const RowArgs& a, int per_sm, const DeviceInfo* d, const char* what) {
  static SmemOptIn opt;
  auto kernel = rows_kernel<T, kMode, kGroup, kA, kB>;
  constexpr int groups = cta_threads<kGroup>() / kGroup;
  const int smem = 2 * groups * a.teacher_bytes;
  if (smem > 40 * 1024) B2_RETURN_IF_ERROR(opt.ensure(reinterpret_cast<const void*>(kernel), d->device, smem));
  const int64_t need = ceil_div(a.rows, groups), most = (int64_t)persistent_ctas(d) * per_sm;
  kernel<<<(unsigned)(need < most ? need : most), cta_threads<kGroup>(), smem, s>>>(a);
  return check_launch(s, what);
}

constexpr int64_t kLongRow = 16 * 1024;     // bytes; shorter rows end too often for long_kernel
constexpr int64_t kSliceBytes = 140 * 1024;  // of a row that is read twice, see long_kernel
constexpr int64_t kWideSlice = 96 * 1024;    // from here 16 warps and not 8
// Bytes of a teacher (256 entries) that a row of rows_kernel may have.  With more
// its warp is what the CTA waits for: 65536 x 4000 bf16, 1024 entries, takes 6.0 ms
// there and 2.5 as CTAs with a warp for it.
constexpr int kFewEntries = 4096;

// kA: pass 1 (statistics and loss), kB: pass 2 (gradient).
template <class T, int kMode, bool kA, bool kB>
int launch_rows_as(cudaStream_t s, RowArgs a, const DeviceInfo* d, const char* what) {
  const int64_t sms = d->sm_count;
  constexpr int resident = resident_threads<kMode, kA, kB>();
  if (kMode == kDistill) {
    // 32 bits an entry, so that few entries look repeated without being it: 8192 x 32000
    // bf16, 1024 entries, takes 534 us, with 4 bits an entry 1192.
    a.filter_words = 4;
    while (a.filter_words < (a.top > 256 ? 512 : 128) && a.filter_words < a.top) a.filter_words *= 2;
    a.teacher_bytes = (int)ceil_div(4 * (2 * a.filter_words + 3 * a.top), 16) * 16;
  }
  const bool fill8 = a.rows * 8 >= sms * resident, fill32 = a.rows * 32 >= sms * resident;
  // Forward alone: lanes of a warp keep up to rows of 16384 values, when there are twice as many as run at once.
  if (!kB && a.classes > 4096 && a.classes <= 16384 && a.rows * 32 >= 2 * sms * resident &&
      a.teacher_bytes <= kFewEntries)
    return launch_groups<T, kMode, 32, kA, kB>(s, a, resident / 256, d, what);
  if (a.classes >= kLongRow / (int64_t)sizeof(T) || (a.rows <= 2 * sms && a.classes >= 4096) ||
      a.teacher_bytes > kFewEntries) {
    // A cluster for a row whose slice L2 would not keep, and, for few rows, while
    // there are fewer CTAs than SMs and a slice keeps 2048 values.
    auto slice_of = [&](int ctas) { return ceil_div(ceil_div((int64_t)a.classes, ctas), 8) * 8; };
    int ctas = 1;
    while (ctas < kMaxCluster && ((kA && kB && slice_of(ctas) * (int64_t)sizeof(T) > kSliceBytes) ||
                                  (a.rows * ctas <= sms && slice_of(2 * ctas) >= 2048)))
      ctas *= 2;
    a.slice = (int)slice_of(ctas);
    if constexpr (!kA) return launch_long<T, kMode, kBackward, 12>(s, a, ctas, what);
    if constexpr (!kB) return launch_long<T, kMode, kForward, 8>(s, a, ctas, what);
    if constexpr (kA && kB) {
      if (slice_of(ctas) * (int64_t)sizeof(T) > kWideSlice) return launch_long<T, kMode, kStep, 16>(s, a, ctas, what);
      return launch_long<T, kMode, kStep, 8>(s, a, ctas, what);
    }
  }
  // As few threads a row as keep the SMs full; where each writes, 8 lanes' 128
  // bytes a row are too small a piece of longer rows.
  if (a.classes <= (!kB ? 4096 : kA ? 2048 : 1024) && fill8 && a.teacher_bytes <= 640)
    return launch_groups<T, kMode, 8, kA, kB>(s, a, resident / 256, d, what);
  if ((a.classes <= 1024 || (fill32 && a.classes <= 8192)) && a.teacher_bytes <= kFewEntries)
    return launch_groups<T, kMode, 32, kA, kB>(s, a, resident / 256, d, what);
  return launch_groups<T, kMode, 256, kA, kB>(s, a, resident / 256, d, what);
}

template <class T>
int launch_rows_of(cudaStream_t s, const RowArgs& a, Mode mode, bool stats, bool grad, const DeviceInfo* d,
                   const char* what) {
  if (mode == kPolicy) return launch_rows_as<T, kPolicy, true, true>(s, a, d, what);
  if (mode == kLogProb)
    return stats ? launch_rows_as<T, kLogProb, true, false>(s, a, d, what)
                 : launch_rows_as<T, kLogProb, false, true>(s, a, d, what);
  if (!stats) return launch_rows_as<T, kDistill, false, true>(s, a, d, what);
  return grad ? launch_rows_as<T, kDistill, true, true>(s, a, d, what)
              : launch_rows_as<T, kDistill, true, false>(s, a, d, what);
}

}  // namespace
}  // namespace b2
