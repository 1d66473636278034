// Rows of vocabulary logits as the token losses and the top-logit kernels read
// them: where a row lies, its soft-max statistics, and the walk over a row that
// may start and end anywhere.
#pragma once

#include "common.h"

namespace ts {

constexpr float kVrLog2e = 1.4426950408889634f;
constexpr double kVrLn2 = 0.69314718055994530942;
constexpr float kVrLowest = -3.402823466e38f;  // stand-in for -inf: keeps differences from it free of inf - inf

// Row r is token r % seq_len of sequence r / seq_len: sequences lie ld_seq
// elements apart and tokens ld_tok, so that a slice of every sequence (the
// logits without their last position, say) is read where it lies.
struct VocabRows {
  const void* s;
  int64_t n_rows, seq_len, V, ld_seq, ld_tok;
  // 2^(x k) = e^(x / T); k is log2(e) / T rounded to fp32 and k_rel what the
  // rounding took, relative: (log2(e) / T - k) / k.  Every exponent of a row is
  // off by that same factor, which would add up over a sequence of rows, so the
  // log-sum-exp is corrected for it to first order.
  float k, k_rel;
  double inv_T;
};

inline VocabRows vocab_rows(const void* s, int64_t n_rows, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok,
                            double temperature) {
  VocabRows a;
  a.s = s;
  a.n_rows = n_rows;
  a.seq_len = seq_len;
  a.V = V;
  a.ld_seq = ld_seq;
  a.ld_tok = ld_tok;
  const double k = 1.4426950408889634074 / temperature;
  a.k = (float)k;
  a.k_rel = (float)((k - (double)a.k) / (double)a.k);
  a.inv_T = 1.0 / temperature;
  return a;
}

// Status of the geometry arguments every entry point on such rows takes.
inline int vocab_rows_status(const void* s, int64_t n_seq, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok,
                             double temperature, int dtype) {
  if (dtype != TS_F32 && dtype != TS_BF16 && dtype != TS_F16) return TS_ERR_ARG;
  if (n_seq < 0 || seq_len < 0 || V <= 0 || ld_seq < 0 || ld_tok < 0) return TS_ERR_ARG;
  // the factor log2(e) / T has to be a normal fp32 number
  if (!(temperature >= 1e-30 && temperature <= 1e30)) return TS_ERR_ARG;
  if (V > 0x7fffffffLL - 64) return TS_ERR_RANGE;
  // a grid of one workgroup of up to 1024 threads per row stays below 2^32 threads
  if (n_seq >= (1 << 22) || seq_len >= (1 << 22) || n_seq * seq_len >= (1 << 22)) return TS_ERR_RANGE;
  if (n_seq * seq_len > 0 && !s) return TS_ERR_ARG;
  if ((uintptr_t)s & (dtype == TS_F32 ? 3u : 1u)) return TS_ERR_ALIGN;
  return TS_OK;
}

template <typename T>
__device__ __forceinline__ const T* vocab_row(const VocabRows& a, int64_t row) {
  const int64_t q = row / a.seq_len;
  return reinterpret_cast<const T*>(a.s) + q * a.ld_seq + (row - q * a.seq_len) * a.ld_tok;
}

// m = max x, z = sum 2^((x - m) k), a = sum 2^((x - m) k) (x - m) k
struct VocabStat {
  float m, z, a;
};

__device__ __forceinline__ VocabStat vstat_init() { return VocabStat{kVrLowest, 0.f, 0.f}; }

// The state re-based onto the larger maximum m.
__device__ __forceinline__ VocabStat vstat_rebase(VocabStat s, float m, float k) {
  const float d = fmaxf((s.m - m) * k, -1e30f);  // finite, so that an empty state stays 0 and not 0 * inf
  const float r = fast_exp2(d);
  return VocabStat{m, s.z * r, r * fmaf(s.z, d, s.a)};
}

__device__ __forceinline__ VocabStat vstat_merge(VocabStat p, VocabStat q, float k) {
  const float m = fmaxf(p.m, q.m);
  p = vstat_rebase(p, m, k);
  q = vstat_rebase(q, m, k);
  return VocabStat{m, p.z + q.z, p.a + q.a};
}

// Adds one logit to sums whose maximum is settled.  A NaN logit makes z NaN; a
// logit of -inf (a masked vocabulary entry) adds nothing, also not to a.
__device__ __forceinline__ void vstat_add(VocabStat& s, float x, float k) {
  const float d = (x - s.m) * k;
  const float e = fast_exp2(d);
  s.z += e;
  s.a = fmaf(e, fmaxf(d, -1e30f), s.a);
}

template <int N>
__device__ __forceinline__ void vstat_fold(VocabStat& s, const float (&x)[N], float k) {
  float m = s.m;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
  if (m > s.m) s = vstat_rebase(s, m, k);
#pragma unroll
  for (int i = 0; i < N; ++i) vstat_add(s, x[i], k);
}

// Merged over a workgroup of NW wavefronts; every thread gets the result.
template <int NW>
__device__ __forceinline__ VocabStat vstat_block(VocabStat s, float k, VocabStat* lds) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1)
    s = vstat_merge(s, VocabStat{__shfl_xor(s.m, off, kWave), __shfl_xor(s.z, off, kWave), __shfl_xor(s.a, off, kWave)}, k);
  if (NW == 1) return s;
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = s;
  __syncthreads();
  s = lds[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) s = vstat_merge(s, lds[i], k);
  __syncthreads();  // lds may be used again
  return s;
}

// log2 of the row's sum of 2^((x - m) k_exact), in 64 bits; -inf for a row of nothing but -inf.
__device__ __forceinline__ double vstat_log2z(const VocabStat& s, float k_rel) {
  if (s.z == 0.f) return -__builtin_inf();
  return log2((double)s.z) + (double)k_rel * ((double)s.a / (double)s.z);
}

// ln of the soft-max probability of a logit x of the row.
__device__ __forceinline__ double vstat_log_prob(const VocabRows& a, const VocabStat& s, float x) {
  return ((double)x - (double)s.m) * a.inv_T - kVrLn2 * vstat_log2z(s, a.k_rel);
}

// Split of a row into scalar head, 16-byte vectors and scalar tail.
struct VocabGeom {
  int head;
  int64_t nvec, tail0;
};

template <typename T>
__device__ __forceinline__ VocabGeom vocab_geom(const T* row, int64_t V) {
  constexpr int VEC = Vec16<T>::N;
  VocabGeom g;
  g.head = (int)(((16u - (uint32_t)((uintptr_t)row & 15u)) & 15u) / sizeof(T));
  if (g.head > V) g.head = (int)V;
  g.nvec = (V - g.head) / VEC;
  g.tail0 = g.head + g.nvec * VEC;
  return g;
}

// This thread's share of the row's statistics when NT threads walk it.
template <typename T, int NT>
__device__ __forceinline__ VocabStat vocab_stat_walk(const T* row, int64_t V, float k) {
  constexpr int VEC = Vec16<T>::N;
  const VocabGeom g = vocab_geom(row, V);
  VocabStat s = vstat_init();
  float x1[1];
  if ((int)threadIdx.x < g.head) {
    x1[0] = to_f32(row[threadIdx.x]);
    vstat_fold<1>(s, x1, k);
  }
  if (g.tail0 + threadIdx.x < V) {
    x1[0] = to_f32(row[g.tail0 + threadIdx.x]);
    vstat_fold<1>(s, x1, k);
  }
  for (int64_t v = threadIdx.x; v < g.nvec; v += NT) {
    const Vec16<T> r = load16(row + g.head + v * VEC);
    float x[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = to_f32(r.v[i]);
    vstat_fold<VEC>(s, x, k);
  }
  return s;
}

// grad[j] = f(x[j], j) over a row; the gradient row may be aligned differently.
template <typename T, int NT, typename F>
__device__ __forceinline__ void vocab_map_walk(const T* row, T* grow, int64_t V, F f) {
  constexpr int VEC = Vec16<T>::N;
  const VocabGeom g = vocab_geom(row, V);
  if ((int)threadIdx.x < g.head) grow[threadIdx.x] = from_f32<T>(f(to_f32(row[threadIdx.x]), (int)threadIdx.x));
  const int64_t t = g.tail0 + threadIdx.x;
  if (t < V) grow[t] = from_f32<T>(f(to_f32(row[t]), (int)t));
  const bool gvec = (((uintptr_t)grow ^ (uintptr_t)row) & 15u) == 0;
  for (int64_t v = threadIdx.x; v < g.nvec; v += NT) {
    const int64_t e0 = g.head + v * VEC;
    const Vec16<T> r = load16(row + e0);
    Vec16<T> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(f(to_f32(r.v[i]), (int)(e0 + i)));
    if (gvec) {
      store16(grow + e0, o);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) grow[e0 + i] = o.v[i];
    }
  }
}

template <typename T, int NT>
__device__ __forceinline__ void vocab_zero_row(T* grow, int64_t V) {
  constexpr int VEC = Vec16<T>::N;
  const VocabGeom g = vocab_geom(grow, V);
  const T zero = from_f32<T>(0.f);
  if ((int)threadIdx.x < g.head) grow[threadIdx.x] = zero;
  if (g.tail0 + threadIdx.x < V) grow[g.tail0 + threadIdx.x] = zero;
  Vec16<T> z;
#pragma unroll
  for (int i = 0; i < VEC; ++i) z.v[i] = zero;
  for (int64_t v = threadIdx.x; v < g.nvec; v += NT) store16(grow + g.head + v * VEC, z);
}

// Sum of doubles over a workgroup of NW wavefronts, in a fixed order; every
// thread gets the result.
template <int NW>
__device__ __forceinline__ double block_sum_f64(double v, double* lds) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  if (NW == 1) return v;
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int i = 0; i < NW; ++i) r += lds[i];
  return r;
}

}  // namespace ts

// return call with T bound to the storage type of a dtype code
#define TS_BY_DTYPE(dtype, call)                         \
  switch (dtype) {                                       \
    case TS_F32: { using T = float; return call; }       \
    case TS_BF16: { using T = ts::bf16_t; return call; } \
    default: { using T = ts::f16_t; return call; }       \
  }
