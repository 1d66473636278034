// Sparse teachers: the k largest logits of each row with the row's log-sum-exp,
// and the distillation loss from such rows, forward and backward.
#include "vocab_rows.h"

namespace ts {

constexpr int kTopMax = 256;                   // entries a row may keep
constexpr int64_t kTopTailVocab = 1 << 20;     // the kept entries are marked in LDS, a bit per vocabulary entry
constexpr int64_t kTopSelfCountRows = 8192;    // up to this many rows every workgroup counts the mask itself

// ---- the k largest logits --------------------------------------------------------

// Order of logits as unsigned numbers: -inf < ... < -0 = +0 < ... < +inf < NaN.
__device__ __forceinline__ uint32_t top_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = x == 0.f ? 0u : __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Number of the row's elements for which f holds.
template <typename T, int NT, typename F>
__device__ __forceinline__ int top_count(const T* row, int64_t V, int* lds, F f) {
  int c = 0;
  for (int64_t i = threadIdx.x; i < V; i += NT) c += f(to_f32(row[i]), (int)i) ? 1 : 0;
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) c += __shfl_xor(c, off, kWave);
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = c;
  __syncthreads();
  c = 0;
#pragma unroll
  for (int i = 0; i < NT / kWave; ++i) c += lds[i];
  return c;
}

// The logit of an order number (-inf for what lies below it).
__device__ __forceinline__ float top_unkey(uint32_t key) {
  if (key <= 0x007fffffu) return -__builtin_inff();
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

constexpr int kTopCand = 2304;  // candidates a row may have: all of a row that 64 threads hold, and more

template <int NT>
struct TopShared {
  union {
    uint32_t group[2 * NT];  // order numbers of the groups' maxima
    uint64_t kept[kTopMax];
  };
  uint64_t cand[kTopCand];  // order number and place, larger for smaller places
  RowSum sums[NT / kWave];
  VocabStat stats[NT / kWave];
  int counts[NT / kWave];
  int n;
  float bar;
};

// Every thread's rank among n candidates; the first k leave.
template <typename T, int NT>
__device__ __forceinline__ void top_emit(const uint64_t* cand, int n, const T* x, int64_t row, int k,
                                         T* __restrict__ values, int32_t* __restrict__ indices) {
  for (int c = threadIdx.x; c < n; c += NT) {
    const uint64_t me = cand[c];
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += cand[i] > me;
    if (rank < k) {
      const int32_t i = (int32_t)~(uint32_t)me;
      indices[row * k + rank] = i;
      values[row * k + rank] = x[i];
    }
  }
}

// Rows with a NaN, with a sum that needs the true maximum, or with more
// candidates than fit (thousands of equal logits at the border).  The k-th
// largest order number is found bit by bit (the largest t such that at least k
// elements reach it), then the place up to which elements equal to it are
// taken, likewise; the k elements so defined are collected.
template <typename T, int NT>
__device__ __forceinline__ void top_row_walked(const VocabRows& a, int64_t row, const T* x, int k,
                                               T* __restrict__ values, int32_t* __restrict__ indices,
                                               float* __restrict__ lse, TopShared<NT>& sh) {
  const int64_t V = a.V;
  if (lse) {
    const VocabStat s = vstat_block<NT / kWave>(vocab_stat_walk<T, NT>(x, V, a.k), a.k, sh.stats);
    if (threadIdx.x == 0) lse[row] = (float)((double)s.m * a.inv_T + kVrLn2 * vstat_log2z(s, a.k_rel));
  }
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    if (top_count<T, NT>(x, V, sh.counts, [=](float v, int) { return top_key(v) >= c; }) >= k) t = c;
  }
  const int above = top_count<T, NT>(x, V, sh.counts, [=](float v, int) { return top_key(v) > t; });
  int place = 0;  // the largest place such that fewer than k - above elements equal to t lie before it
  for (int bit = 30; bit >= 0; --bit) {
    const int c = place | (1 << bit);
    if (c < V &&
        top_count<T, NT>(x, V, sh.counts, [=](float v, int i) { return i < c && top_key(v) == t; }) < k - above)
      place = c;
  }
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < V; i += NT) {
    const uint32_t key = top_key(to_f32(x[i]));
    if (key > t || (key == t && i <= place)) {
      const int at = atomicAdd(&sh.n, 1);
      if (at < kTopMax) sh.cand[at] = ((uint64_t)key << 32) | (uint32_t)~(uint32_t)i;
    }
  }
  __syncthreads();
  top_emit<T, NT>(sh.cand, k, x, row, k, values, indices);
}

// Reduces n > k candidates to the k largest.
template <int NT>
__device__ __forceinline__ void top_refine(TopShared<NT>& sh, int n, int k) {
  uint64_t t = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t c = t | (1ull << bit);
    int m = 0;
    for (int i = threadIdx.x; i < n; i += NT) m += sh.cand[i] >= c;
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) m += __shfl_xor(m, off, kWave);
    __syncthreads();
    if (threadIdx.x % kWave == 0) sh.counts[threadIdx.x / kWave] = m;
    __syncthreads();
    m = 0;
    for (int i = 0; i < NT / kWave; ++i) m += sh.counts[i];
    if (m >= k) t = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT)
    if (sh.cand[i] >= t) {
      const int at = atomicAdd(&sh.n, 1);
      if (at < kTopMax) sh.kept[at] = sh.cand[i];  // (places differ, so exactly k reach t)
    }
  __syncthreads();
  for (int i = threadIdx.x; i < k; i += NT) sh.cand[i] = sh.kept[i];
  __syncthreads();
}

// One pass over a row by one workgroup, in pieces of NT * KREG vectors.  The
// first piece gives a bar: the threads' maxima (two each when k is large) are
// maxima of disjoint groups, so the k-th largest of them is reached by at least
// k elements.  Every element that reaches the bar is a candidate -- few more
// than k, since the best k mostly lie in different groups (k = 64 of 512
// groups: 68 expected) -- and the candidates' ranks are counted.  The row's sum
// is taken in the same walk over the registers.
template <typename T, int NT, int KREG>
__global__ __launch_bounds__(NT) void top_logits_kernel(const VocabRows a, int k, T* __restrict__ values,
                                                        int32_t* __restrict__ indices, float* __restrict__ lse) {
  constexpr int VEC = Vec16<T>::N;
  __shared__ TopShared<NT> sh;
  const int64_t row = blockIdx.x, V = a.V;
  const T* x = vocab_row<T>(a, row);
  const VocabGeom g = vocab_geom(x, V);
  const float kk = a.k;
  const int tid = threadIdx.x;
  const bool two = k > NT / 4;  // two groups per thread
  RowRegs<T, NT, KREG> r;
  regs_load(r, x, V, g);
  if (tid == 0) sh.n = 0;
  const float c = regs_anchor(r, g, kk);
  float z = 0.f, s_a = 0.f, m0 = fmaxf(r.h, r.t), m1 = -__builtin_inff();
  auto add = [&](float xv) {
    const float d = fmaf(xv, kk, c), e = fast_exp2(d);
    z += e;
    s_a = fmaf(e, fmaxf(d, -1e30f), s_a);
  };
  if (tid < kWave) {
    add(r.h);
    add(r.t);
  }
  float bar = 0.f;
  for (int64_t v0 = 0;; v0 += NT * KREG) {
#pragma unroll
    for (int j = 0; j < KREG; ++j) {
      if (v0 + tid + j * NT < g.nvec) {
        forget(r.v[j]);
        float m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xv = to_f32(r.v[j].v[i]);
          add(xv);
          m = fmaxf(m, xv);
        }
        if (j < KREG / 2)
          m0 = fmaxf(m0, m);
        else
          m1 = fmaxf(m1, m);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (v0 == 0) {
      sh.group[tid] = top_key(two ? m0 : fmaxf(m0, m1));
      if (two) sh.group[NT + tid] = top_key(m1);
      __syncthreads();
      if (tid < kWave) {
        const int n = two ? 2 * NT : NT;
        uint32_t key[2 * NT / kWave];
#pragma unroll
        for (int i = 0; i < 2 * NT / kWave; ++i) key[i] = i * kWave < n ? sh.group[i * kWave + tid] : 0u;
        uint32_t t = 0;
        const int enough = k + k / 8 + 4;
        for (int bit = 31; bit >= 0; --bit) {
          const uint32_t cnd = t | (1u << bit);
          int cnt = 0;
#pragma unroll
          for (int i = 0; i < 2 * NT / kWave; ++i) cnt += (int)__popcll(__ballot(key[i] >= cnd));
          if (cnt >= k) {
            t = cnd;
            if (cnt <= enough) break;
          }
        }
        if (tid == 0) sh.bar = top_unkey(t);
      }
      __syncthreads();
      bar = sh.bar;
    }
    // candidates among the registers (and the end elements, with the first piece)
    auto take = [&](float xv, int64_t i) {
      if (xv >= bar) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < kTopCand) sh.cand[at] = ((uint64_t)top_key(xv) << 32) | (uint32_t)~(uint32_t)i;
      }
    };
    if (v0 == 0) {
      if (tid < g.head) take(r.h, tid);
      if (g.tail0 + tid < V) take(r.t, g.tail0 + tid);
    }
    if (fmaxf(m0, m1) >= bar) {
#pragma unroll
      for (int j = 0; j < KREG; ++j) {
        const int64_t v = v0 + tid + j * NT;
        if (v < g.nvec) {
          forget(r.v[j]);
#pragma unroll
          for (int i = 0; i < VEC; ++i) take(to_f32(r.v[j].v[i]), g.head + v * VEC + i);
        }
      }
    }
    if (v0 + NT * KREG >= g.nvec) break;
#pragma unroll
    for (int j = 0; j < KREG; ++j) {
      const int64_t v = v0 + NT * KREG + tid + j * NT;
      if (v < g.nvec) r.v[j] = load16_stream(x + g.head + v * VEC);
    }
    m0 = m1 = -__builtin_inff();
    __syncthreads();
    const int n = sh.n;
    __syncthreads();  // (nobody adds to it before everybody has read it)
    if (n > kTopCand / 2) {  // room for the next piece's
      if (n > kTopCand) break;
      top_refine<NT>(sh, n, k);
    }
  }
  const RowSum s = rowsum_block<NT / kWave, kSumMean>(c, z, s_a, sh.sums);
  __syncthreads();
  int n = sh.n;
  if (!s.ok || n > kTopCand) {
    __syncthreads();
    top_row_walked<T, NT>(a, row, x, k, values, indices, lse, sh);
    return;
  }
  if (tid == 0 && lse) lse[row] = -rowsum_log_prob<true>(a, s, 0.f).hi;  // the log probability of a logit of 0
  if (n > 2 * kTopMax) {
    __syncthreads();
    top_refine<NT>(sh, n, k);
    n = k;
  }
  top_emit<T, NT>(sh.cand, n, x, row, k, values, indices);
}

// ---- distillation from a teacher's largest logits ----------------------------------

struct TopDistilArgs {
  VocabRows r;
  const void* t_values;
  int t_dtype;
  const int32_t* t_indices;
  const float* t_lse;  // null: the kept entries' probabilities are normalised among themselves
  int k;
  const uint8_t* mask;  // may be null
  const int* live;      // number of rows of the mask, or null: counted by every workgroup
  float gscale;         // weight * T
  double* row_loss;
  void* grad;  // may be null
};

__device__ __forceinline__ float top_value(const void* v, int dtype, int64_t i) {
  if (dtype == TS_F32) return reinterpret_cast<const float*>(v)[i];
  if (dtype == TS_BF16) return to_f32(reinterpret_cast<const bf16_t*>(v)[i]);
  return to_f32(reinterpret_cast<const f16_t*>(v)[i]);
}

// The teacher's entries of a row, NE a thread, and what the row's terms need of
// them.  Probabilities are taken in 64 bits: what the teacher leaves to all other
// tokens is one minus their sum.
template <int NE>
struct TopEntries {
  int idx[NE];  // -1: absent
  float x[NE];  // the student's logit
  double lp[NE], p[NE];
  float p_all[NE];  // of all entries that name this token
  bool first[NE];   // the first to name it
};

template <int NT>
struct TopDistilShared {
  int idx[kTopMax];
  float p[kTopMax];
  RowSum sums[NT / kWave];
  VocabStat stats[NT / kWave];
  double d[NT / kWave];
  float f[NT / kWave];
  float go;  // factor of the other tokens' probabilities
  double P;
};

template <int NT, int NE>
__device__ __forceinline__ double top_entry_probs(const TopDistilArgs& a, int64_t row, TopEntries<NE>& e, float (&v)[NE],
                                                  TopDistilShared<NT>& sh) {
  constexpr int NW = NT / kWave;
  double sum = 0.0;
  if (a.t_lse) {
    const double lse = (double)a.t_lse[row];
#pragma unroll
    for (int i = 0; i < NE; ++i) e.lp[i] = (double)v[i] * a.r.inv_T - lse;
  } else {
    float m = kVrLowest;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (e.idx[i] >= 0) m = fmaxf(m, v[i]);
    m = wave_max(m);
    if (NW > 1) {
      if (threadIdx.x % kWave == 0) sh.f[threadIdx.x / kWave] = m;
      __syncthreads();
      m = sh.f[threadIdx.x % NW];
#pragma unroll
      for (int off = NW / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
    }
    double z = 0.0;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      e.lp[i] = ((double)v[i] - (double)m) * a.r.inv_T;
      if (e.idx[i] >= 0) z += exp(e.lp[i]);
    }
    const double lz = log(block_sum_f64<NW>(z, sh.d));
#pragma unroll
    for (int i = 0; i < NE; ++i) e.lp[i] -= lz;
  }
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    e.p[i] = 0.0;
    if (e.idx[i] >= 0 && v[i] != -__builtin_inff()) e.p[i] = exp(e.lp[i]);
    sum += e.p[i];
  }
  return block_sum_f64<NW>(sum, sh.d);
}

// Bit of element j in the marks: vector v of the row owns bits 8 + v * VEC on, so
// that a vector's marks are one byte (or half of one).
__device__ __forceinline__ uint32_t top_mark_bit(int j, const VocabGeom& g) { return (uint32_t)(j - g.head + 8); }

// KREG = 0: the row is walked for its sums and again for its gradient.
template <typename T, int NT, int KREG, bool TAIL>
__global__ __launch_bounds__(NT) void top_distil_kernel(const TopDistilArgs a) {
  constexpr int NW = NT / kWave, NE = (kTopMax + NT - 1) / NT, VEC = Vec16<T>::N;
  extern __shared__ uint32_t marks[];  // TAIL: a bit per vocabulary entry
  __shared__ TopDistilShared<NT> sh;
  const int64_t row = blockIdx.x, V = a.r.V;
  const int tid = threadIdx.x, k = a.k;
  T* grow = a.grad ? reinterpret_cast<T*>(a.grad) + row * V : nullptr;
  if (a.mask && a.mask[row] == 0) {
    if (tid == 0) a.row_loss[row] = 0.0;
    if (grow) vocab_zero_row<T, NT>(grow, V);
    return;
  }
  const T* x = vocab_row<T>(a.r, row);
  const VocabGeom g = vocab_geom(x, V);
  RowRegs<T, NT, KREG ? KREG : 1> r;
  if constexpr (KREG > 0) regs_load(r, x, V, g);

  TopEntries<NE> e;
  float v[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int at = tid + i * NT;
    e.idx[i] = -1;
    e.x[i] = 0.f;
    v[i] = 0.f;
    if (at < k) {
      const int j = a.t_indices[row * k + at];
      if (j >= 0 && j < V) {
        e.idx[i] = j;
        e.x[i] = to_f32(x[j]);
        v[i] = top_value(a.t_values, a.t_dtype, row * k + at);
      }
    }
  }
  if (TAIL)
    for (int64_t i = tid; i < (V + 8 + 31) / 32; i += NT) marks[i] = 0u;
  const double p_sum = top_entry_probs<NT, NE>(a, row, e, v, sh);
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int at = tid + i * NT;
    if (at < kTopMax) {
      sh.idx[at] = e.idx[i];
      sh.p[at] = (float)e.p[i];
    }
  }
  __syncthreads();
  // the same token named twice: the first naming stands for all of them
  double distinct = 0.0;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    e.first[i] = e.idx[i] >= 0;
    e.p_all[i] = 0.f;
    if (e.idx[i] >= 0) {
      const int at = tid + i * NT;
      for (int q = 0; q < k; ++q) {
        const bool same = sh.idx[q] == e.idx[i];
        e.first[i] = e.first[i] && !(same && q < at);
        e.p_all[i] += same ? sh.p[q] : 0.f;
      }
      if (TAIL) {
        const uint32_t bit = top_mark_bit(e.idx[i], g);
        atomicOr(&marks[bit >> 5], 1u << (bit & 31));
      }
      distinct += e.first[i] ? 1.0 : 0.0;
    }
  }
  const float n_live = a.live ? (float)*a.live
                              : a.mask ? mask_count_block<NT>(a.mask, a.r.n_rows, sh.f) : (float)a.r.n_rows;
  const bool covered = TAIL && block_sum_f64<NW>(distinct, sh.d) == (double)V;
  __syncthreads();
  const float gs = a.gscale / n_live, kk = a.r.k;

  // Loss and gradient factors from the student's sums: lq(x) = ln of its probability of a logit x, and
  // with TAIL the part q_rest of its probability that lies outside the kept entries.
  auto finish = [&](auto lq, double lq_rest, double inv_q_rest) {
    double term = 0.0;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (e.idx[i] >= 0 && !(e.p[i] == 0.0)) term += e.p[i] * (e.lp[i] - lq(e.x[i]));
    term = block_sum_f64<NW>(term, sh.d);
    if (tid == 0) {
      double P = p_sum, outside = p_sum;
      if (TAIL) {
        const double rest = covered ? 0.0 : fmax(1.0 - p_sum, 0.0);
        P += rest;
        outside = P;
        if (rest > 0.0) {
          term += rest * (log(rest) - lq_rest);
          if (inv_q_rest < __builtin_inf()) outside -= rest * inv_q_rest;
        }
      }
      a.row_loss[row] = term;
      sh.go = (float)((double)gs * outside);
      sh.P = P;
    }
    __syncthreads();
  };
  auto patch = [&](auto q_of) {  // the kept entries' gradients replace what the walk over the row wrote
    __syncthreads();
    const float P = (float)sh.P;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (e.first[i]) grow[e.idx[i]] = from_f32<T>(gs * (q_of(e.x[i]) * P - e.p_all[i]));
  };

  if constexpr (KREG > 0) {
    RowSum s;
    if (TAIL) {
      const float c = regs_anchor(r, g, kk);
      float out = 0.f, in = 0.f;
      const uint8_t* mark8 = reinterpret_cast<const uint8_t*>(marks);
      auto marked = [&](uint32_t bit) { return ((marks[bit >> 5] >> (bit & 31)) & 1u) != 0; };
      if (tid < g.head && !marked(top_mark_bit(tid, g))) out += fast_exp2(fmaf(r.h, kk, c));
      if (g.tail0 + tid < V && !marked(top_mark_bit((int)g.tail0 + tid, g))) out += fast_exp2(fmaf(r.t, kk, c));
#pragma unroll
      for (int j = 0; j < KREG; ++j) {
        const int vv = tid + j * NT;
        if (vv < (int)g.nvec) {
          forget(r.v[j]);
          const uint32_t bit0 = 8u + (uint32_t)vv * VEC;
          const uint32_t m = mark8[bit0 >> 3] >> (bit0 & 7u);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float ex = fast_exp2(fmaf(to_f32(r.v[j].v[i]), kk, c));
            out += (m >> i) & 1u ? 0.f : ex;
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (e.first[i]) in += fast_exp2(fmaf(e.x[i], kk, c));
      // (a wavefront of nothing but -inf has no exponent of its own to take entries by)
      if (!(c < kVrNoTerm) && in > 0.f) in = __builtin_inff();
      s = rowsum_block<NW, kSumSecond>(c, out, in, sh.sums);
      s.ok = s.ok && (covered || s.z > 1e-30f);
    } else {
      s = regs_sum<T, NT, KREG>(r, g, kk, sh.sums);
    }
    if (s.ok) {
      const float rest_z = s.z;
      if (TAIL) s.z += s.a;
      double lq_rest = 0.0, inv_q_rest = 0.0;
      if (TAIL && !covered) {
        const Float2x lo = log2_2x(rest_z), la = log2_2x(s.z);
        lq_rest = kVrLn2 * (((double)lo.hi - (double)la.hi) + ((double)lo.lo - (double)la.lo));
        inv_q_rest = (double)s.z / (double)rest_z;
      }
      finish(
          [&](float xv) {
            const Float2x l = rowsum_log_prob<false>(a.r, s, xv);
            return (double)l.hi + (double)l.lo;
          },
          lq_rest, inv_q_rest);
      if (!grow) return;
      const float rz = 1.f / s.z, go = sh.go * rz, c = s.c;
      regs_map(r, g, x, grow, V, -1, [=](float xv) { return go * fast_exp2(fmaf(xv, kk, c)); }, [](float) { return 0.f; });
      patch([&](float xv) { return fast_exp2(fmaf(xv, kk, c)) * rz; });
      return;
    }
    __syncthreads();
  }
  VocabStat out = vstat_init(), all;
  if (TAIL) {
    for (int64_t i = tid; i < V; i += NT) {
      const uint32_t bit = top_mark_bit((int)i, g);
      if ((marks[bit >> 5] >> (bit & 31)) & 1u) continue;
      float x1[1] = {to_f32(x[i])};
      vstat_fold<1>(out, x1, kk);
    }
    out = vstat_block<NW>(out, kk, sh.stats);
    VocabStat in = vstat_init();
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (e.first[i]) {
        float x1[1] = {e.x[i]};
        vstat_fold<1>(in, x1, kk);
      }
    all = vstat_merge(out, vstat_block<NW>(in, kk, sh.stats), kk);
  } else {
    all = vstat_block<NW>(vocab_stat_walk<T, NT>(x, V, kk), kk, sh.stats);
  }
  const double log2z = vstat_log2z(all, a.r.k_rel);
  const double lq_rest =
      TAIL ? ((double)out.m - (double)all.m) * a.r.inv_T + kVrLn2 * (vstat_log2z(out, a.r.k_rel) - log2z) : 0.0;
  finish([&](float xv) { return ((double)xv - (double)all.m) * a.r.inv_T - kVrLn2 * log2z; }, lq_rest, exp(-lq_rest));
  if (!grow) return;
  const float rz = 1.f / all.z, go = sh.go * rz, m = all.m;
  vocab_map_walk<T, NT>(x, grow, V, [=](float xv, int) { return go * fast_exp2((xv - m) * kk); });
  patch([&](float xv) { return fast_exp2((xv - m) * kk) * rz; });
}

__global__ __launch_bounds__(1024) void top_distil_sum_kernel(const double* __restrict__ v, int64_t n,
                                                              const uint8_t* __restrict__ mask, double scale,
                                                              float* __restrict__ out) {
  __shared__ double lds[1024 / kWave];
  __shared__ float lds_f[1024 / kWave];
  const float live = mask ? mask_count_block<1024>(mask, n, lds_f) : (float)n;
  const double s = block_sum_f64<1024 / kWave>(thread_share_of_sum_f64<1024>(v, n), lds);
  if (threadIdx.x == 0) *out = live > 0.f ? (float)(scale * s / (double)live) : __builtin_nanf("");
}

__global__ __launch_bounds__(1024) void top_live_kernel(const uint8_t* __restrict__ mask, int64_t n, int* __restrict__ out) {
  __shared__ float lds[1024 / kWave];
  const float live = mask_count_block<1024>(mask, n, lds);
  if (threadIdx.x == 0) *out = (int)live;
}

template <typename T>
int launch_top_logits(const VocabRows& a, int k, void* values, int32_t* indices, float* lse, hipStream_t st) {
  const RowShape sh = row_shape<T>(a.V);
  T* out = reinterpret_cast<T*>(values);
  const dim3 grid((unsigned)a.n_rows);
  if (sh.nt == 64)
    hipLaunchKernelGGL((top_logits_kernel<T, 64, 4>), grid, dim3(64), 0, st, a, k, out, indices, lse);
  else if (sh.nt == 256)
    hipLaunchKernelGGL((top_logits_kernel<T, 256, 4>), grid, dim3(256), 0, st, a, k, out, indices, lse);
  else
    hipLaunchKernelGGL((top_logits_kernel<T, 512, 8>), grid, dim3(512), 0, st, a, k, out, indices, lse);
  return check_launch();
}

template <typename T, int NT, int KREG, bool TAIL>
int launch_top_distil_rows(const TopDistilArgs& a, hipStream_t st) {
  const size_t marks = TAIL ? (size_t)((a.r.V + 8 + 31) / 32) * 4 : 0;
  if (marks > 32768) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&top_distil_kernel<T, NT, KREG, TAIL>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)marks);
    if (e != hipSuccess) {
      set_last_hip_error((int)e);
      return TS_ERR_LAUNCH;
    }
  }
  hipLaunchKernelGGL((top_distil_kernel<T, NT, KREG, TAIL>), dim3((unsigned)a.r.n_rows), dim3(NT), marks, st, a);
  return check_launch();
}

template <typename T, bool TAIL>
int launch_top_distil_shape(const TopDistilArgs& a, hipStream_t st) {
  const RowShape sh = row_shape<T>(a.r.V);
  if (sh.nt == 64) return launch_top_distil_rows<T, 64, 4, TAIL>(a, st);
  if (sh.nt == 256) return launch_top_distil_rows<T, 256, 4, TAIL>(a, st);
  if (sh.nt == 512) return launch_top_distil_rows<T, 512, 8, TAIL>(a, st);
  if (sh.kreg == 8) return launch_top_distil_rows<T, 1024, 8, TAIL>(a, st);
  if (sh.kreg == 16) return launch_top_distil_rows<T, 1024, 16, TAIL>(a, st);
  return launch_top_distil_rows<T, 1024, 0, TAIL>(a, st);
}

template <typename T>
int launch_top_distil(TopDistilArgs a, int* live, double loss_scale, float* loss_out, hipStream_t st) {
  int rc = TS_OK;
  if (a.mask && a.r.n_rows > kTopSelfCountRows) {
    hipLaunchKernelGGL(top_live_kernel, dim3(1), dim3(1024), 0, st, a.mask, a.r.n_rows, live);
    rc = check_launch();
    if (rc) return rc;
    a.live = live;
  }
  if (a.r.n_rows > 0) rc = a.t_lse ? launch_top_distil_shape<T, true>(a, st) : launch_top_distil_shape<T, false>(a, st);
  if (rc) return rc;
  hipLaunchKernelGGL(top_distil_sum_kernel, dim3(1), dim3(1024), 0, st, a.row_loss, a.r.n_rows, a.mask, loss_scale,
                     loss_out);
  return check_launch();
}

}  // namespace ts

extern "C" {

int ts_top_logits(const void* s, int64_t n_seq, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok, int k,
                  double temperature, void* values, int32_t* indices, float* logsumexp, int dtype,
                  ts_stream_t stream) {
  const int rc = ts::vocab_rows_status(s, n_seq, seq_len, V, ld_seq, ld_tok, temperature, dtype);
  if (rc) return rc;
  if (k < 1 || k > V) return TS_ERR_ARG;
  if (k > ts::kTopMax) return TS_ERR_RANGE;
  if (n_seq * seq_len == 0) return TS_OK;
  if (!values || !indices) return TS_ERR_ARG;
  if (((uintptr_t)values & (dtype == TS_F32 ? 3u : 1u)) || (((uintptr_t)indices | (uintptr_t)logsumexp) & 3u))
    return TS_ERR_ALIGN;
  const ts::VocabRows a = ts::vocab_rows(s, n_seq * seq_len, seq_len, V, ld_seq, ld_tok, temperature);
  hipStream_t st = (hipStream_t)stream;
  TS_BY_DTYPE(dtype, (ts::launch_top_logits<T>(a, k, values, indices, logsumexp, st)))
}

size_t ts_top_distil_workspace_bytes(int64_t n_rows) { return n_rows < 0 ? 0 : 16 + (size_t)n_rows * 8; }

int ts_top_distil_fwd_bwd(const void* s, int64_t n_seq, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok,
                          const void* t_values, int t_dtype, const int32_t* t_indices, const float* t_logsumexp, int k,
                          const uint8_t* row_mask, double temperature, double weight, void* workspace, float* loss_out,
                          void* grad, int dtype, ts_stream_t stream) {
  const int rc = ts::vocab_rows_status(s, n_seq, seq_len, V, ld_seq, ld_tok, temperature, dtype);
  if (rc) return rc;
  if (t_dtype != TS_F32 && t_dtype != TS_BF16 && t_dtype != TS_F16) return TS_ERR_ARG;
  if (k < 1 || !workspace || !loss_out) return TS_ERR_ARG;
  if (k > ts::kTopMax || (t_logsumexp && V > ts::kTopTailVocab)) return TS_ERR_RANGE;
  if (n_seq * seq_len > 0 && (!t_values || !t_indices)) return TS_ERR_ARG;
  if (((uintptr_t)t_values & (t_dtype == TS_F32 ? 3u : 1u)) || ((uintptr_t)grad & (dtype == TS_F32 ? 3u : 1u)) ||
      (((uintptr_t)t_indices | (uintptr_t)t_logsumexp | (uintptr_t)loss_out) & 3u) || ((uintptr_t)workspace & 15u))
    return TS_ERR_ALIGN;
  ts::TopDistilArgs a;
  a.r = ts::vocab_rows(s, n_seq * seq_len, seq_len, V, ld_seq, ld_tok, temperature);
  a.t_values = t_values;
  a.t_dtype = t_dtype;
  a.t_indices = t_indices;
  a.t_lse = t_logsumexp;
  a.k = k;
  a.mask = row_mask;
  a.gscale = (float)(weight * temperature);
  a.live = nullptr;
  a.row_loss = reinterpret_cast<double*>((char*)workspace + 16);
  a.grad = grad;
  const double scale = weight * temperature * temperature;
  hipStream_t st = (hipStream_t)stream;
  TS_BY_DTYPE(dtype, (ts::launch_top_distil<T>(a, reinterpret_cast<int*>(workspace), scale, loss_out, st)))
}

}  // extern "C"
