// Sparse teachers: the k largest logits of each row with the row's log-sum-exp,
// and the distillation loss from such rows, forward and backward.
#include "vocab_rows.h"

namespace ts {

constexpr int kTopBlock = 256;
constexpr int kTopMax = 256;                   // entries a row may keep
constexpr int64_t kTopTailVocab = 1 << 20;     // the kept entries are marked in LDS, a bit per vocabulary entry

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

// One workgroup per row.  The k-th largest order number is found bit by bit
// (the largest t such that at least k elements reach it), then the place up to
// which elements equal to it are taken, likewise; the k elements so defined are
// collected and each one's rank counted.
template <typename T>
__global__ __launch_bounds__(kTopBlock) void top_logits_kernel(const VocabRows a, int k, T* __restrict__ values,
                                                               int32_t* __restrict__ indices,
                                                               float* __restrict__ lse) {
  __shared__ VocabStat lds_s[kTopBlock / kWave];
  __shared__ int lds_c[kTopBlock / kWave];
  __shared__ uint64_t cand[kTopMax];
  __shared__ int n_cand;
  const int64_t row = blockIdx.x;
  const T* x = vocab_row<T>(a, row);
  const int64_t V = a.V;
  if (lse) {
    const VocabStat s = vstat_block<kTopBlock / kWave>(vocab_stat_walk<T, kTopBlock>(x, V, a.k), a.k, lds_s);
    if (threadIdx.x == 0) lse[row] = (float)((double)s.m * a.inv_T + kVrLn2 * vstat_log2z(s, a.k_rel));
  }
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    if (top_count<T, kTopBlock>(x, V, lds_c, [=](float v, int) { return top_key(v) >= c; }) >= k) t = c;
  }
  const int above = top_count<T, kTopBlock>(x, V, lds_c, [=](float v, int) { return top_key(v) > t; });
  int place = 0;  // the largest place such that fewer than k - above elements equal to t lie before it
  for (int bit = 30; bit >= 0; --bit) {
    const int c = place | (1 << bit);
    if (c < V &&
        top_count<T, kTopBlock>(x, V, lds_c, [=](float v, int i) { return i < c && top_key(v) == t; }) < k - above)
      place = c;
  }
  if (threadIdx.x == 0) n_cand = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < V; i += kTopBlock) {
    const uint32_t key = top_key(to_f32(x[i]));
    if (key > t || (key == t && i <= place)) {
      const int at = atomicAdd(&n_cand, 1);
      if (at < kTopMax) cand[at] = ((uint64_t)key << 32) | (uint32_t)~(uint32_t)i;
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < k) {
    const uint64_t me = cand[threadIdx.x];
    int rank = 0;
    for (int i = 0; i < k; ++i) rank += cand[i] > me;
    const int32_t i = (int32_t)~(uint32_t)me;
    indices[row * k + rank] = i;
    values[row * k + rank] = x[i];
  }
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
  float gscale;         // weight * T
  double* row_loss;
  void* grad;  // may be null
};

__device__ __forceinline__ float top_value(const void* v, int dtype, int64_t i) {
  if (dtype == TS_F32) return reinterpret_cast<const float*>(v)[i];
  if (dtype == TS_BF16) return to_f32(reinterpret_cast<const bf16_t*>(v)[i]);
  return to_f32(reinterpret_cast<const f16_t*>(v)[i]);
}

template <typename T, bool TAIL>
__global__ __launch_bounds__(kTopBlock) void top_distil_kernel(const TopDistilArgs a) {
  constexpr int NW = kTopBlock / kWave;
  extern __shared__ uint32_t marks[];  // TAIL: a bit per vocabulary entry
  __shared__ VocabStat lds_s[NW];
  __shared__ double lds_d[NW];
  __shared__ float lds_f[NW];
  __shared__ int ent_idx[kTopMax];
  __shared__ float ent_p[kTopMax];
  const int64_t row = blockIdx.x, V = a.r.V;
  const int tid = threadIdx.x, k = a.k;
  T* grow = a.grad ? reinterpret_cast<T*>(a.grad) + row * V : nullptr;
  if (a.mask && a.mask[row] == 0) {
    if (tid == 0) a.row_loss[row] = 0.0;
    if (grow) vocab_zero_row<T, kTopBlock>(grow, V);
    return;
  }
  const T* x = vocab_row<T>(a.r, row);
  const float n_live = a.mask ? mask_count_block<kTopBlock>(a.mask, a.r.n_rows, lds_f) : (float)a.r.n_rows;

  // the teacher's entries, one a thread, probabilities in 64 bits
  int idx = -1;
  float v = kVrLowest;
  bool in = false;
  if (tid < k) {
    idx = a.t_indices[row * k + tid];
    in = idx >= 0 && idx < V;
    if (in) v = top_value(a.t_values, a.t_dtype, row * k + tid);
  }
  double lp;  // ln p
  if (TAIL) {
    lp = (double)v * a.r.inv_T - (double)a.t_lse[row];
  } else {
    VocabStat e = vstat_init();
    if (in) e.m = fmaxf(e.m, v);
    const float m = vstat_block<NW>(e, a.r.k, lds_s).m;
    lp = ((double)v - (double)m) * a.r.inv_T;
    const double z = block_sum_f64<NW>(in ? exp(lp) : 0.0, lds_d);
    lp -= log(z);
  }
  double p = in ? exp(lp) : 0.0;
  if (in && v == -__builtin_inff()) p = 0.0;
  ent_idx[tid] = in ? idx : -1;
  ent_p[tid] = (float)p;
  if (TAIL)
    for (int64_t i = tid; i < (V + 31) / 32; i += kTopBlock) marks[i] = 0u;
  __syncthreads();
  // the same token named twice: the first naming stands for all of them
  bool first = in;
  float p_all = 0.f;
  if (in) {
    for (int i = 0; i < k; ++i) {
      const bool same = ent_idx[i] == idx;
      first = first && !(same && i < tid);
      p_all += same ? ent_p[i] : 0.f;
    }
    if (TAIL) atomicOr(&marks[idx >> 5], 1u << (idx & 31));
  }
  const double p_sum = block_sum_f64<NW>(p, lds_d);
  const double distinct = block_sum_f64<NW>(first ? 1.0 : 0.0, lds_d);

  // the student's statistics; with TAIL those outside the kept entries apart
  VocabStat out, all;
  const float xi = in ? to_f32(x[idx]) : 0.f;
  if (TAIL) {
    out = vstat_init();
    for (int64_t i = tid; i < V; i += kTopBlock) {
      if ((marks[i >> 5] >> (i & 31)) & 1u) continue;
      float x1[1] = {to_f32(x[i])};
      vstat_fold<1>(out, x1, a.r.k);
    }
    out = vstat_block<NW>(out, a.r.k, lds_s);
    VocabStat e = vstat_init();
    if (first) {
      float x1[1] = {xi};
      vstat_fold<1>(e, x1, a.r.k);
    }
    all = vstat_merge(out, vstat_block<NW>(e, a.r.k, lds_s), a.r.k);
  } else {
    all = vstat_block<NW>(vocab_stat_walk<T, kTopBlock>(x, V, a.r.k), a.r.k, lds_s);
  }

  // the row's loss
  const double log2z = vstat_log2z(all, a.r.k_rel);
  const double lq = ((double)xi - (double)all.m) * a.r.inv_T - kVrLn2 * log2z;
  double term = block_sum_f64<NW>(p > 0.0 || p != p ? p * (lp - lq) : 0.0, lds_d);
  double P = p_sum, outside = 1.0;
  if (TAIL) {
    // what the teacher leaves to all other tokens against what the student leaves to them
    const double rest = distinct == (double)V ? 0.0 : fmax(1.0 - p_sum, 0.0);
    P += rest;
    outside = P;
    if (rest > 0.0) {
      const double lq_rest =
          ((double)out.m - (double)all.m) * a.r.inv_T + kVrLn2 * (vstat_log2z(out, a.r.k_rel) - log2z);
      term += out.z > 0.f || out.z != out.z ? rest * (log(rest) - lq_rest) : __builtin_inf();
      if (out.z > 0.f) outside = P - rest * exp(-lq_rest);
    }
  } else {
    outside = P;
  }
  if (tid == 0) a.row_loss[row] = term;
  if (!grow) return;
  const float g = a.gscale / n_live, rz = 1.f / all.z;
  const float go = (float)((double)g * outside) * rz, m = all.m, kk = a.r.k;
  vocab_map_walk<T, kTopBlock>(x, grow, V, [=](float xv, int) { return go * fast_exp2((xv - m) * kk); });
  __syncthreads();  // the kept entries' gradients replace what the walk wrote
  if (first) grow[idx] = from_f32<T>(g * (fast_exp2((xi - m) * kk) * rz * (float)P - p_all));
}

__global__ __launch_bounds__(1024) void top_distil_sum_kernel(const double* __restrict__ v, int64_t n,
                                                              const uint8_t* __restrict__ mask, double scale,
                                                              float* __restrict__ out) {
  __shared__ double lds[1024 / kWave];
  __shared__ float lds_f[1024 / kWave];
  const float live = mask ? mask_count_block<1024>(mask, n, lds_f) : (float)n;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += v[i];
  s = block_sum_f64<1024 / kWave>(s, lds);
  if (threadIdx.x == 0) *out = live > 0.f ? (float)(scale * s / (double)live) : __builtin_nanf("");
}

template <typename T>
int launch_top_logits(const VocabRows& a, int k, void* values, int32_t* indices, float* lse, hipStream_t st) {
  hipLaunchKernelGGL((top_logits_kernel<T>), dim3((unsigned)a.n_rows), dim3(kTopBlock), 0, st, a, k,
                     reinterpret_cast<T*>(values), indices, lse);
  return check_launch();
}

template <typename T>
int launch_top_distil(const TopDistilArgs& a, double loss_scale, float* loss_out, hipStream_t st) {
  if (a.r.n_rows > 0) {
    if (a.t_lse) {
      const size_t marks = (size_t)((a.r.V + 31) / 32) * 4;
      const void* fn = reinterpret_cast<const void*>(&top_distil_kernel<T, true>);
      if (marks > 32768) {
        const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)marks);
        if (e != hipSuccess) {
          set_last_hip_error((int)e);
          return TS_ERR_LAUNCH;
        }
      }
      hipLaunchKernelGGL((top_distil_kernel<T, true>), dim3((unsigned)a.r.n_rows), dim3(kTopBlock), marks, st, a);
    } else {
      hipLaunchKernelGGL((top_distil_kernel<T, false>), dim3((unsigned)a.r.n_rows), dim3(kTopBlock), 0, st, a);
    }
    const int rc = check_launch();
    if (rc) return rc;
  }
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
  a.row_loss = reinterpret_cast<double*>(workspace);
  a.grad = grad;
  const double scale = weight * temperature * temperature;
  hipStream_t st = (hipStream_t)stream;
  TS_BY_DTYPE(dtype, (ts::launch_top_distil<T>(a, scale, loss_out, st)))
}

}  // extern "C"
