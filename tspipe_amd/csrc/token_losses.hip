// Losses on the log probabilities of sampled tokens, forward and backward:
//   token log probability   ln softmax(s / T)[label] per row, and its gradient,
//   preference loss         paired log ratios against a reference model,
//   clipped policy loss     probability ratios against the sampling policy,
//                           clipped, with a KL term against a reference model.
// All three come down to d loss / d s = c (onehot(label) - softmax(s / T)) / T
// with one factor c per row; they differ in where c comes from: the caller, the
// sums over both sequences of a pair, or the row itself.
#include "vocab_rows.h"

namespace ts {

constexpr int kTokBlock = 256;

// Which rows count, and for which token.
struct TokenRows {
  VocabRows r;
  const int64_t* labels;
  const uint8_t* mask;  // may be null (all rows)
  int64_t ignore_index;
};

// `scalar`: the row is the same in every lane.
template <bool scalar>
__device__ __forceinline__ bool token_live(const TokenRows& a, int64_t row, int64_t* label) {
  const int64_t l = scalar ? scalar_load(a.labels + row) : a.labels[row];
  *label = l;
  return l != a.ignore_index && l >= 0 && l < a.r.V && (!a.mask || a.mask[row] != 0);
}

// ---- token log probabilities ------------------------------------------------
// stats[row] = (c, z): the row's sum z of 2^(x k + c), or (m, -z) with z the sum
// of 2^((x - m) k) where that sum over- or underflows.

// d loss / d x from a row's stats and its factor c / T.
struct TokenGrad {
  float k, off, cz, c;
  bool by_max;
  __device__ __forceinline__ TokenGrad(float k_, float2 st, float c_) {
    k = k_;
    off = st.x;
    by_max = !(st.y > 0.f);
    cz = c_ / fabsf(st.y);
    c = c_;
  }
  __device__ __forceinline__ float prob_c(float x) const {  // c * probability
    return cz * fast_exp2(by_max ? (x - off) * k : fmaf(x, k, off));
  }
  __device__ __forceinline__ float other(float x) const { return -prob_c(x); }
  __device__ __forceinline__ float label(float x) const { return c - prob_c(x); }
};

// One workgroup per row, all of whose loads are in flight before the first sum:
// ln p = ln2 (x_label k + c - log2 z), z = sum 2^(x k + c).  Beside z it takes the
// sum of terms times exponents, the row's mean of x k, by which ln p is corrected
// for the rounding of k.  An element costs six vector instructions, one of them a
// quarter-rate exponential, which is about what its two bytes take to arrive:
// 2044 x 50257 bf16 36 us (5.1 TB/s), 5735 x 32000 bf16 62 us (5.9).
//
// log_ratio (optional): the log probability minus ref[row] in 64 bits, for the
// sums over whole sequences.  The threads' sums are joined and the logarithm is
// taken in 64 bits as well (the row's registers are free by then): a sequence's
// sum of differences to a reference that nearly agrees shows every unit of fp32.
// Rows longer than NT * KREG vectors are walked in pieces of that size.  Eight
// wavefronts a SIMD: 64 registers, which fit (without the bound one type or the
// other takes 67 to 71, and one workgroup fewer is resident).
template <typename T, int NT, int KREG>
__global__ __launch_bounds__(NT, KREG > 4 ? 8 : 1) void token_stat_kernel(const TokenRows a, const float* __restrict__ ref,
                                                        float* __restrict__ logp, double* __restrict__ log_ratio,
                                                        float2* __restrict__ stats, unsigned* __restrict__ ticket) {
  if (ticket && blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0u;  // of the next kernel
  constexpr int VEC = Vec16<T>::N;
  constexpr int NW = NT / kWave;
  __shared__ double lds_z[NW];
  __shared__ float lds_c[NW], lds_a[NW];
  __shared__ VocabStat lds_v[NW];
  const int64_t row = blockIdx.x;
  int64_t label;
  if (!token_live<true>(a, row, &label)) {
    if (threadIdx.x == 0) {
      if (logp) logp[row] = 0.f;
      if (log_ratio) log_ratio[row] = 0.0;
      if (stats) stats[row] = make_float2(0.f, 1.f);
    }
    return;
  }
  const T* srow = vocab_row<T>(a.r, row);
  const int64_t V = a.r.V;
  const float k = a.r.k;
  const VocabGeom g = vocab_geom(srow, V);
  const T label_logit = srow[label];
  RowRegs<T, NT, KREG> r;
  regs_load(r, srow, V, g);
  float c = regs_anchor<true>(r, g, k), z = 0.f, s_a = 0.f;
  auto add = [&](float x) {
    const float d = fmaf(x, k, c), e = fast_exp2(d);
    z += e;
    s_a = fmaf(e, fmaxf(d, -1e30f), s_a);
  };
  if (threadIdx.x < kWave) {
    add(r.h());
    add(r.t());
  }
  regs_each(r, g, add);
  float before = 0.f;  // sum over earlier pieces
  for (int64_t v0 = NT * KREG; v0 < g.nvec; v0 += NT * KREG) {
    const int left = g.nvec - v0 < NT * KREG ? (int)(g.nvec - v0) : NT * KREG;
    const VecBuffer piece = vec_buffer(srow + g.head + v0 * VEC, left);
#pragma unroll
    for (int j = 0; j < KREG; ++j) r.v[j] = vec_load<T>(piece, threadIdx.x + j * NT);
    const float shift = regs_raise(r, left, k, c);
    s_a = __builtin_amdgcn_ldexpf(fmaf(before + z, shift, s_a), (int)shift);
    long_carry(before, z, (int)shift);
#pragma unroll
    for (int j = 0; j < KREG; ++j) {
      if ((int)threadIdx.x + j * NT < left) {
        forget(r.v[j]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) add(to_f32(r.v[j].v[i]));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  double sum = wave_sum_f64((double)before + (double)z);
  s_a = wave_sum(s_a);
  if (NW > 1) {  // (as rowsum_put and rowsum_get do it; s_a = sum of terms times their exponents)
    if (threadIdx.x % kWave == 0) {
      lds_z[threadIdx.x / kWave] = sum;
      lds_c[threadIdx.x / kWave] = c;
      lds_a[threadIdx.x / kWave] = s_a;
    }
    __syncthreads();
    const int w = threadIdx.x % NW;
    const float wc = lds_c[w], wz = (float)lds_z[w];
    c = wc;
#pragma unroll
    for (int off = NW / 2; off > 0; off >>= 1) c = fminf(c, __shfl_xor(c, off, kWave));
    const float d = c - wc;
    const int shift = (int)fmaxf(d, -1000.f);
    sum = __builtin_amdgcn_ldexp(lds_z[w], shift);
    s_a = __builtin_amdgcn_ldexpf(fmaf(wz, d, lds_a[w]), shift);
#pragma unroll
    for (int off = NW / 2; off > 0; off >>= 1) {
      sum += __shfl_xor(sum, off, kWave);
      s_a += __shfl_xor(s_a, off, kWave);
    }
  }
  z = (float)sum;
  const float x = to_f32(label_logit);
  double lp;
  float2 st;
  if (z > 1e-30f && z < __builtin_inff() && c < kVrNoTerm) {  // uniform
    if (threadIdx.x != 0) return;
    const double xk = (double)x * (double)k, mean = (double)(s_a / z) - (double)c;  // mean of x k under the soft-max
    lp = x == -__builtin_inff() ? (double)x : kVrLn2 * (xk + (double)c + (double)a.r.k_rel * (xk - mean)) - log(sum);
    st = make_float2(c, z);
  } else {
    const VocabStat sv = vstat_block<NW>(vocab_stat_walk<T, NT>(srow, V, k), k, lds_v);
    if (threadIdx.x != 0) return;
    const Float2x l = vstat_log_prob(a.r, sv, x);
    lp = (double)l.hi + (double)l.lo;
    st = make_float2(sv.m, -sv.z);
  }
  if (logp) logp[row] = (float)lp;
  if (log_ratio) log_ratio[row] = lp - (ref ? (double)ref[row] : 0.0);
  if (stats) stats[row] = st;
}

// One workgroup per part of a row: every element depends on its row's two
// numbers only, so this is a copy with an exponential, bound by memory (8192 x
// 32000 bf16 with 70 % of the rows counting: 891 MB in 135 us, 6.6 TB/s).  The
// factor c of a row is coef[row] or, with per_seq, coef[row / seq_len].
constexpr int kGradVecs = 8;                           // 16-byte vectors per thread, all loads in flight at once
constexpr int kGradPart = kTokBlock * kGradVecs;       // vectors per workgroup

template <typename T>
__global__ __launch_bounds__(kTokBlock) void token_grad_kernel(const TokenRows a, int64_t row0, int parts,
                                                               const float2* __restrict__ stats,
                                                               const float* __restrict__ coef, int per_seq,
                                                               T* __restrict__ grad) {
  constexpr int VEC = Vec16<T>::N;
  const int64_t local = blockIdx.x / (unsigned)parts, row = row0 + local;
  const int part = (int)(blockIdx.x - (unsigned)local * (unsigned)parts);
  const int64_t V = a.r.V, v0 = (int64_t)part * kGradPart;
  const int tid = threadIdx.x;
  T* grow = grad + row * V;
  int64_t label;
  if (!token_live<true>(a, row, &label)) {
    const VocabGeom g = vocab_geom(grow, V);
    const T zero = from_f32<T>(0.f);
    if (part == 0 && tid < g.head) grow[tid] = zero;
    if (part == parts - 1 && g.tail0 + tid < V) grow[g.tail0 + tid] = zero;
    Vec16<T> z;
#pragma unroll
    for (int i = 0; i < VEC; ++i) z.v[i] = zero;
#pragma unroll
    for (int j = 0; j < kGradVecs; ++j) {
      const int64_t v = v0 + tid + j * kTokBlock;
      if (v < g.nvec) store16(grow + g.head + v * VEC, z);
    }
    return;
  }
  const T* srow = vocab_row<T>(a.r, row);
  const VocabGeom g = vocab_geom(srow, V);
  Vec16<T> x[kGradVecs];
  const int64_t e0 = g.head + v0 * VEC, some = g.nvec - v0;  // this part's first element and vectors
  const int left = some < kGradPart ? (int)some : kGradPart;
  const VecBuffer from = vec_buffer(srow + e0, left);
#pragma unroll
  for (int j = 0; j < kGradVecs; ++j) x[j] = vec_load<T>(from, tid + j * kTokBlock);
  const TokenGrad f(a.r.k, scalar_load(stats + row),
                    scalar_load(coef + (per_seq ? (uint32_t)row / (uint32_t)a.r.seq_len : row)) * (float)a.r.inv_T);
  auto one = [&](float xv, int64_t j) { return from_f32<T>(j == label ? f.label(xv) : f.other(xv)); };
  if (part == 0 && tid < g.head) grow[tid] = one(to_f32(srow[tid]), tid);
  if (part == parts - 1 && g.tail0 + tid < V) grow[g.tail0 + tid] = one(to_f32(srow[g.tail0 + tid]), g.tail0 + tid);
  const bool gvec = (((uintptr_t)grow ^ (uintptr_t)srow) & 15u) == 0;
  const VecBuffer to = vec_buffer(grow + e0, gvec ? left : 0);
  const int64_t at = label - e0;
  const int lv = at >= 0 && at / VEC < kGradPart ? (int)(at / VEC) : -1;
  const int li = lv < 0 ? 0 : (int)(at - (int64_t)lv * VEC);
#pragma unroll
  for (int j = 0; j < kGradVecs; ++j) {
    const int v = tid + j * kTokBlock;
    if (v < left) {
      forget(x[j]);
      Vec16<T> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(f.other(to_f32(x[j].v[i])));
      if (v == lv) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (i == li) o.v[i] = from_f32<T>(f.label(to_f32(x[j].v[i])));
      }
      if (gvec) {
        vec_store(to, (uint32_t)v, o);
      } else {
        T* p = grow + e0 + v * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[i] = o.v[i];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// ---- preference loss ---------------------------------------------------------

enum { kPrefSigmoid = 0, kPrefHinge = 1, kPrefIpo = 2 };

struct PrefArgs {
  const double* log_ratio;  // per row, the per-token reference already taken off
  const float* ref_seq;     // per sequence, or null
  double beta, smoothing, weight;
  int kind, average;
  float* rewards;       // per sequence, may be null
  float* coef;          // per sequence
  double* pair_loss;    // per pair
  unsigned* ticket;
  float* loss;
};

__device__ __forceinline__ double softplus_f64(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// TEAM threads per pair, a wavefront for short sequences: both sequences' sums,
// the pair's loss and the factors c of its two sequences; the last workgroup takes
// the mean of all pairs' losses.  A bounded number of workgroups, because each one
// draws a ticket (2048 pairs of 2 tokens, a workgroup each: 28 us instead of 10).
constexpr int kPrefGrid = 256;
constexpr int64_t kPrefShort = 64;  // tokens (8 pairs of 512, a wavefront each: 11 us instead of 6.5)

template <int TEAM>
__global__ __launch_bounds__(kTokBlock) void pref_join_kernel(const TokenRows a, const PrefArgs p, int64_t pairs) {
  constexpr int NW = TEAM / kWave, TEAMS = kTokBlock / TEAM;
  __shared__ double lds[kTokBlock / kWave];
  __shared__ bool last;
  const int lane = threadIdx.x % TEAM;
  const int64_t L = a.r.seq_len;
  for (int64_t pair = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM; pair < pairs; pair += (int64_t)gridDim.x * TEAMS) {
    double R[2], n[2];
    for (int side = 0; side < 2; ++side) {
      const int64_t row0 = (2 * pair + side) * L;
      double s = 0.0, c = 0.0;
      for (int64_t i = lane; i < L; i += TEAM) {
        s += p.log_ratio[row0 + i];
        if (p.average) {
          int64_t label;
          c += token_live<false>(a, row0 + i, &label) ? 1.0 : 0.0;
        }
      }
      R[side] = block_sum_f64<NW>(s, lds);
      n[side] = p.average ? fmax(block_sum_f64<NW>(c, lds), 1.0) : 1.0;
      R[side] = R[side] / n[side] - (p.ref_seq ? (double)p.ref_seq[2 * pair + side] : 0.0);
    }
    if (lane != 0) continue;
    const double h = R[0] - R[1], bh = p.beta * h;
    double loss, slope;  // slope = d loss / d h
    if (p.kind == kPrefSigmoid) {
      loss = (1.0 - p.smoothing) * softplus_f64(-bh) + p.smoothing * softplus_f64(bh);
      slope = p.beta * (p.smoothing - 1.0 / (1.0 + exp(bh)));
    } else if (p.kind == kPrefHinge) {
      loss = bh < 1.0 ? 1.0 - bh : (bh >= 1.0 ? 0.0 : bh);  // (a NaN stays one)
      slope = bh < 1.0 ? -p.beta : (bh >= 1.0 ? 0.0 : bh);
    } else {
      const double e = h - 0.5 / p.beta;
      loss = e * e;
      slope = 2.0 * e;
    }
    const double c = slope * p.weight / (double)pairs;
    for (int side = 0; side < 2; ++side) {
      p.coef[2 * pair + side] = (float)((side ? -c : c) / n[side]);
      if (p.rewards) p.rewards[2 * pair + side] = (float)(p.beta * R[side]);
    }
    publish_term(p.pair_loss + pair, loss);
  }
  __syncthreads();  // all of this workgroup's terms have arrived
  if (threadIdx.x == 0) last = draw_ticket(p.ticket) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  const double s = sum_terms<kTokBlock>(p.pair_loss, pairs, lds);
  if (threadIdx.x == 0) *p.loss = (float)(s * p.weight / (double)pairs);
}

// The mean over nothing.
__global__ void nan_kernel(float* __restrict__ out) { *out = __builtin_nanf(""); }

// out = the sum of the rows' terms; without a row that counts the mean is one over nothing.
__global__ __launch_bounds__(1024) void policy_sum_kernel(const double* __restrict__ v, int64_t n,
                                                          const int* __restrict__ live, float* __restrict__ out) {
  __shared__ double lds[1024 / kWave];
  const double s = block_sum_f64<1024 / kWave>(thread_share_of_sum_f64<1024>(v, n), lds);
  if (threadIdx.x == 0) *out = *live > 0 ? (float)s : __builtin_nanf("");
}

// Clears a ticket counter where no other kernel runs in front.
__global__ void clear_ticket_kernel(unsigned* __restrict__ ticket) { *ticket = 0u; }

// ---- clipped policy loss ------------------------------------------------------

struct PolicyArgs {
  const float* old_logp;
  const float* ref_logp;  // may be null when kl_weight is 0
  const float* adv;
  int adv_per_seq;
  float kl_weight, clip_lo, clip_hi;
  const float* seq_weight;  // weight of a sequence's tokens
  float* logp;              // per row, may be null
  double* row_loss;
  void* grad;  // may be null
};

// Weight of every sequence's tokens: weight / (live rows), or with per_seq
// weight / (sequences with a live row) / (live rows of this one).
// counts[0] = live rows.  One workgroup; the smallest power of two of lanes that
// is no smaller than a sequence takes it, up to a wavefront (4096 sequences of one
// token, a wavefront each: 175 us), with eight loads in flight, of that sequence
// or of eight sequences.
constexpr int kWeightBlock = 1024;

__global__ __launch_bounds__(kWeightBlock) void policy_weight_kernel(const TokenRows a, int64_t n_seq, int per_seq,
                                                                     float weight, float* __restrict__ seq_weight,
                                                                     int* __restrict__ counts) {
  constexpr int kInFlight = 8;
  __shared__ int total, full;
  if (threadIdx.x == 0) total = full = 0;
  const int L = (int)a.r.seq_len, n = (int)n_seq;  // (their product is below 2^22)
  int lanes = kWave;
  while (lanes / 2 >= L) lanes /= 2;
  const int sub = (int)threadIdx.x & (lanes - 1), first = (int)threadIdx.x / lanes, step = kWeightBlock / lanes;
  int rows = 0, some = 0;
  auto finish = [&](int q, int c) {  // c: of this lane
    for (int off = lanes / 2; off > 0; off >>= 1) c += __shfl_xor(c, off, kWave);
    if (sub != 0 || q >= n) return;
    seq_weight[q] = (float)c;  // exact: fewer than 2^24 rows
    rows += c;
    some += c > 0;
  };
  // rows at + u * stride, as far as place + u * by lies below end
  auto count = [&](int at, int stride, int place, int by, int end, int (&c)[kInFlight]) {
    int64_t label[kInFlight];
    bool on[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {  // (all loads before the first use; out of range, row 0's)
      const bool in = place + u * by < end;
      const int row = in ? at + u * stride : 0;
      label[u] = a.labels[row];
      on[u] = in && (!a.mask || a.mask[row] != 0);
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      c[u] += on[u] && label[u] != a.ignore_index && label[u] >= 0 && label[u] < a.r.V;
  };
  if (L > kWave) {
    for (int q = first; q < n; q += step) {
      int c[kInFlight] = {}, sum = 0;
      for (int i = sub; i < L; i += kWave * kInFlight) count(q * L + i, kWave, i, kWave, L, c);
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) sum += c[u];
      finish(q, sum);
    }
  } else {
    for (int q0 = first; q0 - first < n; q0 += step * kInFlight) {  // uniform
      int c[kInFlight] = {};
      if (sub < L) count(q0 * L + sub, step * L, q0, step, n, c);
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) finish(q0 + u * step, c[u]);
    }
  }
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    rows += __shfl_xor(rows, off, kWave);
    some += __shfl_xor(some, off, kWave);
  }
  __syncthreads();
  if (threadIdx.x % kWave == 0) {
    atomicAdd(&total, rows);
    atomicAdd(&full, some);
  }
  __syncthreads();
  for (int q = threadIdx.x; q < n; q += kWeightBlock) {
    const float c = seq_weight[q];
    seq_weight[q] = per_seq ? weight / ((float)full * fmaxf(c, 1.f)) : weight / (float)total;
  }
  if (threadIdx.x == 0) counts[0] = total;
}

// Loss term and d loss / d logp of one token, in fp32: the log probability comes
// as two floats, so that differences to the other models' keep their accuracy, and
// each part of the term is off by about 2^-22 of itself.  64-bit exponentials would
// take registers from the row.
__device__ __forceinline__ void policy_term(const PolicyArgs& p, Float2x lp, float old_lp, float ref_lp, float A,
                                            float* term, float* slope) {
  const float r = expf((lp.hi - old_lp) + lp.lo);
  const float held = r < p.clip_lo ? p.clip_lo : (r > p.clip_hi ? p.clip_hi : r);
  const float f = r * A, h = held * A;
  // min(f, h): the gradient flows where the ratio itself decides (f + h: one of them is NaN, and so is all)
  *term = f <= h ? -f : (h < f ? -h : f + h);
  *slope = f <= h ? -f : (h < f ? 0.f : f + h);
  if (p.kl_weight != 0.f) {
    const float d = (ref_lp - lp.hi) - lp.lo;
    const float em1 = expm1f(d);
    // e^d - 1 - d: its leading terms where the difference would cancel
    const float kl = fabsf(d) < 0.03f ? d * d * (0.5f + d * (1.f / 6.f + d * (1.f / 24.f + d * (1.f / 120.f)))) : em1 - d;
    *term = fmaf(p.kl_weight, kl, *term);
    *slope = fmaf(-p.kl_weight, em1, *slope);
  }
}

// A row's numbers besides its logits, fetched before them: after the row's sum
// they would be waited for with the row's registers held.
template <typename T>
struct PolicyRow {
  float old_lp, ref_lp, adv, weight;
  T label_logit;
  __device__ __forceinline__ PolicyRow() {}
  __device__ __forceinline__ PolicyRow(const TokenRows& a, const PolicyArgs& p, int64_t row, const T* srow, int64_t label) {
    const int64_t seq = (uint32_t)row / (uint32_t)a.r.seq_len;
    old_lp = scalar_load(p.old_logp + row);
    ref_lp = p.ref_logp ? scalar_load(p.ref_logp + row) : 0.f;
    adv = scalar_load(p.adv + (p.adv_per_seq ? seq : row));
    weight = scalar_load(p.seq_weight + seq);
    label_logit = srow[label];
  }
};

// What one thread does with a row's log probability: outputs, and the factor of
// its gradient.
template <typename T>
__device__ __forceinline__ float policy_finish(const TokenRows& a, const PolicyArgs& p, const PolicyRow<T>& r,
                                               int64_t row, Float2x lp) {
  float term, slope;
  policy_term(p, lp, r.old_lp, r.ref_lp, r.adv, &term, &slope);
  if (p.logp) p.logp[row] = lp.hi;
  p.row_loss[row] = (double)r.weight * (double)term;
  return r.weight * slope * (float)a.r.inv_T;
}

// Rows whose sum needs the true maximum: two walks over the row.
template <typename T, int NT>
__device__ __forceinline__ void policy_row_walked(const TokenRows& a, const PolicyArgs& p, const PolicyRow<T>& pr,
                                                  int64_t row, const T* srow, T* grow, int64_t label, float& coef) {
  __shared__ VocabStat lds[NT / kWave];
  const float k = a.r.k;
  const VocabStat s = vstat_block<NT / kWave>(vocab_stat_walk<T, NT>(srow, a.r.V, k), k, lds);
  if (threadIdx.x == 0) coef = policy_finish(a, p, pr, row, vstat_log_prob(a.r, s, to_f32(pr.label_logit)));
  if (!grow) return;
  __syncthreads();
  const TokenGrad f(k, make_float2(s.m, -s.z), coef);
  vocab_map_walk<T, NT>(srow, grow, a.r.V, [&](float x, int j) { return j == (int)label ? f.label(x) : f.other(x); });
}

// A row's factor c follows from the row itself, so the row stays in registers
// between its sum and its gradient and is read once.  Bound by memory: 8192 x
// 65536 bf16 with 70 % of the rows counting, 1826 MB in 316 us (5.8 TB/s, 281 us
// at best); two workgroups of 1024 threads a CU, one loading while the other
// stores.  512 threads with 16 vectors each take 321 us.
template <typename T, int NT, int KREG>
__global__ __launch_bounds__(NT) void policy_rows_kernel(const TokenRows a, const PolicyArgs p) {
  __shared__ RowSum lds[NT / kWave];
  __shared__ float coef;
  const int64_t row = blockIdx.x, V = a.r.V;
  T* grow = p.grad ? reinterpret_cast<T*>(p.grad) + row * V : nullptr;
  int64_t label;
  if (!token_live<true>(a, row, &label)) {
    if (threadIdx.x == 0) {
      if (p.logp) p.logp[row] = 0.f;
      p.row_loss[row] = 0.0;
    }
    if (grow) vocab_zero_row<T, NT>(grow, V);
    return;
  }
  const T* srow = vocab_row<T>(a.r, row);
  const PolicyRow<T> pr(a, p, row, srow, label);
  const VocabGeom g = vocab_geom(srow, V);
  RowRegs<T, NT, KREG> r;
  regs_load(r, srow, V, g);
  const RowSum s = regs_sum(r, g, a.r.k, lds);
  if (s.ok) {
    if (threadIdx.x == 0) coef = policy_finish(a, p, pr, row, rowsum_log_prob(a.r, s, to_f32(pr.label_logit)));
    if (!grow) return;
    __syncthreads();
    const TokenGrad f(a.r.k, make_float2(s.c, s.z), coef);
    regs_map(r, g, srow, grow, V, (int)label, [&](float x) { return f.other(x); }, [&](float x) { return f.label(x); });
    return;
  }
  __syncthreads();
  policy_row_walked<T, NT>(a, p, pr, row, srow, grow, label, coef);
}

// Rows too long for registers go through the kernels of the log probabilities
// and their gradient, with this one between them: the factor of each row, one
// thread a row.  (One workgroup that reads its row twice: 332 us for 1900 x
// 140000 bf16, this way 283.)
template <typename T>
__global__ __launch_bounds__(kTokBlock) void policy_coef_kernel(const TokenRows a, const PolicyArgs p,
                                                                const double* __restrict__ lp, float* __restrict__ coef) {
  const int64_t row = (int64_t)blockIdx.x * kTokBlock + threadIdx.x;
  if (row >= a.r.n_rows) return;
  int64_t label;
  if (!token_live<false>(a, row, &label)) {
    if (p.logp) p.logp[row] = 0.f;
    p.row_loss[row] = 0.0;
    coef[row] = 0.f;
    return;
  }
  const int64_t seq = row / a.r.seq_len;
  const double l = lp[row];
  const float hi = (float)l;
  PolicyRow<T> r;
  r.old_lp = p.old_logp[row];
  r.ref_lp = p.ref_logp ? p.ref_logp[row] : 0.f;
  r.adv = p.adv[p.adv_per_seq ? seq : row];
  r.weight = p.seq_weight[seq];
  // (the gradient kernel takes the temperature itself; divided out and multiplied in again
  // the factor is the same, but for one tie in forty million)
  coef[row] = policy_finish(a, p, r, row, Float2x{hi, fabsf(hi) < __builtin_inff() ? (float)(l - (double)hi) : 0.f}) /
              (float)a.r.inv_T;
}

// ---- host side ------------------------------------------------------------------

inline size_t pad16(size_t b) { return (b + 15) / 16 * 16; }

struct TokenWs {
  double* row;     // n_rows: log ratios or loss terms
  float2* stats;   // n_rows
  double* lp;      // n_rows: log probabilities
  float* coef;     // n_rows: gradient factors
  double* pair;    // n_seq / 2
  float* seq;      // n_seq: factors or weights
  int* counts;     // 4
};

inline size_t token_ws_bytes(int64_t n_rows, int64_t n_seq) {
  return 16 + pad16((size_t)n_rows * 8) * 3 + pad16((size_t)n_rows * 4) + pad16((size_t)(n_seq / 2) * 8) +
         pad16((size_t)n_seq * 4);
}

inline TokenWs token_carve(void* ws, int64_t n_rows, int64_t n_seq) {
  char* b = reinterpret_cast<char*>(ws);
  TokenWs w;
  w.counts = reinterpret_cast<int*>(b);
  b += 16;
  w.row = reinterpret_cast<double*>(b);
  b += pad16((size_t)n_rows * 8);
  w.stats = reinterpret_cast<float2*>(b);
  b += pad16((size_t)n_rows * 8);
  w.lp = reinterpret_cast<double*>(b);
  b += pad16((size_t)n_rows * 8);
  w.coef = reinterpret_cast<float*>(b);
  b += pad16((size_t)n_rows * 4);
  w.pair = reinterpret_cast<double*>(b);
  b += pad16((size_t)(n_seq / 2) * 8);
  w.seq = reinterpret_cast<float*>(b);
  return w;
}

template <typename T>
int launch_token_stat(const TokenRows& a, const float* ref, float* logp, double* log_ratio, float2* stats,
                      unsigned* ticket, hipStream_t st) {
  const RowShape sh = row_shape<T>(a.r.V);
#define TS_STAT(NT, KREG)                                                                                         \
  hipLaunchKernelGGL((token_stat_kernel<T, NT, KREG>), dim3((unsigned)a.r.n_rows), dim3(NT), 0, st, a, ref, logp, \
                     log_ratio, stats, ticket)
  if (sh.nt == 64)
    TS_STAT(64, 4);
  else if (sh.nt == 256 && sh.kreg == 4)
    TS_STAT(256, 4);
  else if (sh.nt == 256)
    TS_STAT(256, 8);
  else
    TS_STAT(512, 8);
#undef TS_STAT
  return check_launch();
}

template <typename T>
int launch_token_grad(const TokenRows& a, const float2* stats, const float* coef, int per_seq, void* grad,
                      hipStream_t st) {
  const int64_t vecs = a.r.V / Vec16<T>::N;
  const int64_t parts = vecs <= kGradPart ? 1 : (vecs + kGradPart - 1) / kGradPart;
  // (the grid counts threads in 32 bits)
  for (int64_t row0 = 0; row0 < a.r.n_rows;) {
    int64_t n = a.r.n_rows - row0;
    if (n * parts > (1 << 23)) n = (1 << 23) / parts;
    if (n < 1) return TS_ERR_RANGE;
    hipLaunchKernelGGL((token_grad_kernel<T>), dim3((unsigned)(n * parts)), dim3(kTokBlock), 0, st, a, row0,
                       (int)parts, stats, coef, per_seq, reinterpret_cast<T*>(grad));
    const int rc = check_launch();
    if (rc) return rc;
    row0 += n;
  }
  return TS_OK;
}

inline int launch_nan(float* out, hipStream_t st) {
  hipLaunchKernelGGL(nan_kernel, dim3(1), dim3(1), 0, st, out);
  return check_launch();
}

// Three launches: the rows' log ratios, the pairs (which need whole sequences of
// them), the gradient.  The logits are read twice, 734 + 524 MB at 16 sequences
// of 512 x 32000 bf16 with 70 % of the rows counting.  (Pair by pair, so that the
// second reading finds the rows in the last-level cache, is no faster: the
// gradient's writes bound that kernel, 34 us for two pairs either way, and the
// smaller launches cost more than they save, 275 against 226 us in all.)
template <typename T>
int launch_preference(const TokenRows& a, const float* ref_tok, const PrefArgs& p, const TokenWs& w, int64_t n_seq,
                      void* grad, hipStream_t st) {
  const int64_t pairs = n_seq / 2;
  if (pairs == 0) return launch_nan(p.loss, st);
  int rc;
  if (a.r.n_rows > 0) {
    rc = launch_token_stat<T>(a, ref_tok, nullptr, w.row, w.stats, p.ticket, st);
  } else {
    hipLaunchKernelGGL(clear_ticket_kernel, dim3(1), dim3(1), 0, st, p.ticket);
    rc = check_launch();
  }
  if (rc) return rc;
  const bool small = a.r.seq_len <= kPrefShort;
  const int64_t groups = small ? (pairs + kTokBlock / kWave - 1) / (kTokBlock / kWave) : pairs;
  const dim3 grid((unsigned)(groups < kPrefGrid ? groups : kPrefGrid));
  if (small)
    hipLaunchKernelGGL((pref_join_kernel<kWave>), grid, dim3(kTokBlock), 0, st, a, p, pairs);
  else
    hipLaunchKernelGGL((pref_join_kernel<kTokBlock>), grid, dim3(kTokBlock), 0, st, a, p, pairs);
  rc = check_launch();
  if (rc || !grad || a.r.n_rows == 0) return rc;
  return launch_token_grad<T>(a, w.stats, w.seq, 1, grad, st);
}

template <typename T>
int launch_policy(const TokenRows& a, const PolicyArgs& p, const TokenWs& w, int64_t n_seq, int per_seq, float weight,
                  float* loss_out, hipStream_t st) {
  if (a.r.n_rows == 0) return launch_nan(loss_out, st);
  hipLaunchKernelGGL(policy_weight_kernel, dim3(1), dim3(kWeightBlock), 0, st, a, n_seq, per_seq, weight, w.seq, w.counts);
  int rc = check_launch();
  if (rc) return rc;
  const dim3 grid((unsigned)a.r.n_rows);
  const RowShape sh = row_shape<T>(a.r.V);
#define TS_POLICY(NT, KREG) hipLaunchKernelGGL((policy_rows_kernel<T, NT, KREG>), grid, dim3(NT), 0, st, a, p)
  if (sh.nt == 64)
    TS_POLICY(64, 4);
  else if (sh.nt == 256 && sh.kreg == 4)
    TS_POLICY(256, 4);
  else if (sh.nt == 256)
    TS_POLICY(256, 8);
  else if (sh.nt == 512)
    TS_POLICY(512, 8);
  else if (sh.kreg == 8)
    TS_POLICY(1024, 8);
  else if (sh.kreg == 16)
    TS_POLICY(1024, 16);
  else {
    rc = launch_token_stat<T>(a, nullptr, nullptr, w.lp, w.stats, nullptr, st);
    if (rc) return rc;
    hipLaunchKernelGGL((policy_coef_kernel<T>), dim3((unsigned)((a.r.n_rows + kTokBlock - 1) / kTokBlock)),
                       dim3(kTokBlock), 0, st, a, p, w.lp, w.coef);
    rc = check_launch();
    if (rc) return rc;
    if (p.grad) rc = launch_token_grad<T>(a, w.stats, w.coef, 0, p.grad, st);
    if (rc) return rc;
  }
#undef TS_POLICY
  rc = check_launch();
  if (rc) return rc;
  hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(1024), 0, st, w.row, a.r.n_rows, (const int*)w.counts, loss_out);
  return check_launch();
}

// Checks shared by the entry points; `grad` and `f32s` may be null.
inline int token_status(const void* s, int64_t n_seq, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok,
                        const int64_t* labels, double temperature, const void* grad, int dtype) {
  const int rc = vocab_rows_status(s, n_seq, seq_len, V, ld_seq, ld_tok, temperature, dtype);
  if (rc) return rc;
  if (n_seq * seq_len > 0 && !labels) return TS_ERR_ARG;
  if ((uintptr_t)labels & 7u) return TS_ERR_ALIGN;
  if ((uintptr_t)grad & (dtype == TS_F32 ? 3u : 1u)) return TS_ERR_ALIGN;
  return TS_OK;
}

inline TokenRows token_rows(const void* s, int64_t n_seq, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok,
                            const int64_t* labels, const uint8_t* mask, int64_t ignore_index, double temperature) {
  TokenRows a;
  a.r = vocab_rows(s, n_seq * seq_len, seq_len, V, ld_seq, ld_tok, temperature);
  a.labels = labels;
  a.mask = mask;
  a.ignore_index = ignore_index;
  return a;
}

}  // namespace ts

extern "C" {

int ts_token_logp_fwd(const void* s, int64_t n_seq, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok,
                      const int64_t* labels, const uint8_t* row_mask, int64_t ignore_index, double temperature,
                      float* logp, float* stats, int dtype, ts_stream_t stream) {
  const int rc = ts::token_status(s, n_seq, seq_len, V, ld_seq, ld_tok, labels, temperature, nullptr, dtype);
  if (rc) return rc;
  if (n_seq * seq_len == 0) return TS_OK;
  if (!logp) return TS_ERR_ARG;
  if (((uintptr_t)logp & 3u) || ((uintptr_t)stats & 7u)) return TS_ERR_ALIGN;
  const ts::TokenRows a =
      ts::token_rows(s, n_seq, seq_len, V, ld_seq, ld_tok, labels, row_mask, ignore_index, temperature);
  hipStream_t st = (hipStream_t)stream;
  TS_BY_DTYPE(dtype, (ts::launch_token_stat<T>(a, nullptr, logp, nullptr, (float2*)stats, nullptr, st)))
}

int ts_token_logp_bwd(const void* s, int64_t n_seq, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok,
                      const int64_t* labels, const uint8_t* row_mask, int64_t ignore_index, double temperature,
                      const float* stats, const float* grad_logp, void* grad, int dtype, ts_stream_t stream) {
  const int rc = ts::token_status(s, n_seq, seq_len, V, ld_seq, ld_tok, labels, temperature, grad, dtype);
  if (rc) return rc;
  if (n_seq * seq_len == 0) return TS_OK;
  if (!stats || !grad_logp || !grad) return TS_ERR_ARG;
  if (((uintptr_t)grad_logp & 3u) || ((uintptr_t)stats & 7u)) return TS_ERR_ALIGN;
  const ts::TokenRows a =
      ts::token_rows(s, n_seq, seq_len, V, ld_seq, ld_tok, labels, row_mask, ignore_index, temperature);
  hipStream_t st = (hipStream_t)stream;
  TS_BY_DTYPE(dtype, (ts::launch_token_grad<T>(a, (const float2*)stats, grad_logp, 0, grad, st)))
}

size_t ts_token_loss_workspace_bytes(int64_t n_seq, int64_t seq_len) {
  if (n_seq < 0 || seq_len < 0) return 0;
  return ts::token_ws_bytes(n_seq * seq_len, n_seq);
}

int ts_preference_fwd_bwd(const void* s, int64_t n_seq, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok,
                          const int64_t* labels, const uint8_t* row_mask, int64_t ignore_index, const float* ref_logp,
                          int ref_per_token, double beta, int kind, double smoothing, int average, double weight,
                          void* workspace, float* loss_out, float* rewards, void* grad, int dtype,
                          ts_stream_t stream) {
  const int rc = ts::token_status(s, n_seq, seq_len, V, ld_seq, ld_tok, labels, 1.0, grad, dtype);
  if (rc) return rc;
  if (n_seq % 2 || !workspace || !loss_out) return TS_ERR_ARG;
  if (!(beta > 0.0) || !(smoothing >= 0.0 && smoothing <= 1.0)) return TS_ERR_ARG;
  if (kind != ts::kPrefSigmoid && kind != ts::kPrefHinge && kind != ts::kPrefIpo) return TS_ERR_ARG;
  if (smoothing != 0.0 && kind != ts::kPrefSigmoid) return TS_ERR_ARG;
  if (n_seq * (ref_per_token ? seq_len : 1) > 0 && !ref_logp) return TS_ERR_ARG;
  if (((uintptr_t)workspace & 15u) || (((uintptr_t)ref_logp | (uintptr_t)loss_out | (uintptr_t)rewards) & 3u))
    return TS_ERR_ALIGN;
  const ts::TokenRows a = ts::token_rows(s, n_seq, seq_len, V, ld_seq, ld_tok, labels, row_mask, ignore_index, 1.0);
  const ts::TokenWs w = ts::token_carve(workspace, a.r.n_rows, n_seq);
  ts::PrefArgs p;
  p.log_ratio = w.row;
  p.ref_seq = ref_per_token ? nullptr : ref_logp;
  p.beta = beta;
  p.smoothing = smoothing;
  p.weight = weight;
  p.kind = kind;
  p.average = average;
  p.rewards = rewards;
  p.coef = w.seq;
  p.pair_loss = w.pair;
  p.ticket = reinterpret_cast<unsigned*>(w.counts);
  p.loss = loss_out;
  const float* ref_tok = ref_per_token ? ref_logp : nullptr;
  hipStream_t st = (hipStream_t)stream;
  TS_BY_DTYPE(dtype, (ts::launch_preference<T>(a, ref_tok, p, w, n_seq, grad, st)))
}

int ts_policy_fwd_bwd(const void* s, int64_t n_seq, int64_t seq_len, int64_t V, int64_t ld_seq, int64_t ld_tok,
                      const int64_t* labels, const uint8_t* row_mask, int64_t ignore_index, double temperature,
                      const float* old_logp, const float* ref_logp, const float* advantages, int adv_per_seq,
                      double kl_weight, double clip_lo, double clip_hi, int per_seq, double weight, void* workspace,
                      float* loss_out, float* logp, void* grad, int dtype, ts_stream_t stream) {
  const int rc = ts::token_status(s, n_seq, seq_len, V, ld_seq, ld_tok, labels, temperature, grad, dtype);
  if (rc) return rc;
  if (!workspace || !loss_out || !(clip_lo <= clip_hi)) return TS_ERR_ARG;
  if (n_seq * seq_len > 0 && (!old_logp || !advantages || (!ref_logp && kl_weight != 0.0))) return TS_ERR_ARG;
  if (((uintptr_t)workspace & 15u) || (((uintptr_t)old_logp | (uintptr_t)ref_logp | (uintptr_t)advantages |
                                        (uintptr_t)loss_out | (uintptr_t)logp) & 3u))
    return TS_ERR_ALIGN;
  const ts::TokenRows a =
      ts::token_rows(s, n_seq, seq_len, V, ld_seq, ld_tok, labels, row_mask, ignore_index, temperature);
  const ts::TokenWs w = ts::token_carve(workspace, a.r.n_rows, n_seq);
  ts::PolicyArgs p;
  p.old_logp = old_logp;
  p.ref_logp = ref_logp;
  p.adv = advantages;
  p.adv_per_seq = adv_per_seq;
  p.kl_weight = (float)kl_weight;
  p.clip_lo = (float)clip_lo;
  p.clip_hi = (float)clip_hi;
  p.seq_weight = w.seq;
  p.logp = logp;
  p.row_loss = w.row;
  p.grad = grad;
  hipStream_t st = (hipStream_t)stream;
  TS_BY_DTYPE(dtype, (ts::launch_policy<T>(a, p, w, n_seq, per_seq, (float)weight, loss_out, st)))
}

}  // extern "C"
