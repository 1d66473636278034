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
  // rounding took, relative: (log2(e) / T - k) / k, at most 2^-24.  Every exponent
  // of a row is off by that same factor, which would add up over a sequence of
  // rows and show in the log-sum-exp of a row far from zero: token_stat_kernel and
  // top_logits_kernel correct for it to first order.  The policy loss and the
  // distillation, which add up no sequence's log probabilities, leave it in them,
  // times their distance from the row's mean (16: 1e-6).
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

// The row's address, the same in every lane of the wavefront: said to the
// compiler, whose 64-bit division leaves it in vector registers, so that it and
// all that follows from it stay scalar.
template <typename T>
__device__ __forceinline__ const T* vocab_row(const VocabRows& a, int64_t row) {
  const uint32_t q = (uint32_t)row / (uint32_t)a.seq_len;  // fewer than 2^22 rows
  const T* p = reinterpret_cast<const T*>(a.s) + q * a.ld_seq + (row - (int64_t)q * a.seq_len) * a.ld_tok;
  const uint64_t b = (uint64_t)p;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32));
  return reinterpret_cast<const T*>(((uint64_t)hi << 32) | lo);
}

// A number that is the same in every lane, said to the compiler as the address above.
__device__ __forceinline__ float same_in_wave(float x) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
}

// An fp32 number and what its rounding left out.  The log probabilities of a row
// are formed in this type: a sum over a sequence of them, or the difference of
// two that nearly agree, would show the last bits of fp32, and 64-bit
// logarithms and exponentials in a kernel that holds a row in registers spill
// (28 % of the policy loss's time at 8192 x 65536 bf16).
struct Float2x {
  float hi, lo;
};

__device__ __forceinline__ Float2x two_sum(float x, float y) {
#pragma clang fp contract(off)
  const float s = x + y, v = s - x;
  return Float2x{s, (x - (s - v)) + (y - v)};
}

__device__ __forceinline__ Float2x two_mul(float x, float y) {
#pragma clang fp contract(off)
  const float p = x * y;
  return Float2x{p, __builtin_fmaf(x, y, -p)};
}

// log2(z) within 2e-7 for normal z > 0 (-inf for 0): the hardware's logarithm, corrected by what
// its own power of two leaves of z.
__device__ __forceinline__ Float2x log2_2x(float z) {
  if (!(z > 0.f && z < __builtin_inff())) return Float2x{__builtin_amdgcn_logf(z), 0.f};
  const float e = (float)(__builtin_amdgcn_frexp_expf(z));  // z = f 2^e, f in [1/2, 1)
  const float f = __builtin_amdgcn_frexp_mantf(z);
  const float l = __builtin_amdgcn_logf(f);
  const Float2x s = two_sum(e, l);
  return Float2x{s.hi, s.lo + kVrLog2e * fmaf(f, fast_exp2(-l), -1.f)};
}

// ln 2 times (e - log2 z): the log probability of a term 2^e of a sum z.
__device__ __forceinline__ Float2x ln_share(Float2x e, float z) {
#pragma clang fp contract(off)
  const Float2x l = log2_2x(z), h = two_sum(e.hi, -l.hi);
  if (!(__builtin_fabsf(h.hi) < __builtin_inff())) return Float2x{h.hi, 0.f};  // a logit of -inf
  const float lo = e.lo + (h.lo - l.lo);
  const Float2x m = two_mul(h.hi, 0.693147182464599609375f);
  return two_sum(m.hi, m.lo + (lo * 0.693147182464599609375f + h.hi * -1.904654323e-09f));
}

// m = max x, z = sum 2^((x - m) k)
struct VocabStat {
  float m, z;
};

__device__ __forceinline__ VocabStat vstat_init() { return VocabStat{kVrLowest, 0.f}; }

// The state re-based onto the larger maximum m.
__device__ __forceinline__ VocabStat vstat_rebase(VocabStat s, float m, float k) {
  return VocabStat{m, s.z * fast_exp2((s.m - m) * k)};
}

__device__ __forceinline__ VocabStat vstat_merge(VocabStat p, VocabStat q, float k) {
  const float m = fmaxf(p.m, q.m);
  return VocabStat{m, vstat_rebase(p, m, k).z + vstat_rebase(q, m, k).z};
}

// A NaN logit makes z NaN; a logit of -inf (a masked vocabulary entry) adds nothing.
template <int N>
__device__ __forceinline__ void vstat_fold(VocabStat& s, const float (&x)[N], float k) {
  float m = s.m;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
  if (m > s.m) s = vstat_rebase(s, m, k);
#pragma unroll
  for (int i = 0; i < N; ++i) s.z += fast_exp2((x[i] - s.m) * k);
}

// Merged over a workgroup of NW wavefronts; every thread gets the result.
template <int NW>
__device__ __forceinline__ VocabStat vstat_block(VocabStat s, float k, VocabStat* lds) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1)
    s = vstat_merge(s, VocabStat{__shfl_xor(s.m, off, kWave), __shfl_xor(s.z, off, kWave)}, k);
  if (NW == 1) return s;
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = s;
  __syncthreads();
  // lane i takes state i % NW, and the lanes merge (NW states at once would need 2 NW registers a lane)
  s = lds[threadIdx.x % NW];
#pragma unroll
  for (int off = NW / 2; off > 0; off >>= 1)
    s = vstat_merge(s, VocabStat{__shfl_xor(s.m, off, kWave), __shfl_xor(s.z, off, kWave)}, k);
  __syncthreads();  // lds may be used again
  return s;
}

// ln of the soft-max probability of a logit x of the row.
__device__ __forceinline__ Float2x vstat_log_prob(const VocabRows& r, const VocabStat& s, float x) {
#pragma clang fp contract(off)
  const float k = r.k;
  const Float2x d = two_sum(x, -s.m), p = two_mul(d.hi, k);
  if (d.hi < -1e38f && d.hi > -__builtin_inff()) return Float2x{(float)((double)d.hi * r.inv_T), 0.f};  // (d k may overflow)
  return ln_share(Float2x{p.hi, p.lo + d.lo * k}, s.z);
}

// A value at a uniform address that nothing writes while the kernel runs, through
// the scalar unit: it takes no vector register, and waiting for it is no wait for
// the row's loads.
template <typename X>
__device__ __forceinline__ X scalar_load(const X* p) {
  static_assert(sizeof(X) % 4 == 0, "whole words");
  const auto* w = (const __attribute__((address_space(4))) uint32_t*)(uint64_t)p;
  uint32_t words[sizeof(X) / 4];
#pragma unroll
  for (unsigned i = 0; i < sizeof(X) / 4; ++i) words[i] = w[i];
  X x;
  __builtin_memcpy(&x, words, sizeof(X));
  return x;
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

// Statistics of many elements: 64 at a time, and those of these.  (A sum of n terms
// is off by up to n 2^-25 of itself where logits are coarse and every addition rounds
// the same way: 1e-5 for 300.)
struct VocabStatSum {
  VocabStat s = vstat_init(), before = vstat_init();
  int n = 0;
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float k) {
    vstat_fold<N>(s, x, k);
    n += N;
    if (n >= 64) {
      before = vstat_merge(before, s, k);
      s.z = 0.f;
      n = 0;
    }
  }
  __device__ __forceinline__ VocabStat whole(float k) const { return vstat_merge(before, s, k); }
};

// This thread's share of the row's statistics when NT threads walk it.
template <typename T, int NT>
__device__ __forceinline__ VocabStat vocab_stat_walk(const T* row, int64_t V, float k) {
  constexpr int VEC = Vec16<T>::N;
  const VocabGeom g = vocab_geom(row, V);
  VocabStatSum s;
  float x1[1];
  if ((int)threadIdx.x < g.head) {
    x1[0] = to_f32(row[threadIdx.x]);
    s.add(x1, k);
  }
  if (g.tail0 + threadIdx.x < V) {
    x1[0] = to_f32(row[g.tail0 + threadIdx.x]);
    s.add(x1, k);
  }
  for (int64_t v = threadIdx.x; v < g.nvec; v += NT) {
    const Vec16<T> r = load16(row + g.head + v * VEC);
    float x[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = to_f32(r.v[i]);
    s.add(x, k);
  }
  return s.whole(k);
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

// ---------------------------------------------------------------------------
// Rows held in registers.  NT threads hold a row of up to NT * KREG 16-byte
// vectors, thread t the vectors t, t + NT, ...; what lies in front of the first
// and behind the last 16-byte boundary is one element per lane of the first
// wavefront.
//
// Sums are taken of 2^(x k + c) with an integer c per wavefront, so that
// moving a sum from one c to another is exact and no maximum of the whole row is
// needed in front: c = -rint(k x_0) with x_0 an element of the wavefront near its
// largest.  Elements may exceed x_0; a sum that overflows for it (or comes out 0
// or NaN) is not ok, and the caller walks the row again with its true maximum.
// How near x_0 is decides the rounding of the exponents: the gradient of a row
// whose probability is nearly all in one token shows it, so there x_0 is taken
// over all of the wavefront's vectors, by their raw bits (an instruction for two
// 16-bit logits); a log-sum-exp does with the first vectors' maximum, and its
// first exponential then waits for one vector instead of for all.
// ---------------------------------------------------------------------------
// c of a wavefront without an element above -1e7 / k (masked vocabulary): with it such an element's
// term is 0, so that the others' sum stands alone, or infinite, and the row is walked.
constexpr float kVrNoTerm = 1e9f;
constexpr float kVrLeast = -1e7f;

// `count` 16-byte vectors behind a 16-byte aligned address, the same in every
// lane.  Loads beyond them return 0 and stores beyond them do nothing (the
// buffer's own range check), so that a thread issues all its loads with no
// branch between them and one register of addresses; vectors that a lane does
// not have are left out where they are used.  With predicated loads the
// compiler kept an address and a mask for each and spilled them between the
// loads.  All of the offset is the lane's (the range check takes a scalar
// offset off the length first).
struct VecBuffer {
  __amdgpu_buffer_rsrc_t rsrc;
};
constexpr int kNonTemporal = 2;

template <typename T>
__device__ __forceinline__ VecBuffer vec_buffer(const T* base, int count) {
  return VecBuffer{__builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), (short)0, count * 16, 0x00020000)};
}
template <typename T>
__device__ __forceinline__ Vec16<T> vec_load(const VecBuffer& b, uint32_t v) {
  const auto raw = __builtin_amdgcn_raw_buffer_load_b128(b.rsrc, (int)(v * 16u), 0, kNonTemporal);
  Vec16<T> r;
  __builtin_memcpy(&r, &raw, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ void vec_store(const VecBuffer& b, uint32_t v, const Vec16<T>& x) {
  u32x4 raw;
  __builtin_memcpy(&raw, &x, 16);
  __builtin_amdgcn_raw_buffer_store_b128(raw, b.rsrc, (int)(v * 16u), 0, kNonTemporal);
}

// Element i of `count` (0 beyond them), as fp32.
template <typename T>
__device__ __forceinline__ T elem_load(const T* base, int count, uint32_t i) {
  const VecBuffer b{__builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), (short)0, count * (int)sizeof(T), 0x00020000)};
  T r;
  if constexpr (sizeof(T) == 4) {
    const auto raw = __builtin_amdgcn_raw_buffer_load_b32(b.rsrc, (int)(i * 4u), 0, 0);
    __builtin_memcpy(&r, &raw, 4);
  } else {
    const auto raw = __builtin_amdgcn_raw_buffer_load_b16(b.rsrc, (int)(i * 2u), 0, 0);
    __builtin_memcpy(&r, &raw, 2);
  }
  return r;
}

template <typename T, int NT, int KREG>
struct RowRegs {
  Vec16<T> v[KREG];
  T head, tail;  // end elements
  bool has_h, has_t;
  __device__ __forceinline__ float h() const { return has_h ? to_f32(head) : -__builtin_inff(); }
  __device__ __forceinline__ float t() const { return has_t ? to_f32(tail) : -__builtin_inff(); }
};

template <typename T, int NT, int KREG>
__device__ __forceinline__ void regs_load(RowRegs<T, NT, KREG>& r, const T* row, int64_t V, const VocabGeom& g) {
  // (the end elements without a branch as well: a wait for them inside one would be a wait for all)
  r.has_h = (int)threadIdx.x < g.head;
  r.has_t = g.tail0 + threadIdx.x < V;
  r.head = elem_load(row, g.head, threadIdx.x);
  r.tail = elem_load(row + g.tail0, (int)(V - g.tail0), threadIdx.x);
  const VecBuffer body = vec_buffer(row + g.head, g.nvec < NT * KREG ? (int)g.nvec : NT * KREG);
#pragma unroll
  for (int j = 0; j < KREG; ++j) r.v[j] = vec_load<T>(body, threadIdx.x + j * NT);
}

// Makes the compiler forget what it knows of a vector, so that each pass
// unpacks it again instead of keeping eight floats alive for it.
template <typename T>
__device__ __forceinline__ void forget(Vec16<T>& v) {
  u32x4 b;
  __builtin_memcpy(&b, &v, 16);
  asm volatile("" : "+v"(b));
  __builtin_memcpy(&v, &b, 16);
}

// The largest of a vector's elements by their bits as signed numbers: two
// sixteen-bit maxima, or one of 32 bits.  For logits above zero that is their
// order; of a vector without such a one it is just one of its elements.
template <typename T>
struct RawMax {
  int32_t m;
  static constexpr int32_t kNone = sizeof(T) == 4 ? (int32_t)0x80000000 : (int32_t)0x80008000;
  __device__ __forceinline__ static int32_t max2(int32_t a, int32_t b) {
    if constexpr (sizeof(T) == 4) {
      return a > b ? a : b;
    } else {
      typedef int16_t s16x2 __attribute__((ext_vector_type(2)));
      s16x2 x, y;
      __builtin_memcpy(&x, &a, 4);
      __builtin_memcpy(&y, &b, 4);
      const s16x2 z = __builtin_elementwise_max(x, y);
      int32_t r;
      __builtin_memcpy(&r, &z, 4);
      return r;
    }
  }
  __device__ __forceinline__ static int32_t of(const Vec16<T>& v) {
    int32_t w[4];
    __builtin_memcpy(w, &v, 16);
    return max2(max2(w[0], w[1]), max2(w[2], w[3]));
  }
  // the element that `m` stands for, as fp32
  __device__ __forceinline__ static float value(int32_t m) {
    if constexpr (sizeof(T) == 4) {
      return __int_as_float(m);
    } else {
      const int16_t lo = (int16_t)(m & 0xffff), hi = (int16_t)(m >> 16);
      const int16_t top = lo > hi ? lo : hi;
      T t;
      __builtin_memcpy(&t, &top, 2);
      return to_f32(t);
    }
  }
  // The smallest by their bits as unsigned numbers: of a vector without a logit above zero, its largest logit.
  __device__ __forceinline__ static int32_t min2(int32_t a, int32_t b) {
    if constexpr (sizeof(T) == 4) {
      return (int32_t)((uint32_t)a < (uint32_t)b ? (uint32_t)a : (uint32_t)b);
    } else {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 x, y;
      __builtin_memcpy(&x, &a, 4);
      __builtin_memcpy(&y, &b, 4);
      const u16x2 z = __builtin_elementwise_min(x, y);
      int32_t r;
      __builtin_memcpy(&r, &z, 4);
      return r;
    }
  }
  __device__ __forceinline__ static int32_t least(const Vec16<T>& v) {
    int32_t w[4];
    __builtin_memcpy(w, &v, 16);
    return min2(min2(w[0], w[1]), min2(w[2], w[3]));
  }
  // The largest logit of elements whose raw maximum and minimum are m and l.
  __device__ __forceinline__ static float value(int32_t m, int32_t l) {
    if constexpr (sizeof(T) == 4) {
      return __int_as_float(m >= 0 ? m : l);
    } else {
      const int32_t lo = (int16_t)(m & 0xffff) >= 0 ? m : l, hi = m >= 0 ? m : l;
      const uint16_t a = (uint16_t)(lo & 0xffff), b = (uint16_t)((uint32_t)hi >> 16);
      T x, y;
      __builtin_memcpy(&x, &a, 2);
      __builtin_memcpy(&y, &b, 2);
      return fmaxf(to_f32(x), to_f32(y));
    }
  }
};

// The largest of m and of the wavefront's elements in its first nvec vectors.
// ALL: of all of them, else of the first ones and, if those are masked, of all.
template <bool ALL, typename T, int NT, int KREG>
__device__ __forceinline__ float regs_max(const RowRegs<T, NT, KREG>& r, int nvec, float m, float k) {
  constexpr int VEC = Vec16<T>::N;
  typedef RawMax<T> Raw;
  if (ALL) {
    int32_t raw = Raw::kNone;
#pragma unroll
    for (int j = 0; j < KREG; ++j)
      if ((int)threadIdx.x + j * NT < nvec) raw = Raw::max2(raw, Raw::of(r.v[j]));
    if ((int)threadIdx.x < nvec) m = fmaxf(m, Raw::value(raw));
  } else {
    if ((int)threadIdx.x < nvec) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) m = fmaxf(m, to_f32(r.v[0].v[i]));
    }
  }
  m = wave_max(m);
  if (!(m * k > (ALL ? 0.f : kVrLeast))) {  // (masked, or, by raw bits, nothing above zero: the true maximum)
#pragma unroll
    for (int j = 0; j < KREG; ++j) {
      if ((int)threadIdx.x + j * NT < nvec) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) m = fmaxf(m, to_f32(r.v[j].v[i]));
      }
    }
    m = wave_max(m);
  }
  return m;
}

// c of the wavefront.
template <bool ALL, typename T, int NT, int KREG>
__device__ __forceinline__ float regs_anchor(const RowRegs<T, NT, KREG>& r, const VocabGeom& g, float k) {
  const float e = regs_max<ALL>(r, (int)g.nvec, fmaxf(r.h(), r.t()), k) * k;
  if (!(e > kVrLeast)) return kVrNoTerm;
  return e < 1e30f ? -rintf(e) : 0.f;  // (an infinite logit makes the sum overflow whatever c is)
}

// A later piece of the row, of nvec vectors, in r: where it holds something larger
// than what c was taken from, c follows it.  Returns the exponent (<= 0) by which
// sums taken so far have to be moved.
template <typename T, int NT, int KREG>
__device__ __forceinline__ float regs_raise(const RowRegs<T, NT, KREG>& r, int nvec, float k, float& c) {
  const float e = regs_max<true>(r, nvec, -__builtin_inff(), k) * k;
  const float old = c;
  if (e > kVrLeast && e < 1e30f) c = fminf(c, -rintf(e));
  return fmaxf(c - old, -1000.f);
}

struct RowSum {  // z = sum 2^(x k + c); a, with TWO: another such sum, and the row's sum is z + a
  float c, z, a;
  bool ok;
};

// Merged over a workgroup of NW wavefronts: each leaves its sums in `lds` (NW
// RowSums), and after a barrier every thread gets the whole.
template <int NW, bool TWO>
__device__ __forceinline__ RowSum rowsum_put(float c, float z, float a, RowSum* lds) {
  z = wave_sum(z);
  if (TWO) a = wave_sum(a);
  const RowSum r{c, z, a, true};
  if (NW > 1 && threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = r;
  return r;
}

template <int NW, bool TWO>
__device__ __forceinline__ RowSum rowsum_get(RowSum r, const RowSum* lds) {
  if (NW > 1) {
    // lane i takes the sum of wavefront i % NW (all NW of them in every lane would need 3 NW registers)
    const RowSum w = lds[threadIdx.x % NW];
    float C = w.c;
#pragma unroll
    for (int off = NW / 2; off > 0; off >>= 1) C = fminf(C, __shfl_xor(C, off, kWave));
    // (by the exponent: 2^d itself may underflow where the sum times it does not)
    const float d = C - w.c;
    const int shift = (int)fmaxf(d, -1000.f);
    r = RowSum{C, __builtin_amdgcn_ldexpf(w.z, shift), 0.f, true};
    if (TWO) r.a = __builtin_amdgcn_ldexpf(w.a, shift);
#pragma unroll
    for (int off = NW / 2; off > 0; off >>= 1) {
      r.z += __shfl_xor(r.z, off, kWave);
      if (TWO) r.a += __shfl_xor(r.a, off, kWave);
    }
  }
  const float all = TWO ? r.z + r.a : r.z;
  r.ok = all > 1e-30f && all < __builtin_inff() && r.c < kVrNoTerm;
  return r;
}

template <int NW, bool TWO>
__device__ __forceinline__ RowSum rowsum_block(float c, float z, float a, RowSum* lds) {
  const RowSum r = rowsum_put<NW, TWO>(c, z, a, lds);
  if (NW > 1) __syncthreads();
  return rowsum_get<NW, TWO>(r, lds);
}

// ln of the soft-max probability of a logit of the row.  The factor k stays as
// rounded, in the logit's own exponent too: what the rounding took then counts
// only for the logit's distance from the row's mean.
__device__ __forceinline__ Float2x rowsum_log_prob(const VocabRows& r, const RowSum& s, float x) {
#pragma clang fp contract(off)
  const Float2x p = two_mul(x, r.k), q = two_sum(p.hi, s.c);
  if (x < -1e38f && x > -__builtin_inff()) return Float2x{(float)((double)x * r.inv_T), 0.f};  // (x k may overflow)
  return ln_share(Float2x{q.hi, p.lo + q.lo}, s.z);
}

// One thread's terms of its registers: f(x, exponent) per element.
template <typename T, int NT, int KREG, typename F>
__device__ __forceinline__ void regs_each(RowRegs<T, NT, KREG>& r, const VocabGeom& g, F f) {
  constexpr int VEC = Vec16<T>::N;
#pragma unroll
  for (int j = 0; j < KREG; ++j) {
    if ((int)threadIdx.x + j * NT < (int)g.nvec) {
      forget(r.v[j]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f(to_f32(r.v[j].v[i]));
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <typename T, int NT, int KREG>
__device__ __forceinline__ RowSum regs_sum(RowRegs<T, NT, KREG>& r, const VocabGeom& g, float k, RowSum* lds) {
  const float c = regs_anchor<true>(r, g, k);
  float z = 0.f;
  auto add = [&](float x) { z += fast_exp2(fmaf(x, k, c)); };
  if (threadIdx.x < kWave) {  // the end elements
    add(r.h());
    add(r.t());
  }
  regs_each(r, g, add);
  return rowsum_block<NT / kWave, false>(c, z, 0.f, lds);
}

// grow[j] = f(x[j]) from registers, but for element `special` (or -1), which
// gets f_special(x).
template <typename T, int NT, int KREG, typename F, typename G>
__device__ __forceinline__ void regs_map(RowRegs<T, NT, KREG>& r, const VocabGeom& g, const T* row, T* grow, int64_t V,
                                         int special, F f, G f_special) {
  constexpr int VEC = Vec16<T>::N;
  if ((int)threadIdx.x < g.head)
    grow[threadIdx.x] = from_f32<T>((int)threadIdx.x == special ? f_special(r.h()) : f(r.h()));
  const int64_t t = g.tail0 + threadIdx.x;
  if (t < V) grow[t] = from_f32<T>((int)t == special ? f_special(r.t()) : f(r.t()));
  const bool gvec = (((uintptr_t)grow ^ (uintptr_t)row) & 15u) == 0;
  const int sv = special >= g.head ? (special - g.head) / VEC : -1;
  const int si = special - g.head - sv * VEC;
  const VecBuffer body = vec_buffer(grow + g.head, gvec ? (int)g.nvec : 0);
#pragma unroll
  for (int j = 0; j < KREG; ++j) {
    const int v = (int)threadIdx.x + j * NT;
    if (v < (int)g.nvec) {
      forget(r.v[j]);
      Vec16<T> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(f(to_f32(r.v[j].v[i])));
      if (v == sv) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (i == si) o.v[i] = from_f32<T>(f_special(to_f32(r.v[j].v[i])));
      }
      if (gvec) {
        vec_store(body, (uint32_t)v, o);
      } else {
        T* p = grow + g.head + v * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[i] = o.v[i];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// Sum of doubles over a workgroup of NW wavefronts, in a fixed order; every
// thread gets the result.
template <int NW>
__device__ __forceinline__ double block_sum_f64(double v, double* lds) {
  v = wave_sum_f64(v);
  if (NW == 1) return v;
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  double r = lds[threadIdx.x % NW];
#pragma unroll
  for (int off = NW / 2; off > 0; off >>= 1) r += __shfl_xor(r, off, kWave);
  return r;
}

// Rows longer than the registers hold, in pieces of NT * KREG vectors: f(vector,
// its place) for each, `later`(its vectors) in front of each piece but the first.
// The first piece is in r; a register that is done with takes the next piece's
// vector at once, so that loads are always under way.
template <typename T, int NT, int KREG, typename F, typename P>
__device__ __forceinline__ void long_each(RowRegs<T, NT, KREG>& r, const T* row, const VocabGeom& g, F f, P later) {
  constexpr int VEC = Vec16<T>::N;
  for (int64_t v0 = 0;; v0 += NT * KREG) {
    const int left = g.nvec - v0 < NT * KREG ? (int)(g.nvec - v0) : NT * KREG;
    const int64_t after = g.nvec - v0 - left;
    if (v0 > 0) later(left);
    const VecBuffer next = vec_buffer(row + g.head + (v0 + left) * VEC, after < NT * KREG ? (int)after : NT * KREG);
#pragma unroll
    for (int j = 0; j < KREG; ++j) {
      if ((int)threadIdx.x + j * NT < left) {
        forget(r.v[j]);
        f(r.v[j], v0 + threadIdx.x + j * NT);
      }
      if (after > 0) r.v[j] = vec_load<T>(next, threadIdx.x + j * NT);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (after == 0) return;
  }
}

// A sum over such a row's pieces, of one piece's sum at a time (see VocabStatSum):
// to = (to + z) 2^shift, and z starts again.
__device__ __forceinline__ void long_carry(float& to, float& z, int shift) {
  to = __builtin_amdgcn_ldexpf(to + z, shift);
  z = 0.f;
}

// regs_sum of such rows.
template <typename T, int NT, int KREG>
__device__ __forceinline__ RowSum long_sum(RowRegs<T, NT, KREG>& r, const T* row, const VocabGeom& g, float k, RowSum* lds) {
  constexpr int VEC = Vec16<T>::N;
  float c = regs_anchor<true>(r, g, k), before = 0.f, z = 0.f;
  auto add = [&](float x) { z += fast_exp2(fmaf(x, k, c)); };
  if (threadIdx.x < kWave) {
    add(r.h());
    add(r.t());
  }
  long_each(
      r, row, g,
      [&](const Vec16<T>& v, int64_t) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) add(to_f32(v.v[i]));
      },
      [&](int left) { long_carry(before, z, (int)regs_raise(r, left, k, c)); });
  return rowsum_block<NT / kWave, false>(c, before + z, 0.f, lds);
}

// This thread's share of sum(v[0..n)) when NT threads walk the array together, in
// a fixed order, eight loads in flight each.
template <int NT>
__device__ __forceinline__ double thread_share_of_sum_f64(const double* __restrict__ v, int64_t n) {
  constexpr int kInFlight = 8;
  double s = 0.0;
  for (int64_t i0 = threadIdx.x; i0 < n; i0 += (int64_t)NT * kInFlight) {
    double x[kInFlight];
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) {
      const int64_t i = i0 + (int64_t)j * NT;
      x[j] = i < n ? v[i] : 0.0;
    }
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) s += x[j];
  }
  return s;
}

// ---- sums over workgroups without a launch of their own ------------------------
// Every workgroup publishes its terms and draws a ticket; the one that draws the
// last adds all the terms up, in the order of their places, so that the sum does
// not depend on who that is.  The ticket counter is 0 when the kernel starts (a
// kernel in front clears it).  For kernels of few workgroups: two chained
// atomics in each of 8192 rows cost the policy loss 40 us, the launch it saves 5.

// The exchange's old value is waited for, so the term has arrived on return.
__device__ __forceinline__ void publish_term(double* at, double term) {
  unsigned long long* p = reinterpret_cast<unsigned long long*>(at);
  const unsigned long long old = __hip_atomic_exchange(p, (unsigned long long)__double_as_longlong(term),
                                                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("" : : "v"((uint32_t)old), "v"((uint32_t)(old >> 32)) : "memory");
}
__device__ __forceinline__ unsigned draw_ticket(unsigned* ticket) {
  return __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The workgroup of the last caller: the sum of all terms, in every thread.
template <int NT>
__device__ __forceinline__ double sum_terms(const double* terms, int64_t n, double* lds) {
  constexpr int kInFlight = 8;
  const unsigned long long* p = reinterpret_cast<const unsigned long long*>(terms);
  double s = 0.0;
  for (int64_t i0 = threadIdx.x; i0 < n; i0 += (int64_t)NT * kInFlight) {
    unsigned long long x[kInFlight];
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) {
      const int64_t i = i0 + (int64_t)j * NT;
      x[j] = i < n ? __hip_atomic_load(p + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0ull;
    }
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) s += __longlong_as_double((long long)x[j]);
  }
  return block_sum_f64<NT / kWave>(s, lds);
}

// How a row of V elements of T is held: threads and vectors per thread of the
// smallest arrangement it fits, 0 threads for rows that fit none.
struct RowShape {
  int nt, kreg;
};
template <typename T>
inline RowShape row_shape(int64_t V) {
  const int64_t vecs = V / Vec16<T>::N;
  if (vecs <= 64 * 4) return RowShape{64, 4};
  if (vecs <= 256 * 4) return RowShape{256, 4};
  if (vecs <= 256 * 8) return RowShape{256, 8};
  if (vecs <= 512 * 8) return RowShape{512, 8};
  if (vecs <= 1024 * 8) return RowShape{1024, 8};
  if (vecs <= 1024 * 16) return RowShape{1024, 16};
  return RowShape{0, 0};
}

}  // namespace ts

// return call with T bound to the storage type of a dtype code
#define TS_BY_DTYPE(dtype, call)                         \
  switch (dtype) {                                       \
    case TS_F32: { using T = float; return call; }       \
    case TS_BF16: { using T = ts::bf16_t; return call; } \
    default: { using T = ts::f16_t; return call; }       \
  }
