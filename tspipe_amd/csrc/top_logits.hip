// Sparse teachers: the k largest logits of each row with the row's log-sum-exp,
// and the distillation loss from such rows, forward and backward.
#include "vocab_rows.h"

namespace ts {

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
  constexpr int VEC = Vec16<T>::N;
  const VocabGeom g = vocab_geom(row, V);
  int c = 0;
  if ((int)threadIdx.x < g.head) c += f(to_f32(row[threadIdx.x]), (int)threadIdx.x) ? 1 : 0;
  const int64_t t = g.tail0 + threadIdx.x;
  if (t < V) c += f(to_f32(row[t]), (int)t) ? 1 : 0;
#pragma unroll 1
  for (int64_t v = threadIdx.x; v < g.nvec; v += NT) {
    const int64_t e0 = g.head + v * VEC;
    const Vec16<T> r = load16(row + e0);
#pragma unroll
    for (int i = 0; i < VEC; ++i) c += f(to_f32(r.v[i]), (int)(e0 + i)) ? 1 : 0;
  }
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

// Short rows come in two arrangements.  FEW, one wavefront, for k up to kTopFew:
// at most 88 of its vectors reach the bar, but for equal logits, and 10 KB of LDS
// are enough.  For larger k, up to the whole row, 256 threads with a vector each.
// (One wavefront with the LDS for a whole row, 26 KB: 8192 x 1000 bf16 k = 64
// takes 63 us instead of 30, k = 128 234 instead of 64.)
constexpr int kTopFew = 64;

// Vectors with a candidate, candidates, and candidates to rank that a row may
// have at a time.
template <int NT, int KREG>
constexpr int top_hit_cap() { return NT == 64 ? 128 : KREG == 1 ? 256 : NT == 256 ? 512 : 1024; }
template <int NT, int KREG>
constexpr int top_cand_cap() { return NT == 64 ? 768 : KREG == 1 ? 2304 : 1536; }
template <int NT>
constexpr int top_rank_cap() { return NT == 64 ? 256 : 2 * kTopMax; }

// Groups per thread when k is large: short rows have few vectors per thread, and
// a group each gives the bar they need (1000 bf16, k = 64, one group per thread:
// 64 groups, 600 candidates, 456 us for 8192 rows); a thread with one vector makes
// four groups of that.
template <int NT>
constexpr int top_groups() { return NT <= 256 ? 4 : 2; }

template <int NT, int KREG>
struct TopShared {
  static constexpr int kMost = NT == 64 ? kTopFew : kTopMax;  // k
  static constexpr int kKept = kMost + kMost / 8 + 4;         // what top_refine leaves
  union {
    uint32_t group[top_groups<NT>() * NT];  // order numbers of the groups' maxima
    uint64_t kept[kKept];
    u32x4 hit[top_hit_cap<NT, KREG>()];  // vectors with a candidate
  };
  int hit_at[top_hit_cap<NT, KREG>()];  // their first elements' places
  alignas(16) uint64_t cand[top_cand_cap<NT, KREG>()];  // order number and place, larger for smaller places
  RowSum sums[NT / kWave];
  VocabStat stats[NT / kWave];
  int counts[NT / kWave];
  int rank[top_rank_cap<NT>()];
  int n, n_hit;
  float bar;
};

// Ranks the n candidates by counting, for each one, those that are larger; the
// first k leave.  With fewer candidates than threads several threads count for
// each.  256 threads with more of them than threads count for two at a reading of
// two: reading bounds it there (8192 x 4000 bf16, k = 256: 145 us, one by one 185;
// with fewer candidates that is slower, 8192 x 1000 and k = 128 73 us, one by one
// 64).  sh.rank is 0 on entry.
template <typename T, int NT, int KREG>
__device__ __forceinline__ void top_emit(TopShared<NT, KREG>& sh, int n, const T* x, int64_t row, int k,
                                         T* __restrict__ values, int32_t* __restrict__ indices) {
  constexpr int NW = NT / kWave;
  const int all = __builtin_amdgcn_readfirstlane(n);
  const int waves = (all + kWave - 1) / kWave;  // wavefronts that hold one candidate a lane
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  int part = 0, first = wave, parts = 1;
  if (waves < NW) {
    parts = 0;
    for (int w = waves; w <= NW; w += waves) ++parts;
    for (; first >= waves; first -= waves) ++part;
  }
  const int per = ((int)(((float)all + (float)parts - 0.5f) / (float)parts) + 1) & ~1;  // all / parts, rounded up, even
  const int lo = part * per, hi = part < parts ? (lo + per < all ? lo + per : all) : lo;
  if (NT == 256 && all > NT) {  // uniform; at most twice as many
    const int c0 = (int)threadIdx.x, c1 = c0 + NT;
    const uint64_t me0 = sh.cand[c0], me1 = c1 < all ? sh.cand[c1] : ~0ull;
    int rank0 = 0, rank1 = 0, i = 0;
#pragma unroll 2
    for (; i + 1 < all; i += 2) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&sh.cand[i]);
      rank0 += (int)(two.x > me0) + (int)(two.y > me0);
      rank1 += (int)(two.x > me1) + (int)(two.y > me1);
    }
    if (i < all) {
      rank0 += (int)(sh.cand[i] > me0);
      rank1 += (int)(sh.cand[i] > me1);
    }
    sh.rank[c0] = rank0;
    if (c1 < all) sh.rank[c1] = rank1;
  } else {
    for (int c = first * kWave + (int)threadIdx.x % kWave; c < all; c += NT) {
      const uint64_t me = sh.cand[c];
      int rank = 0, i = lo;
#pragma unroll 2
      for (; i + 1 < hi; i += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&sh.cand[i]);
        rank += (int)(two.x > me) + (int)(two.y > me);
      }
      if (i < hi) rank += (int)(sh.cand[i] > me);
      if (rank) atomicAdd(&sh.rank[c], rank);
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += NT) {
    const int rank = sh.rank[c];
    if (rank < k) {
      const uint64_t me = sh.cand[c];
      const int32_t i = (int32_t)~(uint32_t)me;
      const uint32_t key = (uint32_t)(me >> 32);
      indices[row * k + rank] = i;
      // (the order number is the logit but for a zero's sign and a NaN's bits)
      values[row * k + rank] = key == 0x80000000u || key == 0xffffffffu ? x[i] : from_f32<T>(top_unkey(key));
    }
  }
}

// Rows with a NaN, with a sum that needs the true maximum, or of which more
// vectors or candidates reach the bar than fit: thousands of equal logits at the
// border, fewer than k logits above -inf or the type's lowest value, the best
// behind the first piece (2048 x 30522 fp32 in rising order: 1.8 ms).  The k-th
// largest order number is the bar's, if fewer than k elements exceed the bar (a
// vocabulary masked but for fewer than k tokens), or found bit by bit (the largest
// t such that at least k elements reach it); then the place up to which elements
// equal to it are taken is found likewise, and the k elements so defined are
// collected.  (4096 x 30522 bf16 with 30 tokens not masked, k = 64: 0.66 ms;
// all of it bit by bit, an element a thread: 3.3.)
template <typename T, int NT, int KREG>
__device__ __forceinline__ void top_row_walked(const VocabRows& a, int64_t row, const T* x, int k,
                                               T* __restrict__ values, int32_t* __restrict__ indices,
                                               float* __restrict__ lse, TopShared<NT, KREG>& sh) {
  const int64_t V = a.V;
  if (lse) {
    const VocabStat s = vstat_block<NT / kWave>(vocab_stat_walk<T, NT>(x, V, a.k), a.k, sh.stats);
    const Float2x lz = log2_2x(s.z);  // (for -inf throughout, z = 0 and m is a stand-in)
    float l = (float)((double)s.m * a.inv_T + kVrLn2 * ((double)lz.hi + (double)lz.lo));
    if (s.m == __builtin_inff() &&  // uniform
        top_count<T, NT>(x, V, sh.counts, [](float v, int) { return v != v; }) == 0)
      l = s.m;
    if (threadIdx.x == 0) lse[row] = l;
  }
  const float bar = sh.bar;
  uint32_t t = top_key(bar);
  int above = top_count<T, NT>(x, V, sh.counts, [=](float v, int) { return !(v <= bar); });
  if (above >= k) {  // uniform
    t = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = t | (1u << bit);
      if (top_count<T, NT>(x, V, sh.counts, [=](float v, int) { return top_key(v) >= c; }) >= k) t = c;
    }
    above = top_count<T, NT>(x, V, sh.counts, [=](float v, int) { return top_key(v) > t; });
  }
  int place = 0;  // the largest place such that fewer than k - above elements equal to t lie before it
  for (int bit = 31 - __builtin_clz((uint32_t)V); bit >= 0; --bit) {
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
      if (at < sh.kMost) sh.cand[at] = ((uint64_t)key << 32) | (uint32_t)~(uint32_t)i;
    }
  }
  __syncthreads();
  top_emit<T>(sh, k, x, row, k, values, indices);
}

// Reduces n > k candidates to the k largest, or some more that can be ranked:
// the search for the border ends as soon as that is so (to the last bit, a row of
// 1000 candidates takes twice as long).
template <int NT, int KREG>
__device__ __forceinline__ void top_refine(TopShared<NT, KREG>& sh, int n, int k) {
  static_assert(sizeof(sh.kept) <= sizeof(sh.hit), "no LDS of its own");
  uint64_t t = 0;
  const int enough = k + k / 8 + 4;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t c = t | (1ull << bit);
    int m = 0;
    if (NT == kWave) {
      for (int i0 = 0; i0 < n; i0 += kWave) {
        const int i = i0 + (int)threadIdx.x;
        m += (int)__popcll(__ballot(i < n && sh.cand[i < n ? i : 0] >= c));
      }
    } else {
      for (int i = threadIdx.x; i < n; i += NT) m += sh.cand[i] >= c;
#pragma unroll
      for (int off = kWave / 2; off > 0; off >>= 1) m += __shfl_xor(m, off, kWave);
      __syncthreads();
      if (threadIdx.x % kWave == 0) sh.counts[threadIdx.x / kWave] = m;
      __syncthreads();
      m = 0;
      for (int i = 0; i < NT / kWave; ++i) m += sh.counts[i];
    }
    if (m >= k) {  // uniform
      t = c;
      if (m <= enough) break;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT)
    if (sh.cand[i] >= t) {
      const int at = atomicAdd(&sh.n, 1);
      if (at < sh.kKept) sh.kept[at] = sh.cand[i];  // (places differ, so that k or at most `enough` reach t)
    }
  __syncthreads();
  const int left = sh.n;
  for (int i = threadIdx.x; i < left; i += NT) sh.cand[i] = sh.kept[i];
  __syncthreads();
}

// The largest order number (to within the `enough` that end the search early)
// that at least k of a wavefront's numbers reach, N of them a lane; 0 when
// fewer than k are above `floor`.  Called by one whole wavefront.
template <int N>
__device__ __forceinline__ uint32_t top_bar(const uint32_t (&key)[N], int k, uint32_t floor) {
  uint32_t t = 0;
  const int enough = k + k / 8 + 4;
  int some = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) some += (int)__popcll(__ballot(key[i] > floor));
  if (some < k) return 0u;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cnd = t | (1u << bit);
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) cnt += (int)__popcll(__ballot(key[i] >= cnd));
    if (cnt >= k) {
      t = cnd;
      if (cnt <= enough) break;
    }
  }
  return t;
}

// Elements that reach the bar, of the vectors noted since the last call, become
// candidates; false when they do not all fit.  With many more vectors noted
// than k the bar first rises to the k-th largest of their maxima: ranking costs
// the square of the candidates (k = 128 of 131072 in two pieces, 270 of them:
// 22 of 105 us).
template <typename T, bool LAST, bool MULTI, int NT, int KREG>
__device__ __forceinline__ bool top_expand(TopShared<NT, KREG>& sh, int k) {
  constexpr int VEC = Vec16<T>::N, kCap = top_cand_cap<NT, KREG>(), kHits = top_hit_cap<NT, KREG>();
  typedef RawMax<T> Raw;
  __syncthreads();
  const int hits = sh.n_hit;
  if (hits > kHits) return false;  // uniform
  if (MULTI && hits > k + k / 2) {
    constexpr int N = (kHits + kWave - 1) / kWave / 2;
    if (hits <= N * kWave && threadIdx.x < kWave) {
      uint32_t key[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = i * kWave + (int)threadIdx.x;
        key[i] = 0u;
        if (at < hits) {
          Vec16<T> v;
          __builtin_memcpy(&v, &sh.hit[at], 16);
          key[i] = top_key(Raw::value(Raw::of(v), Raw::least(v)));
          if (key[i] == 0xffffffffu) key[i] = 0u;  // a NaN sets no bar
        }
      }
      const uint32_t t = top_bar<N>(key, k, top_key(sh.bar));
      if (threadIdx.x == 0 && t) sh.bar = fmaxf(sh.bar, top_unkey(t));
    }
    __syncthreads();
  }
  const float bar = sh.bar;
  for (int e = threadIdx.x; e < hits * VEC; e += NT) {
    const T* v = reinterpret_cast<const T*>(&sh.hit[e / VEC]);
    const float x = to_f32(v[e % VEC]);
    if (x >= bar) {
      const int at = atomicAdd(&sh.n, 1);
      if (at < kCap) sh.cand[at] = ((uint64_t)top_key(x) << 32) | (uint32_t)~(uint32_t)(sh.hit_at[e / VEC] + e % VEC);
    }
  }
  __syncthreads();
  const int n = sh.n;
  if (n > kCap) return false;
  // (a single wavefront ranks slowly: it narrows its candidates down sooner)
  const bool narrow = n > top_rank_cap<NT>() || (NT == kWave && n > 192 && n > k + k / 4);
  if (LAST && !narrow) return true;
  __syncthreads();  // (nobody changes it before everybody has read it)
  if (threadIdx.x == 0) sh.n_hit = 0;
  if (narrow) top_refine(sh, n, k);
  __syncthreads();
  return true;
}

// One pass over a row by one workgroup, in pieces of NT * KREG vectors.  The
// first piece gives a bar: the threads' maxima (several each when k is large) are
// elements of disjoint groups, so the k-th largest of them is reached by at
// least k elements.  Every element that reaches the bar is a candidate -- few
// more than k, since the best k mostly lie in different groups (k = 64 of 512
// groups: 68 expected) -- and the candidates' ranks are counted.  The row's sum
// is taken in the same walk over the registers.
//
// The walk is bound by its vector instructions, four of every seven an
// exponential's.  So the maxima compare raw bits, two 16-bit logits at a time,
// and a vector that reaches the bar is only noted; its elements are looked at
// when the noted vectors are spread over all threads.
//
// MULTI: the row has more than one piece.  Eight wavefronts a SIMD, so 64
// registers, which the forms of one piece fit; that of several leaves three or four
// in scratch memory (16 to 20 bytes a thread; with its sum over pieces in a register
// up to 20, 2048 x 30522 fp32 75 us instead of 61).  With 80 and six wavefronts 4096 x
// 30522 bf16 took 67 us instead of 58 (55 by now), 1024 x 131072 96 instead of 79
// (75 by now).
template <typename T, int NT, int KREG, bool MULTI>
__global__ __launch_bounds__(NT, NT > 256 ? 8 : 1) void top_logits_kernel(const VocabRows a, int k,
                                                                          T* __restrict__ values,
                                                                          int32_t* __restrict__ indices,
                                                                          float* __restrict__ lse) {
  constexpr int VEC = Vec16<T>::N;
  typedef RawMax<T> Raw;
  __shared__ TopShared<NT, KREG> sh;
  __shared__ float before[MULTI ? NT : 1];  // each thread's sum over earlier pieces, added to without a register
  const int64_t row = blockIdx.x, V = a.V;
  const T* x = vocab_row<T>(a, row);
  const VocabGeom g = vocab_geom(x, V);
  const float kk = a.k;
  const int tid = threadIdx.x;
  constexpr int G = top_groups<NT>();
  const bool many = k > NT / 4;  // G groups per thread, else one
  RowRegs<T, NT, KREG> r;
  regs_load(r, x, V, g);
  if (tid == 0) sh.n = sh.n_hit = 0;
  for (int i = tid; i < top_rank_cap<NT>(); i += NT) sh.rank[i] = 0;
  const float c = regs_anchor<false>(r, g, kk);
  float z = 0.f;
  auto add = [&](float xv) { z += fast_exp2(fmaf(xv, kk, c)); };
  if (tid < kWave) {
    add(r.h());
    add(r.t());
  }
  // the first piece: its sum, the groups' maxima, the bar
  const int n0 = g.nvec < NT * KREG ? (int)g.nvec : NT * KREG;
  int32_t mx[G];
#pragma unroll
  for (int q = 0; q < G; ++q) mx[q] = Raw::kNone;
#pragma unroll
  for (int j = 0; j < KREG; ++j) {
    if (tid + j * NT < n0) {
      forget(r.v[j]);
      if (KREG == 1)
        __builtin_memcpy(mx, &r.v[j], 16);
      else
        mx[j * G / KREG] = Raw::max2(mx[j * G / KREG], Raw::of(r.v[j]));
#pragma unroll
      for (int i = 0; i < VEC; ++i) add(to_f32(r.v[j].v[i]));
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (MULTI) {
    before[tid] = z;
    z = 0.f;
  }
  auto publish = [&](auto group_max) {
    uint32_t whole = r.has_h || r.has_t ? top_key(fmaxf(r.h(), r.t())) : 0u;
#pragma unroll
    for (int q = 0; q < G; ++q) {
      uint32_t key = 0u;
      if (tid + (KREG == 1 ? 0 : q * (KREG / G) * NT) < n0) {  // (a NaN sets no bar)
        const float f = group_max(q);
        key = f == f ? top_key(f) : 0u;
      }
      if (many && q > 0) sh.group[q * NT + tid] = key;
      if (!many || q == 0) whole = key > whole ? key : whole;
    }
    sh.group[tid] = whole;
  };
  auto search = [&](uint32_t floor) {
    __syncthreads();
    if (tid < kWave) {
      // in registers: read from LDS for every bit, 4096 rows of 30522 took 76 us instead of 57
      constexpr int kOne = NT / kWave, kAll = G * NT / kWave;
      uint32_t one[kOne], t;
#pragma unroll
      for (int i = 0; i < kOne; ++i) one[i] = sh.group[i * kWave + tid];
      if (many) {  // uniform
        uint32_t all[kAll];
#pragma unroll
        for (int i = 0; i < kAll; ++i) all[i] = i < kOne ? one[i] : sh.group[i * kWave + tid];
        t = top_bar<kAll>(all, k, floor);
      } else {
        t = top_bar<kOne>(one, k, floor);
      }
      if (tid == 0) sh.bar = top_unkey(t);
    }
    __syncthreads();
  };
  publish([&](int q) { return Raw::value(mx[q]); });
  search(top_key(0.f));
  // By raw bits a group has its own maximum if it has a logit above zero, and its smallest logit if not.  With
  // k such groups that makes no difference: the others are below the bar.  Else no bar was found, and the
  // maxima are taken again, of the groups without such a logit by the smallest raw bits.  (With a bar from the
  // first maxima nearly every vector reaches it: 4096 x 30522 bf16, k = 64, logits about -40 took 1740 us; now
  // 62, and 57 where they are about 0.)
  if (!(sh.bar > 0.f)) {  // uniform
    int32_t mn[G];
#pragma unroll
    for (int q = 0; q < G; ++q) mx[q] = Raw::kNone, mn[q] = -1;
    if (KREG == 1) {
      __builtin_memcpy(mx, &r.v[0], 16);
      __builtin_memcpy(mn, &r.v[0], 16);
    } else {
#pragma unroll
      for (int j = 0; j < KREG; ++j) {
        if (tid + j * NT < n0) {
          mx[j * G / KREG] = Raw::max2(mx[j * G / KREG], Raw::of(r.v[j]));
          mn[j * G / KREG] = Raw::min2(mn[j * G / KREG], Raw::least(r.v[j]));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    publish([&](int q) { return Raw::value(mx[q], mn[q]); });
    search(top_key(-__builtin_inff()));
  }
  const float bar = sh.bar;
  // A logit that reaches a bar above zero exceeds `limit` by its raw bits as a signed number; one that reaches
  // another bar lies below `limit` by them as an unsigned number (so do all above zero).
  const bool raw = bar > 0.f;
  int32_t limit;  // (twice, for 16-bit types)
  if constexpr (sizeof(T) == 4) {
    limit = raw ? __float_as_int(bar) - 1 : __float_as_int(bar == 0.f ? -0.f : bar) + 1;
  } else {
    const T t = from_f32<T>(bar == 0.f ? -0.f : bar);
    uint16_t bits;
    __builtin_memcpy(&bits, &t, 2);
    uint32_t b;
    if (raw)  // two steps below the rounded bar: rounding may have gone up; the elements are compared exactly later
      b = bits > 1 ? bits - 2u : 0u;
    else  // the least logit that reaches the bar, and one: a step of 16-bit logits far below zero holds many of them
      b = bits + (to_f32(t) < bar ? 0u : 1u);
    limit = (int32_t)(b * 0x10001u);
  }
  auto take = [&](float xv, int i) {
    if (xv >= bar) {
      const int at = atomicAdd(&sh.n, 1);
      if (at < top_cand_cap<NT, KREG>()) sh.cand[at] = ((uint64_t)top_key(xv) << 32) | (uint32_t)~(uint32_t)i;
    }
  };
  if (tid < g.head) take(r.h(), tid);
  if (g.tail0 + tid < V) take(r.t(), (int)g.tail0 + tid);
  auto reaches = [&](const Vec16<T>& v) {
    return raw ? Raw::max2(Raw::of(v), limit) != limit : Raw::min2(Raw::least(v), limit) != limit;
  };
  // Candidates, piece by piece.  A register that is done with takes the next piece's vector at once, so
  // that loads are always under way; later pieces are summed in this walk.
  bool fits = true;
  for (int64_t v0 = 0; fits; v0 += NT * KREG) {
    const int left = !MULTI ? n0 : g.nvec - v0 < NT * KREG ? (int)(g.nvec - v0) : NT * KREG;
    const int64_t after = MULTI ? g.nvec - v0 - left : 0;  // vectors behind this piece
    const VecBuffer next = vec_buffer(x + g.head + (v0 + left) * VEC, after < NT * KREG ? (int)after : NT * KREG);
#pragma unroll
    for (int j = 0; j < KREG; ++j) {
      if (tid + j * NT < left) {
        forget(r.v[j]);
        if (reaches(r.v[j])) {
          const int at = atomicAdd(&sh.n_hit, 1);
          if (at < top_hit_cap<NT, KREG>()) {
            __builtin_memcpy(&sh.hit[at], &r.v[j], 16);
            sh.hit_at[at] = g.head + ((int)v0 + tid + j * NT) * VEC;
          }
        }
        if (MULTI && v0 > 0) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) add(to_f32(r.v[j].v[i]));
        }
      }
      if (MULTI && after > 0) r.v[j] = vec_load<T>(next, tid + j * NT);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!MULTI || after == 0) break;
    __hip_atomic_fetch_add(&before[tid], z, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    z = 0.f;
    if ((v0 / (NT * KREG)) % 2 == 1) fits = top_expand<T, false, MULTI>(sh, k);
  }
  if (MULTI) z += before[tid];
  const RowSum mine = rowsum_put<NT / kWave, false>(c, z, 0.f, sh.sums);
  fits = fits && top_expand<T, true, MULTI>(sh, k);
  const RowSum s = rowsum_get<NT / kWave, false>(mine, sh.sums);
  if (!s.ok || !fits) {
    __syncthreads();
    for (int i = tid; i < top_rank_cap<NT>(); i += NT) sh.rank[i] = 0;
    top_row_walked<T>(a, row, x, k, values, indices, lse, sh);
    return;
  }
  if (tid == 0 && lse) {
    const Float2x l = rowsum_log_prob(a, s, 0.f);  // the log probability of a logit of 0
    // What k's rounding took is that much of the row's mean; the log-sum-exp stands in for it, a few units away.
    lse[row] = -(l.hi + fmaf(l.hi, a.k_rel, l.lo));
  }
  top_emit<T>(sh, sh.n, x, row, k, values, indices);
}

// ---- distillation from a teacher's largest logits ----------------------------------

// A row's teacher: sum p ln p over its entries (and of the rest r = 1 - sum p,
// r ln r), the probabilities' whole sum, and r.
struct TopTeacher {
  double p_ln_p;
  float whole, rest;
};

struct TopDistilArgs {
  VocabRows r;
  const void* t_values;
  int t_dtype;
  const int32_t* t_indices;
  const float* t_lse;  // null: the kept entries' probabilities are normalised among themselves
  int k;
  const uint8_t* mask;  // may be null
  float gscale;         // weight * T
  int* live;            // rows of the mask
  TopTeacher* teacher;  // per row
  float* entry_p;       // per entry: the probability of all the row's entries for its token; -1 if absent or not the first of them
  double* row_loss;
  struct TopRowGrad* row_grad;  // per row, for rows too long for registers
  void* grad;  // may be null
};

// A row's gradient: go 2^(x k + off) of the tokens without an entry, and rz times
// that power a token's probability; of walked rows go 2^((x - off) k), off the
// largest of these tokens' logits, and with off_all, the row's, a probability.
struct TopRowGrad {
  float off, go, rz, off_all;
  int by_max, unused;  // (a multiple of 8 bytes)
  __device__ __forceinline__ float other(float x, float k) const {
    return go * fast_exp2(by_max ? (x - off) * k : fmaf(x, k, off));
  }
  __device__ __forceinline__ float prob(float x, float k) const {
    return rz * fast_exp2(by_max ? (x - off_all) * k : fmaf(x, k, off));
  }
};

__device__ __forceinline__ float top_value(const void* v, int dtype, int64_t i) {
  if (dtype == TS_F32) return reinterpret_cast<const float*>(v)[i];
  if (dtype == TS_BF16) return to_f32(reinterpret_cast<const bf16_t*>(v)[i]);
  return to_f32(reinterpret_cast<const f16_t*>(v)[i]);
}

// Everything that depends on the teacher alone, in 64 bits (what the teacher
// leaves to all other tokens is one minus a sum), one wavefront per row.  In a
// launch of its own because these few numbers per row would otherwise set the
// registers, and with them the occupancy, of the kernel that holds the
// student's row.  The last workgroup counts the mask.
//
// Whether a token is named twice costs the square of the entries to find out, so
// they are first put into a hash table in LDS (open addressing, half full at
// most), and only a row in which two meet is compared throughout (8192 rows of 256
// entries: 62 us without the table, 18 with it; of 64: 12 and 9.4).
constexpr int kTeacherBlock = 256, kTeacherSlots = 2 * kTopMax;

__global__ __launch_bounds__(kTeacherBlock) void top_teacher_kernel(const TopDistilArgs a) {
  constexpr int NE = kTopMax / kWave;
  __shared__ __align__(16) int ent_idx[kTeacherBlock / kWave][kTopMax];
  __shared__ float ent_p[kTeacherBlock / kWave][kTopMax];
  __shared__ int slots[kTeacherBlock / kWave][kTeacherSlots];
  __shared__ float lds_f[kTeacherBlock / kWave];
  if (blockIdx.x == gridDim.x - 1) {
    const float n = a.mask ? mask_count_block<kTeacherBlock>(a.mask, a.r.n_rows, lds_f) : (float)a.r.n_rows;
    if (threadIdx.x == 0) *a.live = (int)n;
    return;
  }
  const int w = threadIdx.x / kWave, lane = threadIdx.x % kWave, k = a.k;
  const int64_t row = (int64_t)blockIdx.x * (kTeacherBlock / kWave) + w;
  const bool on = row < a.r.n_rows && !(a.mask && a.mask[row] == 0);
  int idx[NE];
  float v[NE], p[NE];
  float m = kVrLowest;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int at = lane + i * kWave;
    idx[i] = -1;
    v[i] = p[i] = 0.f;
    if (i * kWave < k) {  // uniform
      if (on && at < k) {
        idx[i] = a.t_indices[row * k + at];
        v[i] = top_value(a.t_values, a.t_dtype, row * k + at);
        if (idx[i] < 0 || idx[i] >= a.r.V) idx[i] = -1;
        if (idx[i] >= 0) m = fmaxf(m, v[i]);
      }
    }
  }
  // p = e^(v / T - off) / z; without a log-sum-exp z is the entries' own sum
  double off, z = 1.0;
  if (a.t_lse) {
    off = on ? (double)a.t_lse[row] : 0.0;
  } else {
    m = wave_max(m);
    off = (double)m * a.r.inv_T;
    z = 0.0;
  }
  double pd[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    pd[i] = 0.0;
    if (i * kWave < k && idx[i] >= 0 && v[i] != -__builtin_inff()) {
      pd[i] = exp((double)v[i] * a.r.inv_T - off);
      if (!a.t_lse) z += pd[i];
    }
  }
  if (!a.t_lse) z = wave_sum_f64(z);
  const double rz = z > 0.0 ? 1.0 / z : (z == 0.0 ? 0.0 : z), lz = off + (a.t_lse ? 0.0 : log(z));
  double sum = 0.0, p_ln_p = 0.0;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    if (i * kWave < k) {
      p[i] = (float)(pd[i] * rz);
      sum += pd[i] * rz;
      // with p as it was rounded, so that p ln p - p ln q keeps its difference's accuracy
      if (p[i] != 0.f) p_ln_p += (double)p[i] * ((double)v[i] * a.r.inv_T - lz);
    }
    ent_idx[w][lane + i * kWave] = idx[i];
    ent_p[w][lane + i * kWave] = p[i];
  }
  sum = wave_sum_f64(sum);
  p_ln_p = wave_sum_f64(p_ln_p);
  for (int i = lane; i < kTeacherSlots; i += kWave) slots[w][i] = -1;
  __syncthreads();
  bool twice = false;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    if (idx[i] < 0) continue;
    // (at most kTopMax slots are ever taken, so every search ends at a free one)
    for (uint32_t h = ((uint32_t)idx[i] * 2654435761u) / (0x80000000u / (kTeacherSlots / 2));; ++h) {
      const int there = atomicCAS(&slots[w][h % kTeacherSlots], -1, idx[i]);
      twice = twice || there == idx[i];
      if (there == -1 || there == idx[i]) break;
    }
  }
  twice = __any(twice);
  // the same token named twice: the first naming stands for all of them.  Every entry is compared with
  // all others, four at a read; only a second naming takes the branch.
  float all[NE];
  bool first[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    all[i] = p[i];
    first[i] = idx[i] >= 0;
  }
#pragma unroll 4
  for (int q0 = 0; twice && q0 < k; q0 += 4) {  // (entries from k on are absent)
    const int4 other = *reinterpret_cast<const int4*>(&ent_idx[w][q0]);
    const int o[4] = {other.x, other.y, other.z, other.w};
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      if (i * kWave >= k) break;  // uniform
      const int self = lane + i * kWave - q0;  // (out of 0..3 mostly)
      bool again = false;
#pragma unroll
      for (int q = 0; q < 4; ++q) again = again || (o[q] == idx[i] && q != self);
      if (again && idx[i] >= 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (o[q] == idx[i] && q != self) {
            first[i] = first[i] && q > self;
            all[i] += ent_p[w][q0 + q];
          }
      }
    }
  }
  int distinct = 0;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int at = lane + i * kWave;
    if (on && at < k) a.entry_p[row * k + at] = first[i] ? all[i] : -1.f;
    distinct += first[i];
  }
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) distinct += __shfl_xor(distinct, o, kWave);
  if (!on || lane != 0) return;
  // (nothing is left over where every token has an entry)
  const float rest = a.t_lse && distinct < a.r.V ? (float)fmax(1.0 - sum, 0.0) : 0.f;
  if (rest > 0.f) p_ln_p += (double)rest * log((double)rest);
  a.teacher[row] = TopTeacher{p_ln_p, (float)(sum + (double)rest), rest};
}

// Error of a log-sum-exp: that of one of top_logits before its rounding, and of the rounding, a step of fp32.
constexpr float kTopLseError = 4e-6f, kTopLseRounding = 1.1920929e-07f;
// ln of a share of the student's probability, 1e-30, below which a remainder no larger than that is none.
constexpr float kTopOutOfReach = -69.f;

template <int NT>
struct TopDistilShared {
  RowSum sums[NT / kWave];
  VocabStat stats[NT / kWave];
  double d[NT / kWave];
};

// Bit of element j in the marks: vector v of the row owns bits 8 + v * VEC on, so
// that a vector's marks are one byte (or half of one).
__device__ __forceinline__ uint32_t top_mark_bit(int j, const VocabGeom& g) { return (uint32_t)(j - g.head + 8); }

// LONG rows do not fit the registers: this kernel then reads them in pieces and
// leaves the gradient to two others.
//
// Registers: 80 in the 512-thread arrangement, of which six wavefronts a SIMD
// are resident instead of eight (4096 x 30522 bf16 with 85 % of the rows, other
// classes as one outcome: 88 us, 505 MB at 5.7 TB/s; when 80 took 92, 64 took 99).
// Two rows of 1024 threads with eight vectors each share a CU at 64 registers; one
// or two of them are in scratch memory, four in the bf16 form with the other classes
// (13 with a row's sums in vector registers: 2044 x 50257 bf16 108 instead of 106 us a
// call, 4096 x 30522 fp32 208 instead of 204).
template <typename T, int NT, int KREG, bool LONG, bool TAIL>
__global__ __launch_bounds__(NT, (KREG > 8 || LONG ? 4 : NT > 256 ? (NT > 512 ? 8 : 6) : 1)) void top_distil_kernel(
    const TopDistilArgs a) {
  constexpr int NW = NT / kWave, NE = (kTopMax + NT - 1) / NT, VEC = Vec16<T>::N;
  extern __shared__ uint32_t marks[];  // TAIL: a bit per vocabulary entry
  __shared__ TopDistilShared<NT> sh;
  const int64_t row = blockIdx.x, V = a.r.V;
  const int tid = threadIdx.x, k = a.k;
  T* grow = a.grad ? reinterpret_cast<T*>(a.grad) + row * V : nullptr;
  if (a.mask && a.mask[row] == 0) {
    if (tid == 0) a.row_loss[row] = 0.0;
    if (grow && !LONG) vocab_zero_row<T, NT>(grow, V);
    return;
  }
  const T* x = vocab_row<T>(a.r, row);
  const VocabGeom g = vocab_geom(x, V);
  const float kk = a.r.k;
  RowRegs<T, NT, KREG> r;
  int idx[NE];
  float p[NE];  // the teacher's probability of the token
  T xe[NE];     // the student's logit
  auto ex = [&](int i) { return to_f32(xe[i]); };
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int at = tid + i * NT;
    p[i] = -1.f;
    idx[i] = -1;
    if (at < k) {
      p[i] = a.entry_p[row * k + at];
      idx[i] = a.t_indices[row * k + at];
    }
  }
  regs_load(r, x, V, g);
#pragma unroll
  for (int i = 0; i < NE; ++i)
    if (p[i] < 0.f) idx[i] = -1;
#pragma unroll
  for (int i = 0; i < NE; ++i) xe[i] = x[idx[i] >= 0 ? idx[i] : 0];
  if (TAIL) {
    for (int i = tid; i < (int)((V + 8 + 31) / 32); i += NT) marks[i] = 0u;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (idx[i] >= 0) {
        const uint32_t bit = top_mark_bit(idx[i], g);
        atomicOr(&marks[bit >> 5], 1u << (bit & 31));
      }
    __syncthreads();
  }
  const TopTeacher t = scalar_load(a.teacher + row);
  const float gs = a.gscale / (float)scalar_load(a.live);
  // The row's loss, after its gradient (no wavefront waits for it): lq(x) = ln of the student's
  // probability of a logit x, lq_rest that of all tokens without an entry.
  auto loss = [&](auto lq, auto lq_rest, float rest, float p_ln_p_off) {
    double term = 0.0;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (idx[i] >= 0 && !(p[i] == 0.f)) {
        const Float2x l = lq(ex(i));
        term -= (double)p[i] * ((double)l.hi + (double)l.lo);
      }
    term = block_sum_f64<NW>(term, sh.d);
    if (tid == 0) {
      term += t.p_ln_p - (double)p_ln_p_off;
      if (TAIL && rest > 0.f) {
        const Float2x l = lq_rest();
        term -= (double)rest * ((double)l.hi + (double)l.lo);
      }
      a.row_loss[row] = term;
    }
  };
  auto leave = [&](float off, float go, float rz, float off_all, int by_max) {  // LONG
    if (tid == 0) a.row_grad[row] = TopRowGrad{off, go, rz, off_all, by_max, 0};
  };
  auto patch = [&](auto q_of) {  // the kept entries' gradients replace what the walk over the row wrote
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (idx[i] >= 0) grow[idx[i]] = from_f32<T>(gs * fmaf(q_of(ex(i)), t.whole, -p[i]));
  };

  RowSum s;
  if (TAIL) {
    float c = regs_anchor<true>(r, g, kk), out = 0.f, in = 0.f;
    const uint8_t* mark8 = reinterpret_cast<const uint8_t*>(marks);
    auto marked = [&](uint32_t bit) { return ((marks[bit >> 5] >> (bit & 31)) & 1u) != 0; };
    if (tid < g.head && !marked(top_mark_bit(tid, g))) out += fast_exp2(fmaf(r.h(), kk, c));
    if (g.tail0 + tid < V && !marked(top_mark_bit((int)g.tail0 + tid, g))) out += fast_exp2(fmaf(r.t(), kk, c));
    auto add = [&](const Vec16<T>& v, uint32_t at) {
      const uint32_t bit0 = 8u + at * VEC;
      const uint32_t m = mark8[bit0 >> 3] >> (bit0 & 7u);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float e = fast_exp2(fmaf(to_f32(v.v[i]), kk, c));
        out += (m >> i) & 1u ? 0.f : e;
      }
    };
    if (LONG) {
      float before = 0.f;
      long_each(
          r, x, g, [&](const Vec16<T>& v, int64_t at) { add(v, (uint32_t)at); },
          [&](int left) { long_carry(before, out, (int)regs_raise(r, left, kk, c)); });
      out += before;
    } else {
#pragma unroll
      for (int j = 0; j < KREG; ++j) {
        if (tid + j * NT < (int)g.nvec) {
          forget(r.v[j]);
          add(r.v[j], (uint32_t)(tid + j * NT));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (idx[i] >= 0) in += fast_exp2(fmaf(ex(i), kk, c));
    // (a wavefront of nothing but -inf has no exponent of its own to take entries by)
    if (!(c < kVrNoTerm) && in > 0.f) in = __builtin_inff();
    s = rowsum_block<NW, true>(c, out, in, sh.sums);
    s.ok = s.ok && (t.rest == 0.f || s.z > 1e-30f);
    // (as scalars: no register of every thread for the length of the row)
    s = RowSum{same_in_wave(s.c), same_in_wave(s.z), same_in_wave(s.a), s.ok};
  } else {
    s = LONG ? long_sum(r, x, g, kk, sh.sums) : regs_sum(r, g, kk, sh.sums);
  }
  if (s.ok) {
    const float rest_z = s.z;
    if (TAIL) s.z += s.a;
    if (grow) {
      // the other tokens' q (P - r / q_r), q_r what the student leaves to them
      const float rz = 1.f / s.z, c = s.c;
      const float go = gs * (TAIL && t.rest > 0.f ? fmaf(-t.rest, s.z / rest_z, t.whole) : t.whole) * rz;
      auto other = [=](float xv) { return go * fast_exp2(fmaf(xv, kk, c)); };
      auto none = [](float) { return 0.f; };
      if (LONG) {
        leave(c, go, rz, c, 0);
      } else {
        regs_map(r, g, x, grow, V, -1, other, none);
        patch([&](float xv) { return fast_exp2(fmaf(xv, kk, c)) * rz; });
      }
    }
    loss([&](float xv) { return rowsum_log_prob(a.r, s, xv); }, [&]() { return ln_share(log2_2x(rest_z), s.z); }, t.rest,
         0.f);
    return;
  }
  __syncthreads();
  // Rows whose sums need the true maximum: walked.
  VocabStat out = vstat_init(), all;
  if (TAIL) {
    VocabStatSum others;
    for (int64_t i = tid; i < V; i += NT) {
      const uint32_t bit = top_mark_bit((int)i, g);
      if ((marks[bit >> 5] >> (bit & 31)) & 1u) continue;
      float x1[1] = {to_f32(x[i])};
      others.add(x1, kk);
    }
    out = vstat_block<NW>(others.whole(kk), kk, sh.stats);
    VocabStat in = vstat_init();
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (idx[i] >= 0) {
        float x1[1] = {ex(i)};
        vstat_fold<1>(in, x1, kk);
      }
    all = vstat_merge(out, vstat_block<NW>(in, kk, sh.stats), kk);
  } else {
    all = vstat_block<NW>(vocab_stat_walk<T, NT>(x, V, kk), kk, sh.stats);
  }
  // the rest's share: its sum, moved to the row's maximum, which may underflow where its logarithm does not
  Float2x lq_rest{0.f, 0.f};
  float rest = t.rest, r_ln_r = 0.f;
  if (TAIL) {
    const Float2x d = two_sum(out.m, -all.m), e = two_mul(d.hi, kk), l = log2_2x(out.z), h = two_sum(e.hi, l.hi);
    if (out.z > 0.f || out.z != out.z)
      lq_rest = ln_share(Float2x{h.hi, h.lo + (l.lo + (e.lo + d.lo * kk))}, all.z);
    else
      lq_rest.hi = -__builtin_inff();
    // What the teacher leaves to the others is one minus a sum that its log-sum-exp's error moves by as much.
    // Where it is no more than that, and the student leaves them next to nothing, all there is lies in the
    // entries (a vocabulary masked to fewer tokens than entries): no r, rather than an r ln(r / q_r) of noise,
    // infinite where both models cannot reach the others.
    if (rest > 0.f && rest <= kTopLseError + kTopLseRounding * __builtin_fabsf(scalar_load(a.t_lse + row)) &&
        lq_rest.hi < kTopOutOfReach) {
      r_ln_r = rest * (0.69314718f * __builtin_amdgcn_logf(rest));
      rest = 0.f;
    }
  }
  if (grow) {
    // The other tokens' q P - r q / q_r by their own maximum: q_r, and with it all of their q, may underflow
    // where q / q_r does not (where their sum is 0 none of them can be reached, and r / q_r is left out).
    const float rz = same_in_wave(1.f / all.z), m = same_in_wave(all.m), off = same_in_wave(TAIL ? out.m : all.m);
    float go = t.whole * rz;
    if (TAIL) go = go * fast_exp2((off - m) * kk) - (rest > 0.f && out.z != 0.f ? rest / out.z : 0.f);
    go = same_in_wave(gs * go);
    if (LONG) {
      leave(off, go, rz, m, 1);
    } else {
      vocab_map_walk<T, NT>(x, grow, V, [=](float xv, int) { return go * fast_exp2((xv - off) * kk); });
      patch([&](float xv) { return fast_exp2((xv - m) * kk) * rz; });
    }
  }
  loss([&](float xv) { return vstat_log_prob(a.r, all, xv); }, [&]() { return lq_rest; }, rest, r_ln_r);
}

// The gradient of rows too long for registers, a workgroup per part of a row (one
// workgroup that reads its row a second time: 1900 x 140000 bf16 341 us a call
// instead of 303, fp32 606 instead of 566).
constexpr int kMapBlock = 256, kMapVecs = 8, kMapPart = kMapBlock * kMapVecs;

template <typename T>
__global__ __launch_bounds__(kMapBlock) void top_map_kernel(const TopDistilArgs a, int64_t row0, int parts) {
  constexpr int VEC = Vec16<T>::N;
  const int64_t local = blockIdx.x / (unsigned)parts, row = row0 + local;
  const int part = (int)(blockIdx.x - (unsigned)local * (unsigned)parts), tid = threadIdx.x;
  const int64_t V = a.r.V, v0 = (int64_t)part * kMapPart;
  T* grow = reinterpret_cast<T*>(a.grad) + row * V;
  if (a.mask && a.mask[row] == 0) {
    const VocabGeom g = vocab_geom(grow, V);
    const T zero = from_f32<T>(0.f);
    if (part == 0 && tid < g.head) grow[tid] = zero;
    if (part == parts - 1 && g.tail0 + tid < V) grow[g.tail0 + tid] = zero;
    Vec16<T> z;
#pragma unroll
    for (int i = 0; i < VEC; ++i) z.v[i] = zero;
#pragma unroll
    for (int j = 0; j < kMapVecs; ++j) {
      const int64_t v = v0 + tid + j * kMapBlock;
      if (v < g.nvec) store16(grow + g.head + v * VEC, z);
    }
    return;
  }
  const T* x = vocab_row<T>(a.r, row);
  const VocabGeom g = vocab_geom(x, V);
  RowRegs<T, kMapBlock, kMapVecs> r;
  const int64_t e0 = g.head + v0 * VEC, some = g.nvec - v0;  // this part's first element and vectors
  const int left = some < kMapPart ? (int)some : kMapPart;
  const VecBuffer from = vec_buffer(x + e0, left);
#pragma unroll
  for (int j = 0; j < kMapVecs; ++j) r.v[j] = vec_load<T>(from, tid + j * kMapBlock);
  const TopRowGrad f = scalar_load(a.row_grad + row);
  const float k = a.r.k;
  auto other = [&](float xv) { return f.other(xv, k); };
  if (part == 0 && tid < g.head) grow[tid] = from_f32<T>(other(to_f32(x[tid])));
  if (part == parts - 1 && g.tail0 + tid < V) grow[g.tail0 + tid] = from_f32<T>(other(to_f32(x[g.tail0 + tid])));
  const bool gvec = (((uintptr_t)grow ^ (uintptr_t)x) & 15u) == 0;
  const VecBuffer to = vec_buffer(grow + e0, gvec ? left : 0);
#pragma unroll
  for (int j = 0; j < kMapVecs; ++j) {
    const int v = tid + j * kMapBlock;
    if (v < left) {
      forget(r.v[j]);
      Vec16<T> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(other(to_f32(r.v[j].v[i])));
      if (gvec) {
        vec_store(to, (uint32_t)v, o);
      } else {
        T* q = grow + e0 + (int64_t)v * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) q[i] = o.v[i];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The kept entries' gradients replace what top_map_kernel wrote; one thread an entry.
template <typename T>
__global__ __launch_bounds__(kMapBlock) void top_entries_kernel(const TopDistilArgs a) {
  const int64_t e = (int64_t)blockIdx.x * kMapBlock + threadIdx.x;
  if (e >= a.r.n_rows * a.k) return;
  const int64_t row = e / a.k;
  if (a.mask && a.mask[row] == 0) return;
  const float p = a.entry_p[e];
  if (p < 0.f) return;  // absent
  const int idx = a.t_indices[e];
  const int64_t q = row / a.r.seq_len;
  const T* x = reinterpret_cast<const T*>(a.r.s) + q * a.r.ld_seq + (row - q * a.r.seq_len) * a.r.ld_tok;
  const TopRowGrad f = a.row_grad[row];
  const float gs = a.gscale / (float)*a.live;
  reinterpret_cast<T*>(a.grad)[row * a.r.V + idx] =
      from_f32<T>(gs * fmaf(f.prob(to_f32(x[idx]), a.r.k), a.teacher[row].whole, -p));
}

__global__ __launch_bounds__(1024) void top_distil_sum_kernel(const double* __restrict__ v, int64_t n,
                                                              const int* __restrict__ live, double scale,
                                                              float* __restrict__ out) {
  __shared__ double lds[1024 / kWave];
  const double s = block_sum_f64<1024 / kWave>(thread_share_of_sum_f64<1024>(v, n), lds);
  if (threadIdx.x == 0) *out = *live > 0 ? (float)(scale * s / (double)*live) : __builtin_nanf("");
}

template <typename T>
int launch_top_logits(const VocabRows& a, int k, void* values, int32_t* indices, float* lse, hipStream_t st) {
  const RowShape sh = row_shape<T>(a.V);
  T* out = reinterpret_cast<T*>(values);
  const dim3 grid((unsigned)a.n_rows);
  if (sh.nt == 64 && k <= kTopFew)
    hipLaunchKernelGGL((top_logits_kernel<T, 64, 4, false>), grid, dim3(64), 0, st, a, k, out, indices, lse);
  else if (sh.nt == 64)
    hipLaunchKernelGGL((top_logits_kernel<T, 256, 1, false>), grid, dim3(256), 0, st, a, k, out, indices, lse);
  else if (sh.nt == 256 && sh.kreg == 4)
    hipLaunchKernelGGL((top_logits_kernel<T, 256, 4, false>), grid, dim3(256), 0, st, a, k, out, indices, lse);
  else if (sh.nt == 256)
    hipLaunchKernelGGL((top_logits_kernel<T, 256, 8, false>), grid, dim3(256), 0, st, a, k, out, indices, lse);
  else if (sh.nt == 512)
    hipLaunchKernelGGL((top_logits_kernel<T, 512, 8, false>), grid, dim3(512), 0, st, a, k, out, indices, lse);
  else
    hipLaunchKernelGGL((top_logits_kernel<T, 512, 8, true>), grid, dim3(512), 0, st, a, k, out, indices, lse);
  return check_launch();
}

// Bytes of the marks: a bit per vocabulary entry and eight in front.
inline size_t top_marks_bytes(int64_t V) { return (size_t)((V + 8 + 31) / 32) * 4; }

template <typename T, int NT, int KREG, bool LONG, bool TAIL>
int launch_top_distil_rows(const TopDistilArgs& a, hipStream_t st) {
  const size_t marks = TAIL ? top_marks_bytes(a.r.V) : 0;
  if (marks > 32768) {
    // (the largest there is, whatever this call takes: the bound is the function's, and another thread may set
    // it between this call's setting and its launch)
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&top_distil_kernel<T, NT, KREG, LONG, TAIL>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)top_marks_bytes(kTopTailVocab));
    if (e != hipSuccess) {
      set_last_hip_error((int)e);
      return TS_ERR_LAUNCH;
    }
  }
  hipLaunchKernelGGL((top_distil_kernel<T, NT, KREG, LONG, TAIL>), dim3((unsigned)a.r.n_rows), dim3(NT), marks, st, a);
  return check_launch();
}

template <typename T, bool TAIL>
int launch_top_distil_shape(const TopDistilArgs& a, hipStream_t st) {
  const RowShape sh = row_shape<T>(a.r.V);
  if (sh.nt == 64) return launch_top_distil_rows<T, 64, 4, false, TAIL>(a, st);
  if (sh.nt == 256 && sh.kreg == 4) return launch_top_distil_rows<T, 256, 4, false, TAIL>(a, st);
  if (sh.nt == 256) return launch_top_distil_rows<T, 256, 8, false, TAIL>(a, st);
  if (sh.nt == 512) return launch_top_distil_rows<T, 512, 8, false, TAIL>(a, st);
  if (sh.kreg == 8) return launch_top_distil_rows<T, 1024, 8, false, TAIL>(a, st);
  if (sh.kreg == 16) return launch_top_distil_rows<T, 1024, 16, false, TAIL>(a, st);
  int rc = launch_top_distil_rows<T, 512, 8, true, TAIL>(a, st);
  if (rc || !a.grad) return rc;
  const int64_t vecs = a.r.V / Vec16<T>::N, parts = (vecs + kMapPart - 1) / kMapPart;
  for (int64_t row0 = 0; row0 < a.r.n_rows;) {  // (the grid counts threads in 32 bits)
    int64_t n = a.r.n_rows - row0;
    if (n * parts > (1 << 23)) n = (1 << 23) / parts;
    if (n < 1) return TS_ERR_RANGE;
    hipLaunchKernelGGL((top_map_kernel<T>), dim3((unsigned)(n * parts)), dim3(kMapBlock), 0, st, a, row0, (int)parts);
    rc = check_launch();
    if (rc) return rc;
    row0 += n;
  }
  const int64_t entries = a.r.n_rows * a.k;
  hipLaunchKernelGGL((top_entries_kernel<T>), dim3((unsigned)((entries + kMapBlock - 1) / kMapBlock)), dim3(kMapBlock), 0,
                     st, a);
  return check_launch();
}

template <typename T>
int launch_top_distil(const TopDistilArgs& a, double loss_scale, float* loss_out, hipStream_t st) {
  constexpr int64_t kRows = kTeacherBlock / kWave;
  hipLaunchKernelGGL(top_teacher_kernel, dim3((unsigned)((a.r.n_rows + kRows - 1) / kRows + 1)), dim3(kTeacherBlock), 0,
                     st, a);
  int rc = check_launch();
  if (rc) return rc;
  if (a.r.n_rows > 0) rc = a.t_lse ? launch_top_distil_shape<T, true>(a, st) : launch_top_distil_shape<T, false>(a, st);
  if (rc) return rc;
  hipLaunchKernelGGL(top_distil_sum_kernel, dim3(1), dim3(1024), 0, st, a.row_loss, a.r.n_rows, a.live, loss_scale,
                     loss_out);
  return check_launch();
}

// Workspace: live count (16 bytes), teacher and gradient numbers and loss terms per row, probabilities per entry.
inline size_t top_ws_bytes(int64_t n_rows, int64_t k) { return 16 + (size_t)n_rows * (16 + 24 + 8) + (size_t)(n_rows * k) * 4; }

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

size_t ts_top_distil_workspace_bytes(int64_t n_rows, int k) {
  return n_rows < 0 || k < 0 ? 0 : ts::top_ws_bytes(n_rows, k);
}

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
  char* ws = reinterpret_cast<char*>(workspace);
  a.live = reinterpret_cast<int*>(ws);
  a.teacher = reinterpret_cast<ts::TopTeacher*>(ws + 16);
  a.row_grad = reinterpret_cast<ts::TopRowGrad*>(ws + 16 + a.r.n_rows * 16);
  a.row_loss = reinterpret_cast<double*>(ws + 16 + a.r.n_rows * 40);
  a.entry_p = reinterpret_cast<float*>(ws + 16 + a.r.n_rows * 48);
  a.grad = grad;
  hipStream_t st = (hipStream_t)stream;
  TS_BY_DTYPE(dtype, (ts::launch_top_distil<T>(a, weight * temperature * temperature, loss_out, st)))
}

}  // extern "C"
