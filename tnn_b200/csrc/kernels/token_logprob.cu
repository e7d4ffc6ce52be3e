// Log probabilities of given tokens, the entropy of each row's distribution and its most likely tokens, and the gradient.
//
//   x = z / temperature,  M = max x,  s = sum exp(x - M),  t = sum exp(x - M) (x - M)
//   log p_j = x_j - M - log s,  H = log s - t / s,
//   dz_j = (g (delta_j,token - p_j) - h p_j (log p_j + H)) / temperature     for gradients g of log p_token and h of H
//
// One pass over the logits: every thread keeps (M, s, t) of its elements in base 2 (x log2(e) = z c) and rescales them when a new
// maximum turns up; they are joined per warp, block and cluster in a fixed order. fp32 throughout, logarithms of the sums in fp64.
//
// The top alternatives need no second pass over the row. The k-th largest of 64 disjoint groups' maxima bounds the k-th largest logit
// from below; only threads whose own maximum reaches that bound look at their elements again (about k of them), and what they
// find, a few more than k values, is ranked by counting. Order: larger logit first, then the lower index; NaN before everything, as in
// torch's sorts. Rows with so many equal values that the candidates do not fit (all masked, all zero) find the k-th value by
// bisection over its bits instead.
//
// A row that has only -inf logits has no distribution: log probability -inf, entropy 0, gradient 0. A NaN or +inf logit makes
// the row's results NaN.
#include <cmath>

#include "launch.cuh"
#include "ptx.cuh"
#include "values.cuh"

TNNB_BOUNDS_TU(token_logprob)

namespace tnnb {

static constexpr int LP_TOP = 32;      // most alternatives
static constexpr int LP_GROUPS = 64;   // groups of threads whose maxima bound the k-th value
static constexpr int LP_CAND = 1024;   // candidates that fit
static constexpr int LP_CLUSTER = 8;   // most CTAs per row
static constexpr float LP_SLACK = 8.f;
static constexpr float LP_FLOOR = -1000.f;  // 2^-1000 = 0; finite, so that 0 * exponent is 0 and not NaN

struct LogprobParams {
  const void* z;
  long long ld;
  const void* tokens;
  int tokens64;
  long long rows;
  int V, top;
  float c;  // log2(e) / temperature
  long long ignore;
  float* logp;
  float* entropy;
  float* top_logp;
  long long* top_index;
  float* stats;  // [rows][2]: what exponents are relative to, log2 s (null: not wanted)
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 16 bytes of logits as four words: the largest value (NaN if there is one), and the elements as pairs of fp32 that -inf has left
// (0 * -inf would be NaN): at least LP_LOWEST, whose probability beside any logit that huge() lets pass is 0 as well. (fp16 cannot hold
// that bound and is raised to it afterwards.) Whole words throughout: as arrays of 16-bit elements the same took twice the instructions.
static constexpr float LP_LOWEST = -1e20f;
template <typename T> struct Logits;
template <>
struct Logits<float> {
  static constexpr uint32_t NONE = 0xff800000u;  // -inf
  static constexpr float MOST = 3e38f;           // a finite value below +inf
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b))); }
  static __device__ __forceinline__ float largest(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ bool above(uint32_t w, uint32_t limit) { return !(__uint_as_float(w) <= __uint_as_float(limit)); }
  static __device__ __forceinline__ uint32_t word(float x) { return __float_as_uint(x); }
  static __device__ __forceinline__ void pairs(const uint4& v, uint64_t (&x)[2]) {
    x[0] = pack_f2(fmaxf(__uint_as_float(v.x), LP_LOWEST), fmaxf(__uint_as_float(v.y), LP_LOWEST));
    x[1] = pack_f2(fmaxf(__uint_as_float(v.z), LP_LOWEST), fmaxf(__uint_as_float(v.w), LP_LOWEST));
  }
  static __device__ __forceinline__ void values(uint32_t w, float (&x)[1]) { x[0] = __uint_as_float(w); }
  static __device__ __forceinline__ void put(uint4& v, int pair, float a, float b) {
    reinterpret_cast<uint32_t*>(&v)[2 * pair] = __float_as_uint(a), reinterpret_cast<uint32_t*>(&v)[2 * pair + 1] = __float_as_uint(b);
  }
};
template <>
struct Logits<__nv_bfloat16> {
  static constexpr uint32_t NONE = 0xff80ff80u;
  static constexpr float MOST = 3e38f;
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float largest(uint32_t w) { return max_nan(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
  // Whether one of the two elements is not below or equal to its limit; the word that holds x twice.
  static __device__ __forceinline__ bool above(uint32_t w, uint32_t limit) {
    uint32_t p;
    asm("{ .reg .pred a, b; setp.gtu.bf16x2 a|b, %1, %2; or.pred a, a, b; selp.u32 %0, 1, 0, a; }" : "=r"(p) : "r"(w), "r"(limit));
    return p != 0;
  }
  static __device__ __forceinline__ uint32_t word(float x) {
    const __nv_bfloat162 h = __float2bfloat162_rn(x);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void pairs(const uint4& v, uint64_t (&x)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t r;
      asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w[i]), "r"(0xe0aee0aeu));  // the bf16 next below LP_LOWEST, twice
      x[i] = bf16x2_to_f2(r);
    }
  }
  static __device__ __forceinline__ void values(uint32_t w, float (&x)[2]) {
    x[0] = __uint_as_float(w << 16), x[1] = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ void put(uint4& v, int pair, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    reinterpret_cast<uint32_t*>(&v)[pair] = *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Logits<__half> {
  static constexpr uint32_t NONE = 0xfc00fc00u;
  static constexpr float MOST = 65504.f;
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ bool above(uint32_t w, uint32_t limit) {
    uint32_t p;
    asm("{ .reg .pred a, b; setp.gtu.f16x2 a|b, %1, %2; or.pred a, a, b; selp.u32 %0, 1, 0, a; }" : "=r"(p) : "r"(w), "r"(limit));
    return p != 0;
  }
  static __device__ __forceinline__ uint32_t word(float x) {
    const __half2 h = __float2half2_rn(x);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void values(uint32_t w, float (&x)[2]) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    x[0] = f.x, x[1] = f.y;
  }
  static __device__ __forceinline__ float largest(uint32_t w) {
    float x[2];
    values(w, x);
    return max_nan(x[0], x[1]);
  }
  static __device__ __forceinline__ void pairs(const uint4& v, uint64_t (&x)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[2];
      values(w[i], f);
      x[i] = pack_f2(fmaxf(f[0], LP_LOWEST), fmaxf(f[1], LP_LOWEST));
    }
  }
  static __device__ __forceinline__ void put(uint4& v, int pair, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    reinterpret_cast<uint32_t*>(&v)[pair] = *reinterpret_cast<const uint32_t*>(&h);
  }
};
// The larger elements of N vectors and a word, in the two places of a word.
template <typename T, int N>
__device__ __forceinline__ uint32_t larger_of(uint32_t m, const uint4 (&v)[N]) {
  using L = Logits<T>;
#pragma unroll
  for (int i = 0; i < N; ++i) m = L::larger(m, L::larger(L::larger(v[i].x, v[i].y), L::larger(v[i].z, v[i].w)));
  return m;
}

// Order of logits as unsigned integers (0: none at all), NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t key_of(float z) {
  uint32_t b = __float_as_uint(z);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (b == 0x80000000u) b = 0;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

// Exponents relative to a logit m are z c - (m c rounded), one fused operation per element: what is rounded off m c is common to all terms
// of a row. It must stay small, or the whole row's sum overflows or vanishes with it: up to 2^24 it is half a unit at most. From there
// on (rows filled with a finite mask value, small temperatures, infinities, NaN) exponents are (z - m) c: logits that are not within a
// factor of two of m have no probability left, and for the others the difference is exact.
__device__ __forceinline__ bool huge(float m, float c) { return !(fabsf(__fmul_rn(m, c)) < 16777216.f); }
// What exponents relative to m are too large by.
__device__ __forceinline__ float excess(float m, float c) { return huge(m, c) ? 0.f : fmaf(m, c, -__fmul_rn(m, c)); }
// The exponent of one maximum relative to another, 0 for equal ones.
__device__ __forceinline__ float rescale(float m, float to, float c) {
  const float d = huge(m, c) || huge(to, c) ? (m - to) * c - excess(m, c) + excess(to, c) : __fmul_rn(m, c) - __fmul_rn(to, c);
  return fmaxf(d, LP_FLOOR);
}

// Of a set of elements: the sum of 2^d and the sum of 2^d d for their exponents d relative to m, the largest logit or one not far
// below it (-inf: there are only such; NaN, +inf: the set holds one).
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float c) {
  const float m = max_nan(a.m, b.m);
  const float da = rescale(a.m, m, c), db = rescale(b.m, m, c);
  const float fa = exp2f(da), fb = exp2f(db);
  return {m, a.s * fa + b.s * fb, fa * (a.t + a.s * da) + fb * (b.t + b.s * db)};
}

// The sums of N neighbouring lanes; every lane gets the same bits.
template <int N>
__device__ __forceinline__ Sums join_lanes(const Sums& a, float c) {
  float m = a.m;
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float d = rescale(a.m, m, c), f = exp2f(d);
  float s = a.s * f, t = f * (a.t + a.s * d);
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  return {m, s, t};
}

__device__ __forceinline__ float cluster_load(const void* own, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(own), rank)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long cluster_load64(const void* own, int rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(own), rank)) : "memory");
  return v;
}

// The pass keeps LP_RING - 1 groups of LP_VECS vectors per thread on their way through shared memory (cp.async; every thread
// reads its own only). Through registers, with no more in flight than those hold beside the sums, rows came in at 5.2 TB/s
// even where nothing was computed from them.
static constexpr int LP_VECS = 2, LP_RING = 4;
__device__ __forceinline__ void copy16_async(void* smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(gmem) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int NT>  // threads of a CTA
struct LogprobShared {
  union {
    uint4 ring[LP_RING][LP_VECS][NT];  // until the row has been read
    unsigned long long cand[LP_CAND];
  };
  alignas(16) uint32_t group[LP_GROUPS];
  uint32_t bound;
  int winners, found;
  int winner[NT];
  int warp_count[NT / 32];
  Sums part[NT / 32];
  Sums all;
  unsigned long long best[LP_TOP];  // this CTA's, in order; 0 past the last
};

// A row's part: its elements [lo, hi) are the vectors [v_lo, v_hi) (vector v begins at element head + v * PER) and what lies outside of
// vectors (`loose`): the row's first `head` elements in the first part, those behind the last vector in the last.
struct RowPart {
  int head, v_lo, v_hi, lo, hi;
};

template <typename T>
struct RowReader {
  static constexpr int PER = 16 / sizeof(T);
  const T* z;
  RowPart p;
  __device__ __forceinline__ Vec<T, PER> vec(int v) const { return *reinterpret_cast<const Vec<T, PER>*>(z + p.head + v * PER); }
  __device__ __forceinline__ float one(int i) const { return to_f32(z[i]); }
};

template <typename T>
__device__ __forceinline__ RowPart split_row(const T* z, int V, int rank, int parts) {
  constexpr int PER = 16 / sizeof(T);
  RowPart p;
  p.head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T)));
  const int vecs = (V - p.head) / PER;
  p.v_lo = (int)((long long)vecs * rank / parts);
  p.v_hi = (int)((long long)vecs * (rank + 1) / parts);
  p.lo = rank == 0 ? 0 : p.head + p.v_lo * PER;
  p.hi = rank + 1 == parts ? V : p.head + p.v_hi * PER;
  return p;
}

// Element i of the part's loose ones (head of the first part, tail of the last): its index, or -1.
template <typename T>
__device__ __forceinline__ int loose(const RowPart& p, int i) {
  const int heads = p.head > p.lo ? p.head - p.lo : 0;
  if (i < heads) return p.lo + i;
  const int at = p.head + p.v_hi * (int)(16 / sizeof(T)) + (i - heads);
  return at < p.hi ? at : -1;
}

// Number of keys >= x in the part (block-wide; every thread gets it).
template <typename T, int NT>
__device__ int count_from(const RowReader<T>& r, uint32_t x, LogprobShared<NT>& sh) {
  constexpr int PER = 16 / sizeof(T);
  int n = 0;
  for (int v = r.p.v_lo + (int)threadIdx.x; v < r.p.v_hi; v += NT) {
    const Vec<T, PER> w = r.vec(v);
#pragma unroll
    for (int j = 0; j < PER; ++j) n += key_of(to_f32(w.v[j])) >= x;
  }
  const int i = loose<T>(r.p, threadIdx.x);
  if (i >= 0) n += key_of(r.one(i)) >= x;
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) sh.warp_count[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) n += sh.warp_count[w];
  __syncthreads();
  return n;
}

template <int NT>
__device__ __forceinline__ void add_candidate(LogprobShared<NT>& sh, uint32_t key, int index) {
  const int at = atomicAdd(&sh.found, 1);
  if (at < LP_CAND) sh.cand[at] = ((unsigned long long)key << 32) | (uint32_t)~index;
}

// The elements with keys >= `from` among those of the listed threads become candidates. Returns their number (of which LP_CAND at most
// are kept). Block-wide. None of them is below `least`, whose vectors need no closer look.
template <typename T, int NT>
__device__ int collect(const RowReader<T>& r, uint32_t from, float least, LogprobShared<NT>& sh) {
  constexpr int PER = 16 / sizeof(T);
  const int each = (r.p.v_hi - r.p.v_lo + NT - 1) / NT + 1;  // a thread's vectors and its loose element
  for (int it = threadIdx.x; it < sh.winners * each; it += NT) {
    const int w = sh.winner[it / each], q = it % each;
    if (q < each - 1) {
      const int v = r.p.v_lo + w + q * NT;
      if (v >= r.p.v_hi) continue;
      const uint4 raw[1] = {*reinterpret_cast<const uint4*>(r.z + r.p.head + v * PER)};
      if (Logits<T>::largest(larger_of<T>(Logits<T>::NONE, raw)) < least) continue;
      const Vec<T, PER> x = *reinterpret_cast<const Vec<T, PER>*>(raw);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const uint32_t key = key_of(to_f32(x.v[j]));
        if (key >= from) add_candidate(sh, key, r.p.head + v * PER + j);
      }
    } else {
      const int i = loose<T>(r.p, w);
      if (i >= 0 && key_of(r.one(i)) >= from) add_candidate(sh, key_of(r.one(i)), i);
    }
  }
  __syncthreads();
  return sh.found;
}

// Fill up to k candidates with the first elements whose key is `key`; `have` candidates are there.
template <typename T, int NT>
__device__ int fill_equal(const RowReader<T>& r, int have, int k, uint32_t key, LogprobShared<NT>& sh) {
  for (int i0 = r.p.lo; i0 < r.p.hi && have < k; i0 += NT) {
    const int e = i0 + threadIdx.x;
    const bool is = e < r.p.hi && key_of(r.one(e)) == key;
    const unsigned who = __ballot_sync(0xffffffffu, is);
    if ((threadIdx.x & 31) == 0) sh.warp_count[threadIdx.x >> 5] = __popc(who);
    __syncthreads();
    int at = have + __popc(who & ((1u << (threadIdx.x & 31)) - 1)), all = have;
    for (int w = 0; w < NT / 32; ++w) {
      if (w < (int)(threadIdx.x >> 5)) at += sh.warp_count[w];
      all += sh.warp_count[w];
    }
    if (is && at < k) sh.cand[at] = ((unsigned long long)key << 32) | (uint32_t)~e;
    __syncthreads();
    have = min(all, k);
  }
  return have;
}

// Candidates for the k largest elements: those that reach the bound. Where many may equal it (all ruled out, all alike), those
// above it and then the first that equal it; where more lie above it than there is room for (logits in an order that puts the largest
// into few threads' hands), the k-th largest key is found by bisection over its bits. Returns their number, k or more.
template <typename T, int NT>
__device__ int select_candidates(const RowReader<T>& r, int k, uint32_t own_key, LogprobShared<NT>& sh) {
  constexpr uint32_t RULED_OUT = 0x007fffffu;  // the key of -inf
  constexpr int MANY = NT > 128 ? 96 : 48;     // threads; a bound that is not shared by many is reached by about k
  uint32_t bound = sh.bound;
  if (own_key >= bound && own_key != 0) sh.winner[atomicAdd(&sh.winners, 1)] = threadIdx.x;
  __syncthreads();
  if (bound != RULED_OUT && sh.winners <= MANY) {
    const int n = collect(r, bound, value_of(bound), sh);
    if (n <= LP_CAND) return n;
  }
  auto above = [&](uint32_t key, bool mine) {  // candidates above `key`
    __syncthreads();
    if (threadIdx.x == 0) sh.winners = sh.found = 0;
    __syncthreads();
    if (mine) sh.winner[atomicAdd(&sh.winners, 1)] = threadIdx.x;
    __syncthreads();
    return key == 0xffffffffu ? 0 : collect(r, key + 1, value_of(key), sh);
  };
  int n = above(bound, own_key > bound);
  if (n > LP_CAND) {
    uint32_t hi = 0xffffffffu;  // at least k keys are >= bound; the k-th lies in [bound, hi]
    while (bound < hi) {
      const uint32_t mid = bound + (hi - bound) / 2 + 1;
      if (count_from(r, mid, sh) >= k) bound = mid;
      else hi = mid - 1;
    }
    n = above(bound, own_key > bound);  // fewer than k
  }
  return n >= k ? n : fill_equal(r, n, k, bound, sh);
}

// The `k` largest of n candidates into best[], in order (distinct keys: a place is the number of larger ones).
template <int NT>
__device__ __forceinline__ void rank_candidates(const unsigned long long* cand, int n, int k, unsigned long long* best) {
  for (int i = threadIdx.x; i < n; i += NT) {
    const unsigned long long mine = cand[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += cand[j] > mine;
    if (mine != 0 && place < k) best[place] = mine;
  }
}

// A row's results (one warp).
template <typename T>
__device__ __forceinline__ void write_row(const LogprobParams& a, const Sums& all, const unsigned long long* best, long long row, const T* z) {
  const int lane = threadIdx.x & 31;
  const bool dead = all.m == -INFINITY, bad = !(all.m < INFINITY);  // NaN or +inf among the logits
  const double ls = log2((double)all.s);
  const double ln2 = 0.69314718055994530942;
  auto log_prob = [&](float v) -> float {
    if (bad) return NAN;
    if (dead || v == -INFINITY) return -INFINITY;
    const double d = huge(all.m, a.c) ? ((double)v - all.m) * a.c : (double)v * a.c - __fmul_rn(all.m, a.c);
    return (float)((d - ls) * ln2);
  };
  if (lane < a.top) {
    const unsigned long long b = best[lane];
    a.top_logp[row * a.top + lane] = log_prob(value_of((uint32_t)(b >> 32)));
    a.top_index[row * a.top + lane] = (long long)(uint32_t)~(uint32_t)b;
  }
  if (lane == 0) {
    const long long tok = a.tokens64 ? static_cast<const long long*>(a.tokens)[row] : static_cast<const int*>(a.tokens)[row];
    float lp = 0.f;
    if (tok != a.ignore) lp = TNNB_CHECK(tok, a.V) && tok >= 0 && tok < a.V ? log_prob(to_f32(z[tok])) : NAN;
    a.logp[row] = lp;
    a.entropy[row] = bad ? NAN : dead ? 0.f : (float)fmax((ls - (double)all.t / all.s) * ln2, 0.0);
    if (a.stats) {
      a.stats[2 * row] = bad ? NAN : all.m;
      a.stats[2 * row + 1] = dead ? 0.f : (float)ls;
    }
  }
}

// `parts` CTAs (a cluster, where more than one) work on a row. Few rows are split so that more of the GPU's loads are in flight.
template <typename T, int NT, int CTAS>
__global__ void __launch_bounds__(NT, CTAS)
token_logprob_kernel(const LogprobParams a, int parts) {
  constexpr int PER = 16 / sizeof(T);
  __shared__ LogprobShared<NT> sh;
  grid_dep_launch();
  grid_dep_wait();
  const int rank = parts > 1 ? (int)cluster_ctarank() : 0;
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  RowReader<T> r;
  r.z = static_cast<const T*>(a.z) + row * a.ld;
  r.p = split_row(r.z, a.V, rank, parts);

  // ---- the pass: sums of even and odd elements side by side in pairs, two pairs of each; the next loads are on their way
  // while these are worked on. Exponents are relative to the warp's largest logit of its first round; only one that lies LP_SLACK
  // above (in base 2; twice that where the limit's own rounding adds as much) moves that, or nearly every round some lane would, and the
  // warp with it. Instructions bound this (3 of 4 issue slots are taken; the exponentials alone take half of their unit), so the only look
  // at the logits' size is one comparison of packed maxima, and whole rounds know no ends of rows: 8 instructions per element became
  // 6.5, 8192 x 50257 bf16 174 -> 166 us, 152 with 128 threads per row (5.4 TB/s), 132 without alternatives (6.2 TB/s).
  uint32_t tops = Logits<T>::NONE;  // this thread's largest logits, in even and in odd places
  float m = -INFINITY, mc = 0.f;    // what exponents are relative to, and times c
  uint32_t limit = Logits<T>::word(NAN);  // above it, m moves; NaN: look at every round, there is no m yet or a huge one
  uint64_t s2[2] = {0, 0}, t2[2] = {0, 0};
  const uint64_t c2 = both_f2(a.c);
  const float slack = LP_SLACK / a.c;
  auto raise = [&](float to) {  // (NaN stays)
    to = max_nan(m, to);
    const float d = rescale(m, to, a.c);
    const uint64_t d2 = both_f2(d), f2 = both_f2(exp2f(d));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      t2[i] = mul_f2(f2, fma_f2(s2[i], d2, t2[i]));
      s2[i] = mul_f2(s2[i], f2);
    }
    m = to;
    mc = __fmul_rn(to, a.c);
    limit = Logits<T>::word(huge(to, a.c) ? NAN : fminf(fmaxf(to, to + slack), Logits<T>::MOST));  // (rounded: m's own value at least)
  };
  auto add = [&](uint64_t d2, int i) {
    float d0, d1;
    unpack_f2(d2, d0, d1);
    const uint64_t e2 = pack_f2(exp2f(d0), exp2f(d1));
    s2[i] = add_f2(s2[i], e2);
    t2[i] = fma_f2(e2, d2, t2[i]);
  };
  auto work = [&](const uint4 (&v)[LP_VECS], bool first) {
    tops = larger_of<T>(tops, v);
    if (Logits<T>::above(tops, limit)) {
      float to = Logits<T>::largest(tops);
      if (first)  // (all lanes are here)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) to = max_nan(to, __shfl_xor_sync(0xffffffffu, to, o));
      raise(to);
      if (huge(m, a.c)) {
#pragma unroll
        for (int u = 0; u < LP_VECS; ++u) {
          const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x[PER / 4];
            Logits<T>::values(w[j], x);
#pragma unroll
            for (int i = 0; i < PER / 4; ++i) add(pack_f2(fmaxf((x[i] - m) * a.c, LP_FLOOR), LP_FLOOR), 0);
          }
        }
        return;
      }
    }
    const uint64_t nm2 = both_f2(-mc);
#pragma unroll
    for (int u = 0; u < LP_VECS; ++u) {
      uint64_t x[PER / 2];
      Logits<T>::pairs(v[u], x);
#pragma unroll
      for (int j = 0; j < PER / 2; ++j) add(fma_f2(x[j], c2, nm2), j & 1);
    }
  };
  constexpr int ROUND = NT * LP_VECS, DEPTH = LP_RING - 1;
  const int vecs = r.p.v_hi - r.p.v_lo;
  const T* from = r.z + r.p.head + (r.p.v_lo + tid) * PER;  // this thread's vectors of the next round to request
  int left = vecs - tid;                                    // > 0, > NT, ...: as many of them exist
  auto request = [&](int slot) {
#pragma unroll
    for (int u = 0; u < LP_VECS; ++u)
      if (u * NT < left) copy16_async(&sh.ring[slot][u][tid], from + u * (NT * PER));
    copy_commit();
    from += ROUND * PER;
    left -= ROUND;
  };
  auto take = [&](int slot, uint4 (&v)[LP_VECS]) {
    copy_wait<DEPTH - 1>();
#pragma unroll
    for (int u = 0; u < LP_VECS; ++u) v[u] = sh.ring[slot][u][tid];
  };
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) request(i);
  const int rounds = (vecs + ROUND - 1) / ROUND, whole = vecs / ROUND - DEPTH;
  int i = 0;
  for (; i < whole; ++i) {  // rounds whose successors' requests are whole ones
    uint4 v[LP_VECS];
    take(i % LP_RING, v);
#pragma unroll
    for (int u = 0; u < LP_VECS; ++u) copy16_async(&sh.ring[(i + DEPTH) % LP_RING][u][tid], from + u * (NT * PER));
    copy_commit();
    from += ROUND * PER;
    work(v, i == 0);
  }
  left = vecs - tid - (i + DEPTH) * ROUND;
  for (; i < rounds; ++i) {
    uint4 v[LP_VECS];
    take(i % LP_RING, v);
    if (i + 1 == rounds) {  // vectors that do not exist
#pragma unroll
      for (int u = 0; u < LP_VECS; ++u)
        if (i * ROUND + u * NT + tid >= vecs) v[u] = make_uint4(Logits<T>::NONE, Logits<T>::NONE, Logits<T>::NONE, Logits<T>::NONE);
    }
    request((i + DEPTH) % LP_RING);
    work(v, i == 0);
  }
  float top = Logits<T>::largest(tops);
  Sums sum;
  {
    float s0, s1, t0, t1;
    unpack_f2(add_f2(s2[0], s2[1]), s0, s1);
    unpack_f2(add_f2(t2[0], t2[1]), t0, t1);
    sum = {m, s0 + s1, t0 + t1};
  }
  const int single = loose<T>(r.p, tid);
  if (single >= 0) {
    const float z = r.one(single), d = excess(z, a.c), e = exp2f(d);  // as in the pass
    sum = join(sum, {z, e, e * d}, a.c);
    top = max_nan(top, z);
  }

  // ---- the bound for the alternatives, and the block's statistics
  const int k = min(a.top, r.p.hi - r.p.lo);
  const bool nothing = tid >= r.p.v_hi - r.p.v_lo && single < 0;
  const uint32_t own_key = nothing ? 0u : key_of(top);
  if (k > 0) {
    // groups of 4 threads (of 256); of 2 or 1 where there are no more vectors than that makes groups
    int share = 1;
    while (share * LP_GROUPS < NT && r.p.v_hi - r.p.v_lo > share * LP_GROUPS) share *= 2;
    uint32_t g = own_key;
    if (share > 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, 1));
    if (share > 2) g = max(g, __shfl_xor_sync(0xffffffffu, g, 2));
    if (tid % share == 0 && tid / share < LP_GROUPS) sh.group[tid / share] = g;
    if (tid < LP_TOP) sh.best[tid] = 0;
    if (tid == 0) sh.winners = sh.found = 0, sh.bound = 0xffffffffu;
  }
  sum = join_lanes<32>(sum, a.c);
  if (lane == 0) sh.part[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    sum = join_lanes<NT / 32>(sh.part[lane % (NT / 32)], a.c);
    if (parts > 1 && lane == 0) sh.all = sum;
  }
  if (k > 0) {
    if (tid < LP_GROUPS) {  // the smallest of those that fewer than k are larger than
      const uint32_t g = sh.group[tid];
      int larger = 0;
#pragma unroll
      for (int j = 0; j < LP_GROUPS; j += 4) {
        const uint4 o = *reinterpret_cast<const uint4*>(sh.group + j);
        larger += (o.x > g) + (o.y > g) + (o.z > g) + (o.w > g);
      }
      const uint32_t b = __reduce_min_sync(0xffffffffu, larger < k ? g : 0xffffffffu);
      if (lane == 0) atomicMin(&sh.bound, b);
    }
    __syncthreads();
    const int n = select_candidates(r, k, own_key, sh);
    rank_candidates<NT>(sh.cand, n, k, sh.best);
    __syncthreads();
  }

  // ---- the row's results, by the first CTA
  if (parts > 1) cluster_sync_all();
  if (rank == 0) {
    Sums all = sum;  // (warp 0's)
    const unsigned long long* best = sh.best;
    if (parts > 1) {
      for (int q = 1; warp == 0 && q < parts; ++q) {
        const Sums* there = &sh.all;
        const Sums other = {cluster_load(&there->m, q), cluster_load(&there->s, q), cluster_load(&there->t, q)};
        all = join(all, other, a.c);
      }
      if (a.top > 0) {
        for (int i = tid; i < parts * a.top; i += NT) {
          const int q = i / a.top, j = i - q * a.top;
          sh.cand[i] = q == 0 ? sh.best[j] : cluster_load64(&sh.best[j], q);
        }
        __syncthreads();
        if (tid < LP_TOP) sh.best[tid] = 0;
        __syncthreads();
        rank_candidates<NT>(sh.cand, parts * a.top, a.top, sh.best);
        __syncthreads();
      }
    }
    if (warp == 0) write_row(a, all, best, row, r.z);
    __syncwarp();
  }
  if (parts > 1) cluster_sync_all();  // no CTA leaves while its lists are read
}

// ---------------------------------------------------------------------------------------------------------- gradient
// dz_j = p_j (A + B d_j) with d_j = log2 p_j, A = -(g + h H) / temperature, B = -h ln 2 / temperature, and g / temperature more at the
// token. One read, one write, bound by memory: 4096 x 50257 bf16 140 us, 5.9 TB/s.
struct LogprobGradParams {
  const void* z;
  long long ld;
  void* dz;
  long long ldd;
  const void* tokens;
  int tokens64;
  const float* stats;
  const float* entropy;
  const float* g_logp;     // null: zeros
  const float* g_entropy;  // null: zeros
  long long rows;
  int V, splits;
  float c, inv_temp;
  long long ignore;
};

template <typename T>
__global__ void __launch_bounds__(256)
token_logprob_grad_kernel(const LogprobGradParams a) {
  constexpr int PER = 16 / sizeof(T), AHEAD = 4;
  grid_dep_launch();
  grid_dep_wait();
  const long long row = blockIdx.x / a.splits;
  const int part = (int)(blockIdx.x - row * a.splits);
  const T* z = static_cast<const T*>(a.z) + row * a.ld;
  T* dz = static_cast<T*>(a.dz) + row * a.ldd;
  const float m = a.stats[2 * row], ls = a.stats[2 * row + 1], H = a.entropy[row];
  const long long tok = a.tokens64 ? static_cast<const long long*>(a.tokens)[row] : static_cast<const int*>(a.tokens)[row];
  const bool dead = m == -INFINITY;
  float g = a.g_logp && tok != a.ignore && !dead ? a.g_logp[row] : 0.f;
  const float h = a.g_entropy && !dead ? a.g_entropy[row] : 0.f;
  if (tok != a.ignore && !(tok >= 0 && tok < a.V)) g = NAN;  // such a token's log probability is NaN
  const float A = -(g + h * H) * a.inv_temp, B = -h * 0.69314718055994530942f * a.inv_temp, at_token = g * a.inv_temp;
  if (m != m || dead) {  // NaN statistics make the whole row NaN
    const T v = from_f32<T>(dead ? 0.f : NAN);
    for (int j = part * 256 + threadIdx.x; j < a.V; j += a.splits * 256) dz[j] = v;
    return;
  }
  // log2 p = (x - m) c - (log2 s, less what the sum's exponents are too large by)
  const float off = excess(m, a.c) - ls;
  const bool big = huge(m, a.c);
  auto one = [&](float x, int j) {
    const float d = fmaxf(fmaf(x - m, a.c, off), LP_FLOOR);
    const float v = exp2f(d) * fmaf(B, d, A);
    return j == tok ? v + at_token : v;
  };
  if (big || ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) != 0) {  // rows that cannot share vectors
    for (int j = part * 256 + threadIdx.x; j < a.V; j += a.splits * 256) dz[j] = from_f32<T>(one(to_f32(z[j]), j));
    return;
  }
  const RowPart p = split_row(z, a.V, part, a.splits);
  const int single = loose<T>(p, threadIdx.x);
  if (single >= 0) dz[single] = from_f32<T>(one(to_f32(z[single]), single));
  const uint64_t nm2 = both_f2(-m), c2 = both_f2(a.c), off2 = both_f2(off), A2 = both_f2(A), B2 = both_f2(B);
  for (int v0 = p.v_lo + threadIdx.x; v0 < p.v_hi; v0 += 256 * AHEAD) {
    uint4 v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (v0 + u * 256 < p.v_hi) v[u] = *reinterpret_cast<const uint4*>(z + p.head + (v0 + u * 256) * PER);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int vi = v0 + u * 256;
      if (vi >= p.v_hi) break;
      uint64_t x[PER / 2];
      Logits<T>::pairs(v[u], x);
#pragma unroll
      for (int j = 0; j < PER / 2; ++j) {
        float d0, d1, g0, g1;
        unpack_f2(fma_f2(add_f2(x[j], nm2), c2, off2), d0, d1);
        d0 = fmaxf(d0, LP_FLOOR), d1 = fmaxf(d1, LP_FLOOR);  // (a product with B must not overflow where the probability is 0)
        unpack_f2(mul_f2(pack_f2(exp2f(d0), exp2f(d1)), fma_f2(B2, pack_f2(d0, d1), A2)), g0, g1);
        Logits<T>::put(v[u], j, g0, g1);
      }
      T* d = dz + p.head + vi * PER;
      *reinterpret_cast<uint4*>(d) = v[u];
      const long long at = tok - p.head - (long long)vi * PER;  // the token's element, by the thread that has just written it
      if (at >= 0 && at < PER) d[at] = from_f32<T>(one(to_f32(z[tok]), (int)tok));
    }
  }
}

}  // namespace tnnb

using namespace tnnb;

extern "C" {

// Row r of z: V elements from r * ld on. logp, entropy [rows]; top_logp, top_index [rows, top]; stats [rows, 2] or null, for the gradient.
int tnnb_token_logprob(const void* z, long long ld, const void* tokens, int tokens64, void* logp, void* entropy, void* top_logp,
                       void* top_index, void* stats, long long rows, int V, int top, float c, long long ignore, int type, void* stream) {
  if (rows < 0 || V <= 0 || top < 0 || top > LP_TOP || top > V || (rows > 1 && ld < V)) return -3;
  if (rows * LP_CLUSTER > 0x7fffffffLL) return -3;
  if (rows == 0) return 0;
  // A CTA gets about 18 KB per us out of memory when it is alone on its SM; a cluster costs 2 us. Us with 1, 2, 4 and 8 CTAs per row, without
  // alternatives (one call after the other: 8 x 50257 bf16 11.3, 10.6, 9.5, 10.1; 8 x 128001 fp32 19.9, 14.4, 11.2, 9.5; 20 x 20000 bf16 7.0, 8.1, 8.3, 8.5;
  // 148 x 50257 9.7, 10.8, 13.8, 20.8) and with 20 of them (graph replays, whose times come in steps of 2: 12.4 each; 22.6, 18.6, 14.5, 14.5; 10.4,
  // 10.4, 12.4, 13.3; 12.9, 14.4, 17.0, 28.8).
  int parts = 1;
  const long long bytes = (long long)V * (type == VT_FP32 ? 4 : 2);
  while (parts < LP_CLUSTER && rows * parts * 2 <= 148 && bytes / parts >= 48 << 10) parts *= 2;
  const LogprobParams p = {z, ld, tokens, tokens64, rows, V, top, c, ignore, (float*)logp, (float*)entropy, (float*)top_logp,
                           (long long*)top_index, (float*)stats};
  // What a row costs beside its elements (statistics joined, alternatives found) is per warp, so a CTA has few of them where rows fill
  // the GPU all the same. Us with 64, 128 and 256 threads, alternatives included: 20000 x 2000 bf16 71, 105, 176; 1000 x 8000 bf16 14.4,
  // 12.5, 16.5; 10000 x 8000 62, 72, 105; 8192 x 50257 bf16 207, 152, 168; 999 x 128001 fp32 183, 122, 103; 2048 of those 386, 237, 199.
  const int threads = bytes < (rows < 148 * 20 ? 8 << 10 : 16 << 10) ? 64 : bytes < (rows < 148 * 8 ? 32 << 10 : 192 << 10) ? 128 : 256;
  cudaError_t e = cudaSuccess;
  const bool known = with_type(type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    auto kern = threads == 64    ? token_logprob_kernel<T, 64, 20>
                : threads == 128 ? token_logprob_kernel<T, 128, 8>
                                 : token_logprob_kernel<T, 256, sizeof(T) == 4 ? 4 : 5>;
    e = launch_dependent_cluster(kern, parts, dim3((unsigned)(rows * parts)), dim3(threads), 0, (cudaStream_t)stream, p, parts);
  });
  if (!known) return -4;
  return e == cudaSuccess ? 0 : -(int)e - 1000;
}

int tnnb_token_logprob_grad(const void* z, long long ld, void* dz, long long ldd, const void* tokens, int tokens64, const void* stats,
                            const void* entropy, const void* g_logp, const void* g_entropy, long long rows, int V, float c, float inv_temp,
                            long long ignore, int type, void* stream) {
  if (rows < 0 || V <= 0 || (rows > 1 && (ld < V || ldd < V))) return -3;
  if (rows == 0) return 0;
  const int per_block = 256 * 4 * 2 * (type == VT_FP32 ? 4 : 8);  // two rounds of a block's loads
  const int splits = (V + per_block - 1) / per_block;
  if (rows * splits > 0x7fffffffLL) return -3;
  const LogprobGradParams p = {z, ld, dz, ldd, tokens, tokens64, (const float*)stats, (const float*)entropy, (const float*)g_logp,
                               (const float*)g_entropy, rows, V, splits, c, inv_temp, ignore};
  cudaError_t e = cudaSuccess;
  const bool known = with_type(type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    auto kern = token_logprob_grad_kernel<T>;
    e = launch_dependent(kern, dim3((unsigned)(rows * splits)), dim3(256), 0, (cudaStream_t)stream, p);
  });
  if (!known) return -4;
  return e == cudaSuccess ? 0 : -(int)e - 1000;
}

}  // extern "C"
