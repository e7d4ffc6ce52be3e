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
// from below; only threads whose own maximum reaches that bound look at their elements again (about k of 256), and what they
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

static constexpr int LP_THREADS = 256;
static constexpr int LP_TOP = 32;      // most alternatives
static constexpr int LP_GROUPS = 64;   // groups of threads whose maxima bound the k-th value
static constexpr int LP_CAND = 1024;   // candidates that fit
static constexpr int LP_CLUSTER = 8;   // most CTAs per row
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
  float* stats;  // [rows][2]: the largest logit, log2 s (null: not wanted)
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float vec_max(const Vec<float, 4>& v) { return max_nan(max_nan(v.v[0], v.v[1]), max_nan(v.v[2], v.v[3])); }
__device__ __forceinline__ float vec_max(const Vec<__nv_bfloat16, 8>& v) {
  const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(v.v);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
  return max_nan(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float vec_max(const Vec<__half, 8>& v) {
  const __half2* w = reinterpret_cast<const __half2*>(v.v);
  const __half2 m = __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
  return max_nan(__low2float(m), __high2float(m));
}

// Order of logits as unsigned integers (0: none at all), NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t key_of(float z) {
  uint32_t b = __float_as_uint(z);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (b == 0x80000000u) b = 0;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

// Logits from here on might overflow when they are multiplied by c. Numbers of that size differ by far more than any exponent, so
// that (z - m) c, which loses the digits below theirs, is as good there; elsewhere z c - m c, one fused operation, is better: the
// rounding of m c is common to all terms of a row.
__device__ __forceinline__ bool huge(float m) { return !(fabsf(m) < 1e30f); }
__device__ __forceinline__ float exponent(float z, float m, float c) {
  return huge(m) ? (z - m) * c : fmaf(z, c, -__fmul_rn(m, c));
}
// The same between two maxima, 0 for equal ones.
__device__ __forceinline__ float rescale(float m, float to, float c) {
  const float d = huge(m) || huge(to) ? (m - to) * c : __fmul_rn(m, c) - __fmul_rn(to, c);
  return fmaxf(d, LP_FLOOR);
}

// Maximum logit of a set of elements, the sum of 2^d and the sum of 2^d d for their exponents d.
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float c) {
  const float m = max_nan(a.m, b.m);
  const float da = rescale(a.m, m, c), db = rescale(b.m, m, c);
  const float fa = exp2f(da), fb = exp2f(db);
  return {m, a.s * fa + b.s * fb, fa * (a.t + a.s * da) + fb * (b.t + b.s * db)};
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

struct LogprobShared {
  uint32_t group[LP_GROUPS];
  uint32_t bound;
  int winners, found, total;
  int winner[LP_THREADS];
  int warp_count[LP_THREADS / 32];
  Sums part[LP_THREADS / 32];
  Sums all;
  unsigned long long best[LP_TOP];  // this CTA's, in order; 0 past the last
  unsigned long long cand[LP_CAND];
};

// A row's part: elements [head_lo, head_hi) and [tail_lo, tail_hi) one by one, vectors [v_lo, v_hi) between (vector v begins at
// element head + v * PER).
struct RowPart {
  int head, v_lo, v_hi, lo, hi;  // lo, hi: the part's elements
  int singles_lo, singles_n;     // elements outside of vectors: the head in the first part, the tail in the last
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
template <typename T>
__device__ int count_from(const RowReader<T>& r, uint32_t x, LogprobShared& sh) {
  constexpr int PER = 16 / sizeof(T);
  int n = 0;
  for (int v = r.p.v_lo + (int)threadIdx.x; v < r.p.v_hi; v += LP_THREADS) {
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
  for (int w = 0; w < LP_THREADS / 32; ++w) n += sh.warp_count[w];
  __syncthreads();
  return n;
}

__device__ __forceinline__ void add_candidate(LogprobShared& sh, uint32_t key, int index) {
  const int at = atomicAdd(&sh.found, 1);
  if (at < LP_CAND) sh.cand[at] = ((unsigned long long)key << 32) | (uint32_t)~index;
}

// More elements reach the bound than there is room for: find the k-th largest key by bisection, take what lies above it
// (fewer than k elements) and fill up with the first elements equal to it. Returns the number of candidates, k.
template <typename T>
__device__ int select_by_bisection(const RowReader<T>& r, int k, uint32_t bound, LogprobShared& sh) {
  constexpr int PER = 16 / sizeof(T);
  uint32_t lo = bound, hi = 0xffffffffu;  // at least k keys are >= lo; the answer lies in [lo, hi]
  if (count_from(r, lo + 1, sh) < k) hi = lo;  // one value fills the rest, the usual reason (lo is not the largest key: keys that large are few)
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    if (count_from(r, mid, sh) >= k) lo = mid;
    else hi = mid - 1;
  }
  if (threadIdx.x == 0) sh.found = 0;
  __syncthreads();
  for (int v = r.p.v_lo + (int)threadIdx.x; v < r.p.v_hi; v += LP_THREADS) {
    const Vec<T, PER> w = r.vec(v);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t key = key_of(to_f32(w.v[j]));
      if (key > lo) add_candidate(sh, key, r.p.head + v * PER + j);
    }
  }
  const int i = loose<T>(r.p, threadIdx.x);
  if (i >= 0 && key_of(r.one(i)) > lo) add_candidate(sh, key_of(r.one(i)), i);
  __syncthreads();
  int have = sh.found;
  for (int i0 = r.p.lo; i0 < r.p.hi && have < k; i0 += LP_THREADS) {
    const int e = i0 + threadIdx.x;
    const bool is = e < r.p.hi && key_of(r.one(e)) == lo;
    const unsigned who = __ballot_sync(0xffffffffu, is);
    if ((threadIdx.x & 31) == 0) sh.warp_count[threadIdx.x >> 5] = __popc(who);
    __syncthreads();
    int at = have + __popc(who & ((1u << (threadIdx.x & 31)) - 1)), all = have;
    for (int w = 0; w < LP_THREADS / 32; ++w) {
      if (w < (int)(threadIdx.x >> 5)) at += sh.warp_count[w];
      all += sh.warp_count[w];
    }
    if (is && at < k) sh.cand[at] = ((unsigned long long)lo << 32) | (uint32_t)~e;
    __syncthreads();
    have = min(all, k);
  }
  return have;
}

// The `k` largest of n candidates into best[], in order (distinct keys: a place is the number of larger ones).
__device__ __forceinline__ void rank_candidates(const unsigned long long* cand, int n, int k, unsigned long long* best) {
  for (int i = threadIdx.x; i < n; i += LP_THREADS) {
    const unsigned long long mine = cand[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += cand[j] > mine;
    if (mine != 0 && place < k) best[place] = mine;
  }
}

// `parts` CTAs (a cluster, where more than one) work on a row. Few rows are split so that more of the GPU's loads are in flight.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
token_logprob_kernel(const LogprobParams a, int parts) {
  constexpr int PER = 16 / sizeof(T), AHEAD = 4;
  __shared__ LogprobShared sh;
  grid_dep_launch();
  grid_dep_wait();
  const int rank = parts > 1 ? (int)cluster_ctarank() : 0;
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  RowReader<T> r;
  r.z = static_cast<const T*>(a.z) + row * a.ld;
  r.p = split_row(r.z, a.V, rank, parts);

  // ---- the pass
  Sums sum = {-INFINITY, 0.f, 0.f};
  float mc = 0.f;  // sum.m * c
  auto raise = [&](float to) {  // a new maximum (or NaN, which stays)
    to = max_nan(sum.m, to);
    const float d = rescale(sum.m, to, a.c), f = exp2f(d);
    sum = {to, sum.s * f, f * (sum.t + sum.s * d)};
    mc = __fmul_rn(to, a.c);
  };
  auto add = [&](float d) {
    d = fmaxf(d, LP_FLOOR);
    const float e = exp2f(d);
    sum.s += e;
    sum.t = fmaf(e, d, sum.t);
  };
  for (int v0 = r.p.v_lo + tid; v0 < r.p.v_hi; v0 += LP_THREADS * AHEAD) {
    Vec<T, PER> v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (v0 + u * LP_THREADS < r.p.v_hi) {
        v[u] = r.vec(v0 + u * LP_THREADS);
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) v[u].v[j] = from_f32<T>(-INFINITY);
      }
    }
    float g = vec_max(v[0]);
#pragma unroll
    for (int u = 1; u < AHEAD; ++u) g = max_nan(g, vec_max(v[u]));
    if (!(g <= sum.m)) raise(g);
    if (!huge(sum.m)) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int j = 0; j < PER; ++j) add(fmaf(to_f32(v[u].v[j]), a.c, -mc));
    } else {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int j = 0; j < PER; ++j) add((to_f32(v[u].v[j]) - sum.m) * a.c);
    }
  }
  const int single = loose<T>(r.p, tid);
  if (single >= 0) {
    const float z = r.one(single);
    if (!(z <= sum.m)) raise(z);
    add(exponent(z, sum.m, a.c));
  }

  // ---- the bound for the alternatives, and the block's statistics
  const int k = min(a.top, r.p.hi - r.p.lo);
  const bool nothing = tid >= r.p.v_hi - r.p.v_lo && single < 0;
  const uint32_t own_key = nothing ? 0u : key_of(sum.m);
  if (k > 0) {
    uint32_t g = own_key;
#pragma unroll
    for (int o = 1; o < LP_THREADS / LP_GROUPS; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % (LP_THREADS / LP_GROUPS) == 0) sh.group[tid / (LP_THREADS / LP_GROUPS)] = g;
    if (tid < LP_TOP) sh.best[tid] = 0;
    if (tid == 0) sh.winners = sh.found = 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums other = {__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o),
                        __shfl_xor_sync(0xffffffffu, sum.t, o)};
    // the lower lane's sums first in both lanes of a pair, so that both get the same bits
    sum = (lane & o) ? join(other, sum, a.c) : join(sum, other, a.c);
  }
  if (lane == 0) sh.part[warp] = sum;
  __syncthreads();
  if (warp == LP_THREADS / 32 - 1 && lane == 0) {
    Sums all = sh.part[0];
    for (int w = 1; w < LP_THREADS / 32; ++w) all = join(all, sh.part[w], a.c);
    sh.all = all;
  }
  if (k > 0) {
    if (tid < LP_GROUPS) {
      const uint32_t g = sh.group[tid];
      int place = 0;
      for (int j = 0; j < LP_GROUPS; ++j) place += sh.group[j] > g || (sh.group[j] == g && j < tid);
      if (place == k - 1) sh.bound = g;
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    if (own_key >= bound && !nothing) sh.winner[atomicAdd(&sh.winners, 1)] = tid;
    __syncthreads();
    const int each = (r.p.v_hi - r.p.v_lo + LP_THREADS - 1) / LP_THREADS + 1;  // a thread's vectors and its loose element
    for (int it = tid; it < sh.winners * each; it += LP_THREADS) {
      const int w = sh.winner[it / each], q = it % each;
      if (q < each - 1) {
        const int v = r.p.v_lo + w + q * LP_THREADS;
        if (v >= r.p.v_hi) continue;
        const Vec<T, PER> x = r.vec(v);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const uint32_t key = key_of(to_f32(x.v[j]));
          if (key >= bound) add_candidate(sh, key, r.p.head + v * PER + j);
        }
      } else {
        const int i = loose<T>(r.p, w);
        if (i >= 0 && key_of(r.one(i)) >= bound) add_candidate(sh, key_of(r.one(i)), i);
      }
    }
    __syncthreads();
    int n = sh.found;
    if (n > LP_CAND) n = select_by_bisection(r, k, bound, sh);
    rank_candidates(sh.cand, n, k, sh.best);
  }
  __syncthreads();

  // ---- the row's results, by the first CTA
  if (parts > 1) cluster_sync_all();
  if (rank == 0) {
    Sums all = sh.all;
    const unsigned long long* best = sh.best;
    if (parts > 1) {
      for (int q = 1; q < parts; ++q) {
        const Sums* there = &sh.all;
        const Sums other = {cluster_load(&there->m, q), cluster_load(&there->s, q), cluster_load(&there->t, q)};
        all = join(all, other, a.c);
      }
      if (a.top > 0) {
        for (int i = tid; i < parts * a.top; i += LP_THREADS) {
          const int q = i / a.top, j = i - q * a.top;
          sh.cand[i] = q == 0 ? sh.best[j] : cluster_load64(&sh.best[j], q);
        }
        __syncthreads();
        if (tid < LP_TOP) sh.best[tid] = 0;
        __syncthreads();
        rank_candidates(sh.cand, parts * a.top, a.top, sh.best);
        __syncthreads();
      }
    }
    const bool dead = all.m == -INFINITY, bad = !(all.m < INFINITY);  // NaN or +inf among the logits
    const double ls = log2((double)all.s);
    const double ln2 = 0.69314718055994530942;
    auto log_prob = [&](float z) -> float {
      if (bad) return NAN;
      if (dead || z == -INFINITY) return -INFINITY;
      const double d = huge(all.m) ? ((double)z - all.m) * a.c : (double)z * a.c - __fmul_rn(all.m, a.c);
      return (float)((d - ls) * ln2);
    };
    if (tid < a.top) {
      const unsigned long long b = best[tid];
      a.top_logp[row * a.top + tid] = log_prob(value_of((uint32_t)(b >> 32)));
      a.top_index[row * a.top + tid] = (long long)(uint32_t)~(uint32_t)b;
    }
    if (tid == 0) {
      const long long tok = a.tokens64 ? static_cast<const long long*>(a.tokens)[row] : static_cast<const int*>(a.tokens)[row];
      float lp = 0.f;
      if (tok != a.ignore) lp = TNNB_CHECK(tok, a.V) && tok >= 0 && tok < a.V ? log_prob(to_f32(r.z[tok])) : NAN;
      a.logp[row] = lp;
      a.entropy[row] = bad ? NAN : dead ? 0.f : (float)fmax((ls - (double)all.t / all.s) * ln2, 0.0);
      if (a.stats) {
        a.stats[2 * row] = bad ? NAN : all.m;
        a.stats[2 * row + 1] = dead ? 0.f : (float)ls;
      }
    }
  }
  if (parts > 1) cluster_sync_all();  // no CTA leaves while its lists are read
}

// ---------------------------------------------------------------------------------------------------------- gradient
// dz_j = p_j (A + B d_j) with d_j = log2 p_j, A = -(g + h H) / temperature, B = -h ln 2 / temperature, and g / temperature more at the
// token. One read, one write.
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
  // exponent() with the choice made once: (x - sub) c - mc
  const float sub = huge(m) ? m : 0.f, mc = huge(m) ? 0.f : __fmul_rn(m, a.c);
  auto grad = [&](float x, int j) {
    const float d = fmaxf(fmaf(x - sub, a.c, -mc) - ls, LP_FLOOR);
    float v = exp2f(d) * fmaf(B, d, A);
    if (j == tok) v += at_token;
    return dead ? 0.f : v;
  };
  if (m != m) {  // NaN statistics make the whole row NaN (fmaxf above would drop it)
    for (int j = part * 256 + threadIdx.x; j < a.V; j += a.splits * 256) dz[j] = from_f32<T>(NAN);
    return;
  }
  if (((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) != 0) {  // rows that cannot share vectors
    for (int j = part * 256 + threadIdx.x; j < a.V; j += a.splits * 256) dz[j] = from_f32<T>(grad(to_f32(z[j]), j));
    return;
  }
  const RowPart p = split_row(z, a.V, part, a.splits);
  const int single = loose<T>(p, threadIdx.x);
  if (single >= 0) dz[single] = from_f32<T>(grad(to_f32(z[single]), single));
  for (int v0 = p.v_lo + threadIdx.x; v0 < p.v_hi; v0 += 256 * AHEAD) {
    Vec<T, PER> v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (v0 + u * 256 < p.v_hi) v[u] = *reinterpret_cast<const Vec<T, PER>*>(z + p.head + (v0 + u * 256) * PER);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int vi = v0 + u * 256;
      if (vi >= p.v_hi) break;
#pragma unroll
      for (int j = 0; j < PER; ++j) v[u].v[j] = from_f32<T>(grad(to_f32(v[u].v[j]), p.head + vi * PER + j));
      *reinterpret_cast<Vec<T, PER>*>(dz + p.head + vi * PER) = v[u];
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
  // Split rows while the SMs have room for more CTAs and a part still is a few vectors per thread.
  int parts = 1;
  while (parts < LP_CLUSTER && rows * parts < 296 && V / (2 * parts) >= 4096) parts *= 2;
  const LogprobParams p = {z, ld, tokens, tokens64, rows, V, top, c, ignore, (float*)logp, (float*)entropy, (float*)top_logp,
                           (long long*)top_index, (float*)stats};
  cudaError_t e = cudaSuccess;
  const bool known = with_type(type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    auto kern = token_logprob_kernel<T>;
    e = launch_dependent_cluster(kern, parts, dim3((unsigned)(rows * parts)), dim3(LP_THREADS), 0, (cudaStream_t)stream, p, parts);
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
