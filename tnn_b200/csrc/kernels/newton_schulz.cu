// Orthogonalising updates by Newton-Schulz products, for batches of equal matrices (the Muon optimizer's step).
//
//   X = G / (|G| + eps);  several times  A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// (matrices with more rows than columns: A = X^T X and X <- a X + X B). Each step pulls the singular values towards one.
//
// Three tcgen05 products per step for the whole batch. What the mathematics gives away is used:
//   * A and B are symmetric: tiles on and above the diagonal are computed, the others stored as their transposes;
//   * b A and a X are added in the epilogues, nothing is materialised but A, B and X;
//   * neither orientation needs a transposed copy: the operands of X X^T, X^T X, B X and X B are the stored matrices, K-major or
//     MN-major.
//
// Numbers. The products take fp16 operands (11 significant bits; bf16's 8 would leave errors of one per cent after five steps)
// and add up in fp32. Singular values start in [0, 1] and stay below 1.25 (the host checks what other coefficients would do), so
// that powers of two keep all three matrices in fp16's range: X and A are stored times 2^12, B times 2^11. X itself is carried from step to step as the sum of two fp16
// numbers: the products see the first, a X is exact to 22 bits. Without the second, what is rounded off of the large singular
// directions would drown the small ones, which grow 480-fold: a matrix of rank one plus noise came out 6 % off (2-norm), with it
// 0.01 %; matrices of Gaussian numbers 0.15 % either way, less than the rounding of the result to bf16.
#include <cuda_fp16.h>

#include "gemm_tcgen05.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "values.cuh"

namespace tnnb {

static constexpr float NS_X = 4096.f, NS_A = 4096.f, NS_B = 2048.f;  // stored = value times this
static constexpr int NS_EPI_WARPS = 8;
static constexpr int NS_STAGES = 6;
static constexpr int NS_STAGE = 32768;  // 128 rows of either operand, 64 deep
static constexpr int NS_TILE = 4096;    // staging tile of an epilogue warp: [32 rows][32 fp32]
static constexpr int NS_SMEM = NS_STAGES * NS_STAGE + NS_EPI_WARPS * NS_TILE + 512 + 1024;

enum NsKind : int {
  NS_GRAM,  // S = X X^T or X^T X
  NS_POLY,  // B = b A + c A A
  NS_STEP,  // X <- a X + B X or a X + X B, as two fp16 numbers
  NS_LAST,  // the same, as the result
};

struct NsParams {
  int M, N, k_blocks, m_blocks, n_blocks, tiles, items;
  float alpha, beta;  // alpha * product + beta * addend
  const __half* add;     // A (NS_POLY) or the first part of X (NS_STEP, NS_LAST); like the output in shape and pitch
  const __half* add_lo;  // second part of X
  __half* out;           // S, B or the first part of X
  __half* out_lo;        // second part of X (may be add_lo: every element is read and written by one thread)
  __nv_bfloat16* last;   // NS_LAST: packed [items, M, N]
  long long ld, item;    // pitch and distance of matrices of add, add_lo, out and out_lo
  int* status;
};

// Tile t of an item: (row block, column block), for symmetric outputs those with column >= row.
template <bool SYM>
__device__ __forceinline__ void ns_tile(const NsParams& p, int t, int& mb, int& nb) {
  if (SYM) {
    mb = 0;
    for (int row = p.m_blocks; t >= row; --row) {
      t -= row;
      ++mb;
    }
    nb = mb + t;
  } else {
    nb = t / p.m_blocks;
    mb = t - nb * p.m_blocks;
  }
}

struct Half4 {
  __half2 a, b;
};
__device__ __forceinline__ float4 to_f4(const Half4& h) {
  const float2 x = __half22float2(h.a), y = __half22float2(h.b);
  return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ Half4 to_h4(const float4& v) { return {__floats2half2_rn(v.x, v.y), __floats2half2_rn(v.z, v.w)}; }
static_assert(sizeof(Half4) == 8, "");

// PAIR: 256 x 256 tiles over two SMs, each with 128 rows of either operand; else 128 x 128 tiles. In both a stage is 32 KB.
template <int PAIR, int A_MN, int B_MN, int KIND>
__global__ void __launch_bounds__(64 + 32 * NS_EPI_WARPS, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const NsParams p) {
  constexpr bool SYM = KIND == NS_GRAM || KIND == NS_POLY;
  constexpr int TM = PAIR ? 256 : 128, BN = TM;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* epi_tiles = smem + NS_STAGES * NS_STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi_tiles + NS_EPI_WARPS * NS_TILE);
  uint64_t* empty = full + NS_STAGES;
  uint64_t* tfull = empty + NS_STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int total = p.tiles * p.items;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], (1 + PAIR) * NS_EPI_WARPS);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, 2 * BN);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 2 * BN);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the partner's barriers and tensor memory exist before anything refers to them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_dep_launch();
  grid_dep_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, last_stage = -1;
      uint32_t phase = 0, last_phase = 0;
      bool ok = true;
      for (int work = worker; ok && work < total; work += workers) {
        const int item = work / p.tiles;
        int mb, nb;
        ns_tile<SYM>(p, work - item * p.tiles, mb, nb);
        const int row0 = mb * TM + rank * 128, col0 = nb * BN + rank * 128;  // this CTA's rows of A and of B
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!wait_or_abort(&empty[stage], phase ^ 1, abort_flag)) {
            raise_abort(p.status, abort_flag, ST_TIMEOUT_PRODUCER);
            ok = false;
            break;
          }
          uint8_t* a_dst = smem + stage * NS_STAGE;
          uint8_t* b_dst = a_dst + NS_STAGE / 2;
          if (PAIR) {
            if (rank == 0) mbar_expect_tx(&full[stage], 2 * NS_STAGE);
            const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
            if (A_MN == 0) {
              tma_load_3d_pair(a_dst, &tmA, bar, kb * 64, row0, item);
            } else {
              tma_load_3d_pair(a_dst, &tmA, bar, row0, kb * 64, item);
              tma_load_3d_pair(a_dst + 8192, &tmA, bar, row0 + 64, kb * 64, item);
            }
            if (B_MN == 0) {
              tma_load_3d_pair(b_dst, &tmB, bar, kb * 64, col0, item);
            } else {
              tma_load_3d_pair(b_dst, &tmB, bar, col0, kb * 64, item);
              tma_load_3d_pair(b_dst + 8192, &tmB, bar, col0 + 64, kb * 64, item);
            }
          } else {
            mbar_expect_tx(&full[stage], NS_STAGE);
            if (A_MN == 0) {
              tma_load_3d(a_dst, &tmA, &full[stage], kb * 64, row0, item);
            } else {
              tma_load_3d(a_dst, &tmA, &full[stage], row0, kb * 64, item);
              tma_load_3d(a_dst + 8192, &tmA, &full[stage], row0 + 64, kb * 64, item);
            }
            if (B_MN == 0) {
              tma_load_3d(b_dst, &tmB, &full[stage], kb * 64, col0, item);
            } else {
              tma_load_3d(b_dst, &tmB, &full[stage], col0, kb * 64, item);
              tma_load_3d(b_dst + 8192, &tmB, &full[stage], col0 + 64, kb * 64, item);
            }
          }
          last_stage = stage;
          last_phase = phase;
          if (++stage == NS_STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && last_stage >= 0 && rank == 0) drain_stages(full, NS_STAGES, last_stage, last_phase);  // before the CTA retires
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = make_idesc_f16(TM, BN, A_MN, B_MN);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int work = worker; ok && work < total; work += workers) {
        if (!wait_or_abort(&tempty[acc], acc_phase ^ 1, abort_flag)) {
          raise_abort(p.status, abort_flag, ST_TIMEOUT_MMA);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!wait_or_abort(&full[stage], phase, abort_flag)) {
            raise_abort(p.status, abort_flag, ST_TIMEOUT_MMA);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + stage * NS_STAGE), b_addr = a_addr + NS_STAGE / 2;
          const uint64_t ad0 = A_MN ? make_smem_desc(a_addr, 8192, 1024) : make_smem_desc(a_addr, 16, 1024);
          const uint64_t bd0 = B_MN ? make_smem_desc(b_addr, 8192, 1024) : make_smem_desc(b_addr, 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t ad = ad0 + k * (A_MN ? 128 : 2), bd = bd0 + k * (B_MN ? 128 : 2);
            const uint32_t on = (kb > 0 || k > 0) ? 1u : 0u;
            if (PAIR) tc_mma_ss_pair(d_tmem, ad, bd, idesc, on);
            else tc_mma_ss(d_tmem, ad, bd, idesc, on);
          }
          if (PAIR) tc_commit_pair(&empty[stage], 3);
          else tc_commit(&empty[stage]);
          if (++stage == NS_STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if (PAIR) tc_commit_pair(&tfull[acc], 3);
        else tc_commit(&tfull[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  } else {
    const int q = warp & 3;  // TMEM lane quarter this warp may read
    constexpr int WCOLS = BN / 2;
    const int wcol = ((warp - 2) >> 2) * WCOLS;
    uint8_t* tile = epi_tiles + (warp - 2) * NS_TILE;
    const uint32_t tempty_addr = PAIR ? mapa_shared(smem_u32(&tempty[0]), 0) : 0;
    const int sub = lane >> 3, c4 = lane & 7;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int work = worker; work < total; work += workers) {
      const int item = work / p.tiles;
      int mb, nb;
      ns_tile<SYM>(p, work - item * p.tiles, mb, nb);
      const int row_base = mb * TM + rank * 128 + q * 32, col_base = nb * BN + wcol;
      ok = __all_sync(0xffffffffu, wait_or_abort(&tfull[acc], acc_phase, abort_flag));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_addr = tmem_base + acc * BN + (static_cast<uint32_t>(q * 32) << 16) + wcol;
#pragma unroll 1
      for (int c = 0; c < WCOLS; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32_wait(t_addr + c, r);  // warp-collective: never under a per-lane condition
        if (c + 32 == WCOLS) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR) mbar_arrive_cluster(tempty_addr + acc * 8);
            else mbar_arrive(&tempty[acc]);
          }
        }
        const int col0 = col_base + c;
        if (col0 >= p.N || row_base >= p.M) continue;  // (the same for the whole warp)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          *reinterpret_cast<uint4*>(tile + sw128_offset(lane, k)) = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
        __syncwarp();
        // four columns of rows sub, sub + 4, ...: whole segments of memory per instruction. Pitches are multiples of 8, so four
        // columns from a multiple of 4 below N on lie within the row's memory.
        const int col = col0 + c4 * 4;
        const long long at0 = item * p.item + (long long)(row_base + sub) * p.ld + col;
        Half4 add[8], add_lo[8];
        if (KIND != NS_GRAM && col < p.N) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (row_base + sub + i * 4 >= p.M) continue;
            add[i] = *reinterpret_cast<const Half4*>(p.add + at0 + i * 4 * p.ld);
            if (!SYM) add_lo[i] = *reinterpret_cast<const Half4*>(p.add_lo + at0 + i * 4 * p.ld);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = sub + i * 4;
          if (col >= p.N || row_base + row >= p.M) continue;
          float4* staged = reinterpret_cast<float4*>(tile + sw128_offset(row, c4));
          float4 v = *staged;
          v.x *= p.alpha, v.y *= p.alpha, v.z *= p.alpha, v.w *= p.alpha;
          if (KIND != NS_GRAM) {
            float4 o = to_f4(add[i]);
            if (!SYM) {
              const float4 lo = to_f4(add_lo[i]);
              o.x += lo.x, o.y += lo.y, o.z += lo.z, o.w += lo.w;
            }
            v.x = fmaf(p.beta, o.x, v.x), v.y = fmaf(p.beta, o.y, v.y), v.z = fmaf(p.beta, o.z, v.z), v.w = fmaf(p.beta, o.w, v.w);
          }
          if (KIND == NS_LAST) {
            __nv_bfloat16* d = p.last + ((long long)item * p.M + row_base + row) * p.N + col;
            if ((p.N & 3) == 0) {
              const __nv_bfloat162 w[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
              *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(w);
            } else {
              const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (col + j < p.N) d[j] = __float2bfloat16(e[j]);
            }
          } else {
            const Half4 h = to_h4(v);
            *reinterpret_cast<Half4*>(p.out + at0 + i * 4 * p.ld) = h;
            if (KIND == NS_STEP) {
              const float4 f = to_f4(h);
              *reinterpret_cast<Half4*>(p.out_lo + at0 + i * 4 * p.ld) = to_h4(make_float4(v.x - f.x, v.y - f.y, v.z - f.z, v.w - f.w));
            } else {
              *staged = v;
            }
          }
        }
        __syncwarp();
        if (SYM && mb != nb) {  // the transposed tile: 32 consecutive elements per instruction
          const int row = row_base + lane;
#pragma unroll 8
          for (int j = 0; j < 32; ++j) {
            const float v = *reinterpret_cast<const float*>(tile + sw128_offset(lane, j >> 2) + (j & 3) * 4);
            if (row < p.M && col0 + j < p.N) p.out[item * p.item + (long long)(col0 + j) * p.ld + row] = __float2half_rn(v);
          }
          __syncwarp();
        }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (!ok && lane == 0) raise_abort(p.status, abort_flag, ST_TIMEOUT_EPILOGUE);
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // no CTA frees tensor memory or exits while its partner may still touch it
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, 2 * BN);
    else tmem_dealloc(tmem_base, 2 * BN);
  }
}

// ------------------------------------------------------------------------------------------------------ normalisation
// Squares are added up in fp64 (fp32 gradients may be of any size), per block in a fixed order; every block of the second kernel adds
// the blocks' sums up again.
static constexpr int NS_NORM_BLOCKS = 64;  // most per matrix

template <typename T>
__global__ void __launch_bounds__(256)
ns_square_kernel(const T* g, long long item, long long ld, int m, int n, int wide, double* sums) {
  grid_dep_launch();
  grid_dep_wait();
  constexpr int PER = 16 / sizeof(T);
  __shared__ double part[8];
  const T* x = g + blockIdx.y * item;
  double s = 0;
  const int per_row = wide ? n / PER : n;
  for (int r = blockIdx.x; r < m; r += gridDim.x) {
    for (int c = threadIdx.x; c < per_row; c += 256) {
      if (wide) {
        const Vec<T, PER> v = *reinterpret_cast<const Vec<T, PER>*>(x + r * ld + (long long)c * PER);
#pragma unroll
        for (int j = 0; j < PER; ++j) s = fma((double)to_f32(v.v[j]), (double)to_f32(v.v[j]), s);
      } else {
        const double v = to_f32(x[r * ld + c]);
        s = fma(v, v, s);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) s += part[w];
    sums[blockIdx.y * NS_NORM_BLOCKS + blockIdx.x] = s;
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
ns_scale_kernel(const T* g, long long item, long long ld, int m, int n, const double* sums, int blocks, float eps, __half* hi,
                __half* lo, long long ldx, long long item_x) {
  grid_dep_launch();
  grid_dep_wait();
  double total = 0;
  for (int b = 0; b < blocks; ++b) total += sums[blockIdx.y * NS_NORM_BLOCKS + b];
  const double by = NS_X / (sqrt(total) + eps);
  const float by32 = (float)by;
  const bool in_range = by > 1e-30 && by < 1e30;  // else the factor itself is no fp32 number
  const T* x = g + blockIdx.y * item;
  hi += blockIdx.y * item_x, lo += blockIdx.y * item_x;
  for (int r = blockIdx.x; r < m; r += gridDim.x) {
    for (int c = threadIdx.x * 4; c < n; c += 1024) {
      const T* src = x + r * ld + c;
      T e[4];
      if (c + 4 <= n && (reinterpret_cast<uintptr_t>(src) & (4 * sizeof(T) - 1)) == 0) {
        *reinterpret_cast<Vec<T, 4>*>(e) = *reinterpret_cast<const Vec<T, 4>*>(src);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = c + j < n ? src[j] : from_f32<T>(0.f);
      }
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = in_range ? to_f32(e[j]) * by32 : (float)(to_f32(e[j]) * by);
      const float4 f = make_float4(v[0], v[1], v[2], v[3]);
      const Half4 h = to_h4(f);
      const float4 b = to_f4(h);
      *reinterpret_cast<Half4*>(hi + r * ldx + c) = h;  // the pitch has room for whole groups of four
      *reinterpret_cast<Half4*>(lo + r * ldx + c) = to_h4(make_float4(f.x - b.x, f.y - b.y, f.z - b.z, f.w - b.w));
    }
  }
}

// --------------------------------------------------------------------------------------------------------------- host
// Map of `items` fp16 matrices [rows, cols] as an operand: K-major, 64 columns x 128 rows per copy, or MN-major, 64 x 64.
static int ns_map(CUtensorMap* map, const __half* base, int items, int rows, int cols, long long ld, long long item, int mn) {
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)items};
  const uint64_t strides[2] = {(uint64_t)ld * 2, (uint64_t)item * 2};
  const uint32_t box[3] = {64, mn ? 64u : 128u, 1};
  return encode_tmap_bf16(map, base, 3, dims, strides, box, nullptr);  // (16-bit elements: nothing is computed with them on the way)
}

template <int A_MN, int B_MN, int KIND>
static cudaError_t ns_product(const CUtensorMap& a, const CUtensorMap& b, NsParams p, int K, cudaStream_t st) {
  constexpr bool SYM = KIND == NS_GRAM || KIND == NS_POLY;
  p.k_blocks = (K + 63) / 64;
  auto tiles_of = [&](int edge) {
    p.m_blocks = (p.M + edge - 1) / edge;
    p.n_blocks = (p.N + edge - 1) / edge;
    return SYM ? p.m_blocks * (p.m_blocks + 1) / 2 : p.m_blocks * p.n_blocks;
  };
  const int sms = sm_count();
  p.tiles = tiles_of(256);
  if ((long long)p.tiles * p.items >= sms / 2) {
    auto kern = ns_product_kernel<1, A_MN, B_MN, KIND>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM);
    if (e != cudaSuccess) return e;
    return launch_dependent_cluster(kern, 2, dim3(sms / 2 * 2), dim3(64 + 32 * NS_EPI_WARPS), NS_SMEM, st, a, b, p);
  }
  p.tiles = tiles_of(128);
  auto kern = ns_product_kernel<0, A_MN, B_MN, KIND>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM);
  if (e != cudaSuccess) return e;
  const long long work = (long long)p.tiles * p.items;
  return launch_dependent(kern, dim3((unsigned)(work < sms ? work : sms)), dim3(64 + 32 * NS_EPI_WARPS), NS_SMEM, st, a, b, p);
}

}  // namespace tnnb

using namespace tnnb;

extern "C" {

// out [items, m, n] (bf16, packed) = the result of `steps` Newton-Schulz steps with coefficients[3 * steps] on g [items][m, n] (matrices
// `item` apart, rows `ld`). Workspaces: hi0, hi1, lo fp16 [items][m][ldx], gram, poly fp16 [items][l][lds] with l = min(m, n) and pitches
// of n and l rounded up to 8 elements, all on 128 bytes; sums fp64 [items][64].
int tnnb_newton_schulz(const void* g, long long item, long long ld, int type, int items, int m, int n, const float* coefficients, int steps,
                       float eps, void* out, void* hi0, void* hi1, void* lo, void* gram, void* poly, void* sums, int* status, void* stream) {
  if (items <= 0 || items > 65535 || m <= 0 || n <= 0 || ld < n || steps < 1 || steps > 64) return -3;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool tall = m > n;
  const int l = tall ? n : m;
  const long long ldx = (n + 7) / 8 * 8, lds = (l + 7) / 8 * 8;
  const long long item_x = (long long)m * ldx, item_s = (long long)l * lds;

  cudaError_t e = cudaSuccess;
  const int blocks = m < NS_NORM_BLOCKS ? m : NS_NORM_BLOCKS;
  const bool known = with_type(type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int PER = 16 / sizeof(T);
    const int wide = n % PER == 0 && ld % PER == 0 && item % PER == 0 && !((uintptr_t)g & 15);
    auto square = ns_square_kernel<T>;
    e = launch_dependent(square, dim3(blocks, items), dim3(256), 0, st, (const T*)g, item, ld, m, n, wide, (double*)sums);
    if (e != cudaSuccess) return;
    auto scale = ns_scale_kernel<T>;
    e = launch_dependent(scale, dim3(m < 592 ? m : 592, items), dim3(256), 0, st, (const T*)g, item, ld, m, n, (const double*)sums, blocks, eps,
                         (__half*)hi0, (__half*)lo, ldx, item_x);
  });
  if (!known) return -4;
  if (e != cudaSuccess) return -(int)e - 1000;

  CUtensorMap gram_k, poly_k, x_k[2], x_mn[2];
  __half* hi[2] = {(__half*)hi0, (__half*)hi1};
  int rc = ns_map(&gram_k, (const __half*)gram, items, l, l, lds, item_s, 0);
  rc = rc ? rc : ns_map(&poly_k, (const __half*)poly, items, l, l, lds, item_s, 0);
  for (int i = 0; i < 2; ++i) {
    rc = rc ? rc : ns_map(&x_k[i], hi[i], items, m, n, ldx, item_x, 0);
    rc = rc ? rc : ns_map(&x_mn[i], hi[i], items, m, n, ldx, item_x, 1);
  }
  if (rc) return rc;

  NsParams p = {};
  p.items = items;
  p.status = status;
  for (int k = 0; k < steps; ++k) {
    const float a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
    const int x = k & 1;
    p.M = p.N = l, p.ld = lds, p.item = item_s;
    p.alpha = NS_A / (NS_X * NS_X), p.beta = 0.f;
    p.out = (__half*)gram;
    e = tall ? ns_product<1, 1, NS_GRAM>(x_mn[x], x_mn[x], p, m, st) : ns_product<0, 0, NS_GRAM>(x_k[x], x_k[x], p, n, st);
    if (e != cudaSuccess) return -(int)e - 1000;
    p.alpha = c * NS_B / (NS_A * NS_A), p.beta = b * NS_B / NS_A;
    p.add = (const __half*)gram, p.out = (__half*)poly;
    e = ns_product<0, 0, NS_POLY>(gram_k, gram_k, p, l, st);
    if (e != cudaSuccess) return -(int)e - 1000;
    const bool last = k + 1 == steps;
    p.M = m, p.N = n, p.ld = ldx, p.item = item_x;
    p.alpha = last ? 1.f / (NS_B * NS_X) : 1.f / NS_B, p.beta = last ? a / NS_X : a;
    p.add = hi[x], p.add_lo = (const __half*)lo;
    p.out = hi[x ^ 1], p.out_lo = (__half*)lo;
    p.last = (__nv_bfloat16*)out;
    if (last)
      e = tall ? ns_product<0, 0, NS_LAST>(x_k[x], poly_k, p, l, st) : ns_product<0, 1, NS_LAST>(poly_k, x_mn[x], p, l, st);
    else
      e = tall ? ns_product<0, 0, NS_STEP>(x_k[x], poly_k, p, l, st) : ns_product<0, 1, NS_STEP>(poly_k, x_mn[x], p, l, st);
    if (e != cudaSuccess) return -(int)e - 1000;
  }
  return 0;
}

}  // extern "C"
