// Orthogonalising updates by Newton-Schulz products, for batches of equal matrices (the Muon optimizer's step).
//
//   X = G / (|G| + eps);  several times  A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// (matrices with more rows than columns: A = X^T X and X <- a X + X B). Each step pulls the singular values towards one.
//
// All products of all steps run in ONE kernel on the tcgen05 tensor cores. What the mathematics gives away is used:
//   * A and B are symmetric: tiles on and above the diagonal are computed; the others are read as those, across, or stored as their
//     transposes;
//   * b A and a X are added in the epilogues, nothing is materialised but A, B and X;
//   * neither orientation needs a transposed copy: the operands of X X^T, X^T X, B X and X B are the stored matrices, K-major or
//     MN-major;
//   * the matrices of a batch do not depend on one another: a tile waits only for the products of its own matrix, counted in global
//     memory, and the end of one product overlaps the beginning of the next.
//
// Numbers. The products take fp16 operands (11 significant bits; bf16's 8 would leave errors of one per cent after five steps)
// and add up in fp32. Singular values start in [0, 1] and stay below 1.25 (the host checks what other coefficients would do), so
// that powers of two keep all three matrices in fp16's range: X and A are stored times 2^12, B times 2^11. Up to the last two steps X is
// carried as the sum of two fp16 numbers: the products see the first, a X is exact to 22 bits. Without the second, what is
// rounded off of the large singular directions would drown the small ones, which grow 480-fold: a matrix of rank one plus noise came
// out 6 % off (2-norm), with it 0.01 %. What is rounded in front of the last two steps grows 12-fold and 3.4-fold only (0.13 % for that
// matrix); there a is added to B's diagonal and X <- B X reads nothing beside its operands. Matrices of Gaussian numbers are 0.1 %
// off, less than the rounding of the result to bf16; the worst of thousands 0.3 % for 32 x 32, 0.5 % for 8 x 8 and 1.6 % for 2 x 2: the
// quintic's slope is 3.9 where a singular value has come to 1.2, and the roundings of few elements do not average out. Nor do those
// of many equal ones, whatever the size: the identity of 382 rows is 1.2 % off (bf16 result included), a constant matrix of 256 x 768
// 0.5 %, and of the singular values of [1e-4, 1], one element per row and column, the worst (0.62) 2.7 %. That is the price of operands of 11
// bits: X with 22 bits in all steps leaves it at 2.7 %, only all products with operands of 22 bits, three times the products, would mend it.
//
// Figures (five steps; floor: the products with their symmetry at the measured bf16 rate). 12 x 2304 x 768 fp32 413 - 485 us (167) by the
// clock that the power limit leaves: about 60 in front of the products (the two passes of the norm are 48), 61 for each of the last two
// steps, 74 to 78 for one whose epilogue has two addends. The library's fp16 products of these shapes, with half of the symmetric ones,
// take 51 a step. 8 x 1280 x 5120 bf16 1140 - 1400 (670): about 90 in front, 186 to 230 a step, the library's products 195; a K block of a CTA
// pair takes 0.38 to 0.46 us. One 768 x 768 matrix 124 us (6), 9 x 321 x 1155 168 (11): fifteen products in a row, each 1 us to the first
// copy, 0.3 us per K block (what one SM gets out of L2, 80 GB/s), 0.6 to 1.6 us of epilogue and 1.9 us until the next
// product has seen it.
#include <cuda_fp16.h>

#include <atomic>

#include "gemm_tcgen05.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "tp_flags.cuh"
#include "values.cuh"

namespace tnnb {

static constexpr float NS_X = 4096.f, NS_A = 4096.f, NS_B = 2048.f;  // stored = value times this
static constexpr int NS_EPI_WARPS = 8;
static constexpr int NS_THREADS = 96 + 32 * NS_EPI_WARPS;
static constexpr int NS_MAX_STEPS = 64;
static constexpr int NS_DEVICES = 64;  // whose number of CTA pairs is remembered
static constexpr int NS_FOLDED = 2;      // last steps in which B holds a

// The parts of a step, in the order in which tiles are dealt out.
enum NsPhase : int { NS_GRAM, NS_POLY, NS_STEP };

// What an epilogue does.
enum NsKind : int {
  KIND_GRAM,       // A = product
  KIND_POLY,       // B = b A + c product
  KIND_POLY_A,     // B = a I + b A + c product
  KIND_STEP,       // X = a X + product; reads and writes both parts of X
  KIND_STEP_HI,    // the same, writes the first part only
  KIND_FOLD,       // X = product, one part
  KIND_LAST,       // the result = product
};
__host__ __device__ constexpr bool ns_symmetric(int kind) { return kind <= KIND_POLY_A; }

struct NsParams {
  int m, n, l, items, steps;
  int sym_m, sym_n, sym_tiles;     // blocks of A and B, tiles on and above the diagonal
  int x_m, x_n, x_tiles;           // of X
  int k_gram, k_rest;              // K blocks of X X^T, and of the other products
  long long ldx, item_x, lds, item_s;  // pitch and distance of the stored matrices
  __half *hi[2], *lo, *gram, *poly;
  __nv_bfloat16* out;              // packed [items, m, n]
  int out_wide;                    // its rows take 16-byte vectors
  uint32_t* done;                  // [3 * steps][items] epilogue warps that have written their part; one more word: give up
  int* status;
  float coef[3 * NS_MAX_STEPS];
};

// A tile of work.
struct NsTask {
  int step, phase, item, mb, nb;
};
// Tiles on their way through a CTA, found and looked up (their inputs are complete) by a warp of its own: the divisions and the look
// at the counter took 1.5 us between two tiles' copies.
static constexpr int NS_RING = 4;
struct NsRing {
  NsTask task[NS_RING];
  uint64_t full[NS_RING], empty[NS_RING];
};

// A product's tiles in their order. RATIO column blocks are as wide as a row block is high.
template <int RATIO>
__device__ __forceinline__ NsTask ns_task(const NsParams& p, long long work) {
  NsTask t;
  const long long sym = (long long)p.items * p.sym_tiles, per_step = 2 * sym + (long long)p.items * p.x_tiles;
  t.step = (int)(work / per_step);
  long long r = work - t.step * per_step;
  t.phase = r < sym ? NS_GRAM : r < 2 * sym ? NS_POLY : NS_STEP;
  r -= t.phase * sym;
  if (t.phase == NS_STEP) {
    t.item = (int)(r / p.x_tiles);
    const int k = (int)(r - (long long)t.item * p.x_tiles);
    t.nb = k / p.x_m;
    t.mb = k - t.nb * p.x_m;
  } else {
    t.item = (int)(r / p.sym_tiles);
    int k = (int)(r - (long long)t.item * p.sym_tiles);
    t.mb = 0;
    for (int row = p.sym_n; k >= row; row -= RATIO) {
      k -= row;
      ++t.mb;
    }
    t.nb = RATIO * t.mb + k;
  }
  return t;
}

// How a tile's operands lie in memory: the first `a` K blocks of A's operand and the first `b` of B's are MN-major. X's all are or none;
// of a symmetric matrix those left of the diagonal tile that its rows meet, where they are stored across only. (CTA pairs store both
// triangles: reading across saves an epilogue its transposed stores, 127 and 124 us for one 768 x 768, 175 and 168 for 9 x 321 x 1155, but
// MN-major operands cost a busy tensor pipe more than that, 8 x 1280 x 5120 1215 and 1270.)
struct NsTurns {
  int a, b;
};
template <int PAIR, int TM, int BN, int TALL>
__device__ __forceinline__ NsTurns ns_turns(const NsTask& t) {
  constexpr int ALL = 1 << 30;
  const int a = PAIR ? 0 : t.mb * (TM / 64), b = PAIR ? 0 : t.nb * BN / TM * (TM / 64);
  if (t.phase == NS_GRAM) return TALL ? NsTurns{ALL, ALL} : NsTurns{0, 0};
  if (t.phase == NS_POLY) return {a, b};
  return TALL ? NsTurns{0, b} : NsTurns{a, ALL};
}

// Waits until the product that `t` reads is complete (the one before it, of the same matrix). Called by one lane.
__device__ __forceinline__ bool ns_ready(const NsParams& p, const NsTask& t, uint32_t per_tile, volatile uint32_t* abort_flag) {
  const int before = 3 * t.step + t.phase - 1;
  if (before < 0) return true;
  const uint32_t* word = p.done + (long long)before * p.items + t.item;
  const uint32_t want = per_tile * (t.phase == NS_GRAM ? p.x_tiles : p.sym_tiles);
  if (ld_acquire_gpu(word) == want) return true;
  const uint32_t* give_up = p.done + 3ll * p.steps * p.items;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 0;; ++i) {
    if (ld_acquire_gpu(word) == want) return true;
    if ((i & 63u) == 63u && (*abort_flag || ld_acquire_gpu(give_up) != 0 || globaltimer_ns() - t0 > 2000000000ull)) return false;
  }
}
__device__ __forceinline__ void ns_give_up(const NsParams& p, volatile uint32_t* abort_flag, int code) {
  raise_abort(p.status, abort_flag, code);
  atomicExch(p.done + 3ll * p.steps * p.items, 1u);
}

// Eight consecutive fp16 values and their fp32 forms.
__device__ __forceinline__ void from_h8(const uint4& w, float (&v)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 to_h8(const float (&v)[8]) {
  uint4 w;
  __half2* h = reinterpret_cast<__half2*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  return w;
}

// Where an epilogue reads and writes.
struct NsIo {
  const CUtensorMap *add, *add_lo;  // tiles of 32 x 32
  __half *out, *out_lo;             // this item's matrices
  long long ld;
  int item, rows, cols;     // of the output matrix
  float alpha, beta, diag;  // alpha * product + beta * addend (+ diag on the diagonal)
};

// An epilogue warp works on 32 rows x 32 columns at a time, in one of two slots of shared memory: [32 rows][64 bytes] for the
// first and for the second part of a value, 16-byte chunks swizzled by row. The addend arrives there by TMA, two slots ahead (held in
// registers instead, it was spilled, and a tile took 11 us where one without an addend took 3.5); a lane adds its row's
// accumulators and writes the results over it; then the warp writes them out in whole sectors.
static constexpr int NS_PART = 2048, NS_SLOT = 2 * NS_PART, NS_SLOTS = 2;
struct NsWarp {
  uint8_t* slots;
  uint64_t* bars;     // one per slot
  uint32_t phases;    // bit i: parity of slot i's next load
  uint32_t pending;   // bit i: a load into slot i that nobody has waited for
};
__device__ __forceinline__ uint32_t ns_slot_at(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); }

__host__ __device__ constexpr bool ns_reads(int kind) { return kind == KIND_POLY || kind == KIND_POLY_A || kind == KIND_STEP || kind == KIND_STEP_HI; }
__host__ __device__ constexpr bool ns_reads_lo(int kind) { return kind == KIND_STEP || kind == KIND_STEP_HI; }

// Request the addend of columns col .. col + 31 into slot `s`; the warp has finished with the slot.
template <int KIND>
__device__ __forceinline__ void ns_fetch(const NsIo& io, NsWarp& w, int s, int row, int col, int lane) {
  if (lane == 0) {
    fence_proxy_async_smem();
    mbar_expect_tx(w.bars + s, ns_reads_lo(KIND) ? NS_SLOT : NS_PART);
    tma_load_3d(w.slots + s * NS_SLOT, io.add, w.bars + s, col, row, io.item);
    if (ns_reads_lo(KIND)) tma_load_3d(w.slots + s * NS_SLOT + NS_PART, io.add_lo, w.bars + s, col, row, io.item);
  }
  w.pending |= 1u << s;
}

// One part of a slot into memory: 8 rows x 64 bytes per instruction.
__device__ __forceinline__ void ns_flush(const uint8_t* part, __half* out, long long ld, int rows, int cols, int row0, int col0, int lane) {
  const int ch = lane & 3;
  if (col0 + ch * 8 >= cols) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    const uint4 v = *reinterpret_cast<const uint4*>(part + ns_slot_at(r, ch));
    if (row0 + r < rows) *reinterpret_cast<uint4*>(out + (row0 + r) * ld + col0 + ch * 8) = v;
  }
}

// 32 accumulator columns of 32 rows through a slot and out.
template <int KIND>
__device__ __forceinline__ void ns_finish(const NsParams& p, const NsIo& io, uint8_t* slot, const uint32_t (&r)[32], int row0, int col0,
                                          bool mirror, int lane) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint4* hi = reinterpret_cast<uint4*>(slot + ns_slot_at(lane, k));
    uint4* lo = reinterpret_cast<uint4*>(slot + NS_PART + ns_slot_at(lane, k));
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = io.alpha * __uint_as_float(r[8 * k + j]);
    if constexpr (ns_reads(KIND)) {
      float o[8];
      from_h8(*hi, o);
      if constexpr (ns_reads_lo(KIND)) {
        float o2[8];
        from_h8(*lo, o2);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += o2[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fmaf(io.beta, o[j], v[j]);
    }
    if constexpr (KIND == KIND_POLY_A) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (row0 + lane == col0 + 8 * k + j) v[j] += io.diag;
    }
    if constexpr (KIND == KIND_LAST) {
      uint4 w;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      *hi = w;
    } else {
      const uint4 h = to_h8(v);
      *hi = h;
      if constexpr (KIND == KIND_STEP) {
        float f[8];
        from_h8(h, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = v[j] - f[j];
        *lo = to_h8(f);
      }
    }
  }
  __syncwarp();
  if (KIND == KIND_LAST && !p.out_wide) {  // rows without aligned vectors (bf16 and fp16 have the same size)
    for (int i = 0; i < 32; ++i) {
      const uint16_t v = *reinterpret_cast<const uint16_t*>(slot + ns_slot_at(i, lane >> 3) + (lane & 7) * 2);
      if (row0 + i < io.rows && col0 + lane < io.cols) reinterpret_cast<uint16_t*>(io.out)[(row0 + i) * io.ld + col0 + lane] = v;
    }
  } else {
    ns_flush(slot, io.out, io.ld, io.rows, io.cols, row0, col0, lane);
    if (KIND == KIND_STEP) ns_flush(slot + NS_PART, io.out_lo, io.ld, io.rows, io.cols, row0, col0, lane);
  }
  if (ns_symmetric(KIND) && mirror) {  // the transposed tile: a lane takes a column, 64 bytes of an output row (pitches have room for whole vectors)
    const int c = col0 + lane;
    __half* d = io.out + c * io.ld + row0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = k * 8 + 2 * j;
        const uint32_t a = *reinterpret_cast<const uint16_t*>(slot + ns_slot_at(i, lane >> 3) + (lane & 7) * 2);
        const uint32_t b = *reinterpret_cast<const uint16_t*>(slot + ns_slot_at(i + 1, lane >> 3) + (lane & 7) * 2);
        v[j] = a | (b << 16);
      }
      if (c < io.cols && row0 + k * 8 < io.rows) *reinterpret_cast<uint4*>(d + k * 8) = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
  __syncwarp();
}

// A warp's share of a tile: WCOLS columns at tensor memory address t. wait_full() waits for the accumulator, release() hands it
// back. false: a wait ran out.
template <int KIND, int WCOLS, typename Wait, typename Release>
__device__ __forceinline__ bool ns_epilogue(const NsParams& p, const NsIo& io, NsWarp& w, uint32_t t, int row0, int col0, bool mirror,
                                            int lane, volatile uint32_t* abort_flag, Wait wait_full, Release release) {
  const int there = row0 < io.rows ? (min(WCOLS, io.cols - col0) + 31) / 32 : 0;  // groups of 32 columns that exist (not positive: none)
  if constexpr (ns_reads(KIND)) {
#pragma unroll
    for (int s = 0; s < NS_SLOTS; ++s)
      if (s < there) ns_fetch<KIND>(io, w, s, row0, col0 + s * 32, lane);
  }
  if (!wait_full()) return false;
  tc_fence_after();
#pragma unroll 1
  for (int c = 0; c < WCOLS / 32; ++c) {
    const int s = c % NS_SLOTS;
    uint32_t r[32];
    tmem_ld_32x32_wait(t + c * 32, r);  // warp-collective: never under a per-lane condition
    if (c + 1 == WCOLS / 32) {
      tc_fence_before();
      __syncwarp();
      release();
    }
    if (c >= there) continue;
    if constexpr (ns_reads(KIND)) {
      if (!__all_sync(0xffffffffu, wait_or_abort(w.bars + s, (w.phases >> s) & 1, abort_flag))) return false;
      w.phases ^= 1u << s;
      w.pending &= ~(1u << s);
    }
    ns_finish<KIND>(p, io, w.slots + s * NS_SLOT, r, row0, col0 + c * 32, mirror, lane);
    if constexpr (ns_reads(KIND))
      if (c + NS_SLOTS < there) ns_fetch<KIND>(io, w, s, row0, col0 + (c + NS_SLOTS) * 32, lane);
  }
  return true;
}

// After an abort: loads that nobody waited for land before the CTA's shared memory goes away.
__device__ __forceinline__ void ns_drain(const NsWarp& w) {
  const uint64_t t0 = globaltimer_ns();
  for (int s = 0; s < NS_SLOTS; ++s)
    while (((w.pending >> s) & 1) && !mbar_try_wait(w.bars + s, (w.phases >> s) & 1))
      if (globaltimer_ns() - t0 > 200000000ull) return;
}

// Shared memory of a CTA: operand stages from a 1024-byte boundary on, the epilogue warps' slots, barriers.
template <int PAIR, int BN>
struct NsCfg {
  static constexpr int TM = PAIR ? 256 : 128;
  static constexpr int RATIO = TM / BN;
  static constexpr int A_BYTES = 16384;                       // 128 rows, 64 deep
  static constexpr int B_BYTES = (PAIR ? BN / 2 : BN) * 128;  // this CTA's rows of B
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 64 ? 6 : 5;
  static constexpr int SMEM = STAGES * STAGE + NS_EPI_WARPS * NS_SLOTS * NS_SLOT + 512 + 1024;  // (and the ring)
};

struct NsMaps {
  CUtensorMap gram, poly, x[2];           // operands: 64 x 64 elements per copy
  CUtensorMap add_gram, add_x[2], add_lo;  // addends: 32 x 32
};

// PAIR: 256 x 256 tiles over two SMs, each with 128 rows of either operand; else 128 x 128 or 128 x 64 tiles. Persistent; warp 0 copies,
// warp 1 issues the products (two accumulators), warps 2 to 9 are the epilogue, warp 10 finds the tiles. Tile i of the whole computation belongs to worker
// i modulo their number, and a tile reads what tiles before it in this order have written: as all workers run at the same time
// (cooperative launch), the first unfinished tile can always be worked on.
template <int PAIR, int BN, int TALL>
__global__ void __launch_bounds__(NS_THREADS, 1)
ns_products_kernel(const __grid_constant__ NsMaps maps, const __grid_constant__ NsParams p) {
  using Cfg = NsCfg<PAIR, BN>;
  constexpr int TM = Cfg::TM, STAGES = Cfg::STAGES, RATIO = Cfg::RATIO;
  constexpr uint32_t PER_TILE = (1 + PAIR) * NS_EPI_WARPS;  // what a finished tile adds to its product's counter
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* epi_tiles = smem + STAGES * Cfg::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi_tiles + NS_EPI_WARPS * NS_SLOTS * NS_SLOT);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* slot_bars = tempty + 2;  // [epilogue warps][slots]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(slot_bars + NS_EPI_WARPS * NS_SLOTS);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  __shared__ NsRing ring;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  const long long total = (long long)p.steps * p.items * (2 * p.sym_tiles + p.x_tiles);
  constexpr int TMEM_COLS = 2 * BN;  // 128, 256 or 512

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], PER_TILE);
    }
    for (int i = 0; i < NS_EPI_WARPS * NS_SLOTS; ++i) mbar_init(&slot_bars[i], 1);
    for (int i = 0; i < NS_RING; ++i) {
      mbar_init(&ring.full[i], 1);
      mbar_init(&ring.empty[i], NS_EPI_WARPS + (rank == 0 ? 2 : 1));
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the partner's barriers and tensor memory exist before anything refers to them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // The worker's tile number i, once its inputs are complete; next_task(i) ... gave_back(i).
  auto next_task = [&](int i, NsTask& t) {
    bool there = wait_or_abort(&ring.full[i % NS_RING], (i / NS_RING) & 1, abort_flag);
    if (!there && !*abort_flag) there = wait_or_abort(&ring.full[i % NS_RING], (i / NS_RING) & 1, abort_flag);
    if (there) t = ring.task[i % NS_RING];
    return there;
  };
  const int mine = (int)((total - worker + workers - 1) / workers);  // tiles of this worker (no fewer than one: the host's grid)

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, last_stage = -1;
      uint32_t phase = 0, last_phase = 0;
      bool ok = true;
      for (int i = 0; ok && i < mine; ++i) {
        NsTask t;
        if (!next_task(i, t)) {
          ns_give_up(p, abort_flag, ST_TIMEOUT_PRODUCER);
          ok = false;
          break;
        }
        mbar_arrive(&ring.empty[i % NS_RING]);
        const int x = t.step & 1;
        const CUtensorMap* ma = t.phase == NS_POLY ? &maps.gram : t.phase == NS_STEP && !TALL ? &maps.poly : &maps.x[x];
        const CUtensorMap* mb = t.phase == NS_POLY ? &maps.gram : t.phase == NS_STEP && TALL ? &maps.poly : &maps.x[x];
        const NsTurns turns = ns_turns<PAIR, TM, BN, TALL>(t);
        const int row0 = t.mb * TM + rank * 128, col0 = t.nb * BN + rank * (BN / 2);  // this CTA's rows of A and of B
        const int k_blocks = t.phase == NS_GRAM ? p.k_gram : p.k_rest;
        fence_proxy_async_all();  // what other SMs have stored is visible to the copies that follow
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!wait_or_abort(&empty[stage], phase ^ 1, abort_flag)) {
            ns_give_up(p, abort_flag, ST_TIMEOUT_PRODUCER);
            ok = false;
            break;
          }
          uint8_t* a_dst = smem + stage * Cfg::STAGE;
          uint8_t* b_dst = a_dst + Cfg::A_BYTES;
          const bool a_mn = PAIR ? turns.a != 0 : kb < turns.a, b_mn = PAIR ? turns.b != 0 : kb < turns.b;
          if (rank == 0) mbar_expect_tx(&full[stage], (1 + PAIR) * Cfg::STAGE);
          if (PAIR) {
            const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
            if (!a_mn) {
              tma_load_3d_pair(a_dst, ma, bar, kb * 64, row0, t.item);
              tma_load_3d_pair(a_dst + 8192, ma, bar, kb * 64, row0 + 64, t.item);
            } else {
              tma_load_3d_pair(a_dst, ma, bar, row0, kb * 64, t.item);
              tma_load_3d_pair(a_dst + 8192, ma, bar, row0 + 64, kb * 64, t.item);
            }
            if (!b_mn) {
              tma_load_3d_pair(b_dst, mb, bar, kb * 64, col0, t.item);
              tma_load_3d_pair(b_dst + 8192, mb, bar, kb * 64, col0 + 64, t.item);
            } else {
              tma_load_3d_pair(b_dst, mb, bar, col0, kb * 64, t.item);
              tma_load_3d_pair(b_dst + 8192, mb, bar, col0 + 64, kb * 64, t.item);
            }
          } else {
            if (!a_mn) {
              tma_load_3d(a_dst, ma, &full[stage], kb * 64, row0, t.item);
              tma_load_3d(a_dst + 8192, ma, &full[stage], kb * 64, row0 + 64, t.item);
            } else {
              tma_load_3d(a_dst, ma, &full[stage], row0, kb * 64, t.item);
              tma_load_3d(a_dst + 8192, ma, &full[stage], row0 + 64, kb * 64, t.item);
            }
#pragma unroll
            for (int i = 0; i < BN / 64; ++i) {
              if (!b_mn) tma_load_3d(b_dst + i * 8192, mb, &full[stage], kb * 64, col0 + i * 64, t.item);
              else tma_load_3d(b_dst + i * 8192, mb, &full[stage], col0 + i * 64, kb * 64, t.item);
            }
          }
          last_stage = stage;
          last_phase = phase;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && last_stage >= 0 && rank == 0) drain_stages(full, STAGES, last_stage, last_phase);  // before the CTA retires
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int i = 0; ok && i < mine; ++i) {
        NsTask t;
        if (!next_task(i, t)) {
          ns_give_up(p, abort_flag, ST_TIMEOUT_MMA);
          break;
        }
        mbar_arrive(&ring.empty[i % NS_RING]);
        const NsTurns turns = ns_turns<PAIR, TM, BN, TALL>(t);
        const int k_blocks = t.phase == NS_GRAM ? p.k_gram : p.k_rest;
        if (!wait_or_abort(&tempty[acc], acc_phase ^ 1, abort_flag)) {
          ns_give_up(p, abort_flag, ST_TIMEOUT_MMA);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = 0; kb < k_blocks; ++kb) {
          // (longer than the producer's own limit: where that ran out, this thread is told by the abort flag)
          bool there = wait_or_abort(&full[stage], phase, abort_flag);
          if (!there && !*abort_flag) there = wait_or_abort(&full[stage], phase, abort_flag);
          if (!there) {
            ns_give_up(p, abort_flag, ST_TIMEOUT_MMA);
            ok = false;
            break;
          }
          tc_fence_after();
          const int a_mn = PAIR ? turns.a != 0 : kb < turns.a, b_mn = PAIR ? turns.b != 0 : kb < turns.b;
          const uint32_t idesc = make_idesc_f16(TM, BN, a_mn, b_mn);
          const uint32_t a_addr = smem_u32(smem + stage * Cfg::STAGE), b_addr = a_addr + Cfg::A_BYTES;
          const uint64_t ad0 = a_mn ? make_smem_desc(a_addr, 8192, 1024) : make_smem_desc(a_addr, 16, 1024);
          const uint64_t bd0 = b_mn ? make_smem_desc(b_addr, 8192, 1024) : make_smem_desc(b_addr, 16, 1024);
          const int a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t ad = ad0 + k * a_step, bd = bd0 + k * b_step;
            const uint32_t on = (kb > 0 || k > 0) ? 1u : 0u;
            if (PAIR) tc_mma_ss_pair(d_tmem, ad, bd, idesc, on);
            else tc_mma_ss(d_tmem, ad, bd, idesc, on);
          }
          if (PAIR) tc_commit_pair(&empty[stage], 3);
          else tc_commit(&empty[stage]);
          if (++stage == STAGES) {
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
  } else if (warp == 2 + NS_EPI_WARPS) {
    if (lane == 0) {
      for (int i = 0; i < mine; ++i) {
        const NsTask t = ns_task<RATIO>(p, worker + (long long)i * workers);
        if (!ns_ready(p, t, PER_TILE, abort_flag) || !wait_or_abort(&ring.empty[i % NS_RING], ((i / NS_RING) & 1) ^ 1, abort_flag)) {
          ns_give_up(p, abort_flag, ST_TIMEOUT_PRODUCER);
          break;
        }
        ring.task[i % NS_RING] = t;
        mbar_arrive(&ring.full[i % NS_RING]);
      }
    }
  } else {
    const int q = warp & 3;  // TMEM lane quarter this warp may read
    constexpr int WCOLS = BN / 2;
    const int wcol = ((warp - 2) >> 2) * WCOLS;
    NsWarp w = {epi_tiles + (warp - 2) * NS_SLOTS * NS_SLOT, slot_bars + (warp - 2) * NS_SLOTS, 0, 0};
    const uint32_t tempty_addr = PAIR ? mapa_shared(smem_u32(&tempty[0]), 0) : 0;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
      NsTask t;
      ok = __all_sync(0xffffffffu, next_task(i, t));
      if (!ok) break;
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&ring.empty[i % NS_RING]);
        fence_proxy_async_all();  // as in front of the operands' copies, for the addend's
      }
      const int x = t.step & 1;
      const bool folded = t.step + NS_FOLDED >= p.steps, last = t.step + 1 == p.steps;
      const float a = p.coef[3 * t.step], b = p.coef[3 * t.step + 1], c = p.coef[3 * t.step + 2];
      const int row0 = t.mb * TM + rank * 128 + q * 32, col0 = t.nb * BN + wcol;
      const bool mirror = PAIR && t.nb >= RATIO * (t.mb + 1);
      const uint32_t t_addr = tmem_base + acc * BN + (static_cast<uint32_t>(q * 32) << 16) + wcol;
      const auto wait_full = [&] {
        bool there = wait_or_abort(&tfull[acc], acc_phase, abort_flag);
        // (twice: in front of the product may lie a wait for another one)
        if (!there && !*abort_flag) there = wait_or_abort(&tfull[acc], acc_phase, abort_flag);
        return (bool)__all_sync(0xffffffffu, there);
      };
      const auto release = [&] {
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster(tempty_addr + acc * 8);
          else mbar_arrive(&tempty[acc]);
        }
      };
      NsIo io;
      io.item = t.item, io.diag = a * NS_B, io.add_lo = &maps.add_lo;
      if (t.phase == NS_STEP) {
        io.add = &maps.add_x[x], io.ld = p.ldx, io.rows = p.m, io.cols = p.n;
        io.out = p.hi[x ^ 1] + t.item * p.item_x, io.out_lo = p.lo + t.item * p.item_x;
        io.alpha = last ? 1.f / (NS_B * NS_X) : 1.f / NS_B, io.beta = a;
        if (last) io.out = reinterpret_cast<__half*>(p.out) + (long long)t.item * p.m * p.n, io.ld = p.n;
      } else {
        io.add = &maps.add_gram, io.ld = p.lds, io.rows = io.cols = p.l;
        io.out = (t.phase == NS_GRAM ? p.gram : p.poly) + t.item * p.item_s, io.out_lo = nullptr;
        io.alpha = t.phase == NS_GRAM ? NS_A / (NS_X * NS_X) : c * NS_B / (NS_A * NS_A), io.beta = b * NS_B / NS_A;
      }
#define NS_RUN(KIND) ns_epilogue<KIND, WCOLS>(p, io, w, t_addr, row0, col0, mirror, lane, abort_flag, wait_full, release)
      if (t.phase == NS_GRAM) ok = NS_RUN(KIND_GRAM);
      else if (t.phase == NS_POLY) ok = folded ? NS_RUN(KIND_POLY_A) : NS_RUN(KIND_POLY);
      else if (last) ok = NS_RUN(KIND_LAST);
      else if (folded) ok = NS_RUN(KIND_FOLD);
      else ok = t.step + NS_FOLDED + 1 == p.steps ? NS_RUN(KIND_STEP_HI) : NS_RUN(KIND_STEP);
#undef NS_RUN
      if (!ok) break;
      if (!(last && t.phase == NS_STEP)) {  // the warp's part of the tile is there for everyone
        __syncwarp();
        if (lane == 0) {
          asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p.done + (long long)(3 * t.step + t.phase) * p.items + t.item) : "memory");
        }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (!ok && lane == 0) {
      ns_give_up(p, abort_flag, ST_TIMEOUT_EPILOGUE);
      ns_drain(w);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // no CTA frees tensor memory or exits while its partner may still touch it
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------------------ normalisation
// Sums of squares: fp32 per thread, fp64 from there on, per block in a fixed order; a block whose sum leaves fp32's range adds up in
// fp64 from the start (gradients may be of any size). Every block of the second kernel adds the blocks' sums up again.
static constexpr int NS_NORM_BLOCKS = 64;  // most per matrix

template <typename T>
__global__ void __launch_bounds__(256)
ns_square_kernel(const T* g, long long item, long long ld, int m, int n, int wide, double* sums, uint32_t* done, int words) {
  grid_dep_launch();
  grid_dep_wait();
  constexpr int PER = 16 / sizeof(T), AHEAD = 4;
  __shared__ double part[8];
  __shared__ double whole;
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < words; i += 256) done[i] = 0;  // the products' counters
  const T* x = g + blockIdx.y * item;
  const int per_row = wide ? n / PER : n;
  const long long all = (long long)m * per_row;  // vectors or elements
  const long long chunk = (all + gridDim.x - 1) / gridDim.x, lo = blockIdx.x * chunk, hi = min(all, lo + chunk);
  auto block_sum = [&](double s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) s += part[w];
      whole = s;
    }
    __syncthreads();
    return whole;
  };
  auto place = [&](long long i) {
    if (ld == n) return x + i * (wide ? PER : 1);
    const long long r = i / per_row;
    return x + r * ld + (i - r * per_row) * (wide ? PER : 1);
  };
  double s;
  if (wide) {
    float acc[AHEAD] = {};
    for (long long i0 = lo + threadIdx.x; i0 < hi; i0 += 256 * AHEAD) {
      Vec<T, PER> v[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (i0 + u * 256 < hi) v[u] = *reinterpret_cast<const Vec<T, PER>*>(place(i0 + u * 256));
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (i0 + u * 256 < hi)
#pragma unroll
          for (int j = 0; j < PER; ++j) acc[u] = fmaf(to_f32(v[u].v[j]), to_f32(v[u].v[j]), acc[u]);
    }
    s = block_sum((double)acc[0] + acc[1] + acc[2] + acc[3]);
  } else {
    float acc = 0.f;
    for (long long i = lo + threadIdx.x; i < hi; i += 256) acc = fmaf(to_f32(*place(i)), to_f32(*place(i)), acc);
    s = block_sum((double)acc);
  }
  if (!(s > 1e-25 && s < 1e36)) {
    s = 0;
    for (long long i = lo + threadIdx.x; i < hi; i += 256)
      for (int j = 0; j < (wide ? PER : 1); ++j) {
        const double v = to_f32(place(i)[j]);
        s = fma(v, v, s);
      }
    s = block_sum(s);
  }
  if (threadIdx.x == 0) sums[blockIdx.y * NS_NORM_BLOCKS + blockIdx.x] = s;
}

// X, as one or two fp16 numbers per element: eight columns per thread, zeros up to the pitch.
template <typename T>
__global__ void __launch_bounds__(256)
ns_scale_kernel(const T* g, long long item, long long ld, int m, int n, int wide, const double* sums, int blocks, float eps, __half* hi,
                __half* lo, long long ldx, long long item_x) {
  grid_dep_launch();
  grid_dep_wait();
  __shared__ double whole;
  if (threadIdx.x < 32) {
    double s = 0;
    for (int b = threadIdx.x; b < blocks; b += 32) s += sums[blockIdx.y * NS_NORM_BLOCKS + b];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) whole = s;
  }
  __syncthreads();
  const double by = NS_X / (sqrt(whole) + eps);
  const float by32 = (float)by;
  const bool in_range = by > 1e-30 && by < 1e30;  // else the factor itself is no fp32 number
  const T* x = g + blockIdx.y * item;
  hi += blockIdx.y * item_x;
  if (lo) lo += blockIdx.y * item_x;
  const int per_row = (int)(ldx / 8);
  const long long all = (long long)m * per_row;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
    const long long r = i / per_row;
    const int c = (int)(i - r * per_row) * 8;
    Vec<T, 8> e;
    if (wide) {
      e = *reinterpret_cast<const Vec<T, 8>*>(x + r * ld + c);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) e.v[j] = c + j < n ? x[r * ld + c + j] : from_f32<T>(0.f);
    }
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = in_range ? to_f32(e.v[j]) * by32 : (float)(to_f32(e.v[j]) * by);
    const uint4 h = to_h8(v);
    *reinterpret_cast<uint4*>(hi + r * ldx + c) = h;
    if (lo) {
      float f[8];
      from_h8(h, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = v[j] - f[j];
      *reinterpret_cast<uint4*>(lo + r * ldx + c) = to_h8(f);
    }
  }
}

// --------------------------------------------------------------------------------------------------------------- host
// Map of `items` fp16 matrices [rows, cols]: as an operand, 64 x 64 elements per copy, or as an addend, 32 x 32.
static int ns_map(CUtensorMap* map, const __half* base, int items, int rows, int cols, long long ld, long long item, int edge) {
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)items};
  const uint64_t strides[2] = {(uint64_t)ld * 2, (uint64_t)item * 2};
  const uint32_t box[3] = {(uint32_t)edge, (uint32_t)edge, 1};
  // (16-bit elements: nothing is computed with them on the way)
  return edge == 64 ? encode_tmap_bf16(map, base, 3, dims, strides, box, nullptr) : encode_tmap_bf16_sw64(map, base, 3, dims, strides, box);
}

template <int PAIR, int BN>
static void ns_tiles(NsParams& p) {
  using Cfg = NsCfg<PAIR, BN>;
  auto blocks = [](int extent, int edge) { return (extent + edge - 1) / edge; };
  p.sym_m = blocks(p.l, Cfg::TM), p.sym_n = blocks(p.l, BN);
  p.sym_tiles = 0;
  for (int i = 0; i < p.sym_m; ++i) p.sym_tiles += p.sym_n - Cfg::RATIO * i;
  p.x_m = blocks(p.m, Cfg::TM), p.x_n = blocks(p.n, BN);
  p.x_tiles = p.x_m * p.x_n;
}

// Which kernel a batch takes: 2 CTA pairs where their tiles keep all of them busy in every product, else 1 with 128 x 128 tiles, for a few
// tiles 0 with halves of those. Us of the kernels 0, 1 and 2 (the one taken is marked): 768 x 768, 1 matrix 128*, 154, 206, 4 153*, 162, 210, 6 190, 175*,
// 215, 9 267, 200*, 239, 10 294, 210, 241*, 16 462, 303, 269*; 2304 x 768, 2 of them 217, 219*, 245, 4 334, 275*, 272, 8 569, 414*, 328, 12 867, 555, 405*; 256 x
// 512, 20 112, 124*, 139, 40 171, 150*, 166, 64 225, 173, 171*, 120 399, 286, 246*; 321 x 1155, 5 139, 155*, 173, 9 178, 169*, 190, 18 307, 237*, 235, 24 361, 285,
// 276*; 1280 x 5120, 1 493, 457*, 419, 3 1164, 765*, 536, 5 2058, 1179, 801*. Matrices that are much longer than wide would take pairs
// from half as many tiles on (up to 43 % in these), and matrices of one tile never (300 of 128 x 128: 163, 124, 271*).
static int ns_kernel_of(NsParams p) {
  const int sms = sm_count();
  ns_tiles<1, 256>(p);
  if ((long long)p.sym_tiles * p.items >= sms * 2 / 5) return 2;
  ns_tiles<0, 128>(p);
  return (long long)p.x_tiles * p.items > sms ? 1 : 0;
}

template <int PAIR, int BN, int TALL>
static cudaError_t ns_launch(const NsMaps& maps, NsParams p, cudaStream_t st) {
  using Cfg = NsCfg<PAIR, BN>;
  ns_tiles<PAIR, BN>(p);
  auto kern = ns_products_kernel<PAIR, BN, TALL>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
  if (e != cudaSuccess) return e;
  const int sms = sm_count();
  const long long most = (long long)p.items * (p.sym_tiles > p.x_tiles ? p.sym_tiles : p.x_tiles);  // of a product
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;  // all workers at the same time
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.blockDim = dim3(NS_THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1 + PAIR;
  if (PAIR) {
    // Pairs that fit at the same time: a group of SMs may have an odd one over, and GPUs of one machine differ in their groups.
    static std::atomic<int> known[NS_DEVICES];
    int device = 0;
    e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    int pairs = device < NS_DEVICES ? known[device].load(std::memory_order_relaxed) : 0;
    if (pairs == 0) {
      cfg.gridDim = dim3(2);
      cfg.attrs = attr + 1, cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&pairs, kern, &cfg);
      if (e != cudaSuccess) return e;
      pairs = pairs < sms / 2 ? pairs : sms / 2;
      if (pairs < 1) return cudaErrorCooperativeLaunchTooLarge;
      if (device < NS_DEVICES) known[device].store(pairs, std::memory_order_relaxed);
      cfg.attrs = attr, cfg.numAttrs = 2;
    }
    cfg.gridDim = dim3((unsigned)(2 * (most < pairs ? most : pairs)));
  } else {
    cfg.gridDim = dim3((unsigned)(most < sms ? most : sms));
  }
  return cudaLaunchKernelEx(&cfg, kern, maps, p);
}

}  // namespace tnnb

using namespace tnnb;

extern "C" {

// out [items, m, n] (bf16, packed) = the result of `steps` Newton-Schulz steps with coefficients[3 * steps] on g [items][m, n] (matrices
// `item` apart, rows `ld`). Workspaces: hi0, hi1, lo fp16 [items][m][ldx], gram, poly fp16 [items][l][lds] with l = min(m, n) and pitches
// of n and l rounded up to 8 elements, sums fp64 [items][64], done uint32 [3 * steps * items + 1], all on 128 bytes.
int tnnb_newton_schulz(const void* g, long long item, long long ld, int type, int items, int m, int n, const float* coefficients, int steps,
                       float eps, void* out, void* hi0, void* hi1, void* lo, void* gram, void* poly, void* sums, void* done, int* status,
                       void* stream) {
  if (items <= 0 || items > 4096 || m <= 0 || n <= 0 || (m > 1 && ld < n) || steps < 1 || steps > NS_MAX_STEPS) return -3;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool tall = m > n;
  NsParams p = {};
  p.m = m, p.n = n, p.l = tall ? n : m, p.items = items, p.steps = steps;
  p.ldx = (n + 7) / 8 * 8, p.lds = (p.l + 7) / 8 * 8;
  p.item_x = (long long)m * p.ldx, p.item_s = (long long)p.l * p.lds;
  p.k_gram = ((tall ? m : n) + 63) / 64, p.k_rest = (p.l + 63) / 64;
  p.hi[0] = (__half*)hi0, p.hi[1] = (__half*)hi1, p.lo = (__half*)lo, p.gram = (__half*)gram, p.poly = (__half*)poly;
  p.out = (__nv_bfloat16*)out, p.out_wide = n % 8 == 0 && !((uintptr_t)out & 15);
  p.done = (uint32_t*)done, p.status = status;
  for (int i = 0; i < 3 * steps; ++i) p.coef[i] = coefficients[i];

  cudaError_t e = cudaSuccess;
  const int spread = 8 * sm_count() / items;  // blocks per matrix
  const int blocks = spread < 1 ? 1 : spread > NS_NORM_BLOCKS ? NS_NORM_BLOCKS : spread;
  const bool known = with_type(type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int PER = 16 / sizeof(T);
    const int wide = n % 8 == 0 && ld % PER == 0 && item % PER == 0 && !((uintptr_t)g & 15);
    auto square = ns_square_kernel<T>;
    e = launch_dependent(square, dim3(blocks, items), dim3(256), 0, st, (const T*)g, item, ld, m, n, wide, (double*)sums, p.done,
                         3 * steps * items + 1);
    if (e != cudaSuccess) return;
    auto scale = ns_scale_kernel<T>;
    const long long want = (p.item_x / 8 + 255) / 256;
    const int grid = (int)(want < spread ? want : spread < 1 ? 1 : spread);
    e = launch_dependent(scale, dim3(grid, items), dim3(256), 0, st, (const T*)g, item, ld, m, n, wide, (const double*)sums, blocks, eps,
                         p.hi[0], steps > NS_FOLDED ? p.lo : nullptr, p.ldx, p.item_x);
  });
  if (!known) return -4;
  if (e != cudaSuccess) return -(int)e - 1000;

  NsMaps maps;
  int rc = ns_map(&maps.gram, p.gram, items, p.l, p.l, p.lds, p.item_s, 64);
  rc = rc ? rc : ns_map(&maps.poly, p.poly, items, p.l, p.l, p.lds, p.item_s, 64);
  rc = rc ? rc : ns_map(&maps.add_gram, p.gram, items, p.l, p.l, p.lds, p.item_s, 32);
  rc = rc ? rc : ns_map(&maps.add_lo, p.lo, items, m, n, p.ldx, p.item_x, 32);
  for (int i = 0; i < 2; ++i) {
    rc = rc ? rc : ns_map(&maps.x[i], p.hi[i], items, m, n, p.ldx, p.item_x, 64);
    rc = rc ? rc : ns_map(&maps.add_x[i], p.hi[i], items, m, n, p.ldx, p.item_x, 32);
  }
  if (rc) return rc;
  switch (ns_kernel_of(p)) {
    case 2: e = tall ? ns_launch<1, 256, 1>(maps, p, st) : ns_launch<1, 256, 0>(maps, p, st); break;
    case 1: e = tall ? ns_launch<0, 128, 1>(maps, p, st) : ns_launch<0, 128, 0>(maps, p, st); break;
    default: e = tall ? ns_launch<0, 64, 1>(maps, p, st) : ns_launch<0, 64, 0>(maps, p, st);
  }
  return e == cudaSuccess ? 0 : -(int)e - 1000;
}

// Which of its kernels tnnb_newton_schulz takes on the current device (ns_kernel_of).
int tnnb_newton_schulz_kernel(int items, int m, int n) {
  NsParams p = {};
  p.m = m, p.n = n, p.l = m < n ? m : n, p.items = items;
  return ns_kernel_of(p);
}

}  // extern "C"
