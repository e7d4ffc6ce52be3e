// Token embedding with scaling, and its gradient by sorted tokens.
//
//   forward   y[t] = scale * W[id[t]]                       (zeros where id[t] is the padding index)
//   gradient  dW[v] = scale * sum over {t : id[t] = v} of dy[t]
//
// bf16, fp16 and fp32, any width; ids of 32 or 64 bits. Products and sums are fp32, rounded once. An id outside the table reads
// (and adds to) row 0 like the layers' embedding kernels (elementwise.cu); the bounds-checked build records it.
//
// The gradient adds up in an order that depends on the ids alone: the positions of each token as sorted, in chunks of the sorted list,
// then the chunks: the same inputs give the same bits. A row is written once, in the table's own type; sums that are added to a gradient are
// added by the memory, each element by one thread, or by one after the kernel of the others has ended.
#include "launch.cuh"
#include "ptx.cuh"
#include "values.cuh"

TNNB_BOUNDS_TU(embedding)

namespace tnnb {

// ------------------------------------------------------------------------------------------------------------ lookup
// A warp copies up to LOOKUP_VECS vectors per lane of one row: all of a row's loads are in flight together, and rows are many. Bound by
// memory: 16384 x 1024 bf16 11.7 us with a cold L2, 5.7 TB/s of rows read and written (the measured copy: 6.5).
static constexpr int LOOKUP_VECS = 4;

template <typename T, typename ID, int VEC>
__global__ void __launch_bounds__(256)
embed_lookup_kernel(const ID* __restrict__ ids, const T* __restrict__ table, long long ld,
                                                           T* __restrict__ out, long long items, int slices, int width, long long vocab,
                                                           long long padding, float scale) {
  using V = Vec<T, VEC>;
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items; item += warps) {
    const long long t = item / slices;
    const int c0 = ((int)(item - t * slices) * (32 * LOOKUP_VECS) + lane) * VEC;
    long long id = ids[t];
    const bool pad = id == padding;
    if (!pad) (void)TNNB_CHECK(id, vocab);
    if (id < 0 || id >= vocab) id = 0;
    const T* src = table + id * ld;
    T* dst = out + t * width;
    V v[LOOKUP_VECS];
#pragma unroll
    for (int i = 0; i < LOOKUP_VECS; ++i)
      if (c0 + i * 32 * VEC < width && !pad) v[i] = *reinterpret_cast<const V*>(src + c0 + i * 32 * VEC);
#pragma unroll
    for (int i = 0; i < LOOKUP_VECS; ++i) {
      if (c0 + i * 32 * VEC >= width) continue;
      V o;
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.v[j] = from_f32<T>(pad ? 0.f : to_f32(v[i].v[j]) * scale);
      *reinterpret_cast<V*>(dst + c0 + i * 32 * VEC) = o;
    }
  }
}

// -------------------------------------------------------------------------------------------------------------- sort
// Positions sorted by token, in an order that depends on the ids alone, without a pass over global counters: every CTA owns some
// table rows, reads ALL ids (they come from L2: 64 KB for 8192 tokens) and picks its own. The number of ids that belong to CTAs before
// it is the place of its part of the list, so no CTA waits for another. Within the CTA each warp walks a contiguous stretch of the ids
// and has a counter per row: counts, then starting places (rows ascending, warps ascending within a row), then the places
// themselves. On the first look it notes the positions that are its CTA's, as many as there is room for; a warp with more of them
// (a token that fills the batch) looks at its stretch again. A place gets its token with two flags, so that what adds up needs no
// other table: whether it is the token's first position and whether it is its last. Bound by latency: a few dependent loads
// from L2 and barriers, 7 us for 8192 positions, 10 for 50001.
//
// Rows are dealt out in turn (2^bits CTAs; row v is number v >> bits of CTA v mod 2^bits): frequent tokens have neighbouring numbers, and
// with ranges of rows the CTA that had them took 16 us for 8192 tokens of text, 63 for 50001. The list is in this order of rows
// ("slots"), which is as good as any. Looking twice at every position cost 17 us of 97 for 50001 positions
// of 1001 fp32 columns.
//
// Up to 65536 rows there are 128 CTAs, beyond that one per 512 rows, each of which reads all ids: the work grows with positions times
// rows. Sums added to a gradient of 16 columns (nothing is cleared then), 8192 and 65536 positions: 65536 rows 22 and 34 us, 2^18 rows 30
// and 56, 2^20 71 and 127, 2^24 0.9 and 1.5 ms. Clearing the rows that nobody names is dearer there: 2^24 rows of 32 bytes 7.7 ms.
static constexpr int SORT_WARPS = 32;
static constexpr int SORT_ROWS = 512;  // most rows of a CTA, one per thread
static constexpr int SORT_NOTES = 512;  // most positions that a warp notes: row in 9 bits, place in its stretch in 23
static constexpr uint32_t TOKEN_FIRST = 1u << 30, TOKEN_LAST = 1u << 31, TOKEN_ROW = TOKEN_FIRST - 1;

struct Slots {
  int bits, rows;  // rows per CTA, those past the table included
};
__host__ __device__ __forceinline__ Slots slots_of(long long vocab) {
  Slots s;
  s.bits = 0;
  while (s.bits < 7 && (1ll << s.bits) < vocab) ++s.bits;                          // 128 CTAs
  while (((vocab + (1ll << s.bits) - 1) >> s.bits) > SORT_ROWS) ++s.bits;
  s.rows = (int)((vocab + (1ll << s.bits) - 1) >> s.bits);
  return s;
}
__host__ __device__ __forceinline__ int sort_stretch(int n) { return (int)(((n + SORT_WARPS - 1ll) / SORT_WARPS + 127) / 128 * 128); }  // positions of a warp
__device__ __forceinline__ int slot_of(const Slots& s, int row) { return (row & ((1 << s.bits) - 1)) * s.rows + (row >> s.bits); }

// A position's CTA and the row's number there, 16 bits each (NO_CODE: padding). Every CTA looks at every position, and warps with more of
// their own than they can note do so twice: what can be done to an id once is done here, and four instructions are left (200000 positions:
// 28 us per look with the ids themselves).
static constexpr uint32_t NO_CODE = 0xffffffffu;
template <typename ID>
__global__ void __launch_bounds__(256)
embed_code_kernel(const ID* ids, int n, long long vocab, long long padding, Slots slots, uint32_t* codes) {
  grid_dep_wait();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  long long id = ids[i];
  const bool pad = id == padding;
  if (!pad) (void)TNNB_CHECK(id, vocab);
  if (id < 0 || id >= vocab) id = 0;
  codes[i] = pad ? NO_CODE : (uint32_t)(id & ((1 << slots.bits) - 1)) << 16 | (uint32_t)(id >> slots.bits);
}

__global__ void __launch_bounds__(SORT_WARPS * 32)
embed_sort_kernel(const uint32_t* codes, int n, Slots slots, int room, int* order, uint32_t* keys, int* rowptr) {
  extern __shared__ int counters[];  // [SORT_WARPS][slots.rows], [SORT_WARPS][room] notes
  __shared__ int below[SORT_WARPS], scan[SORT_WARPS];
  __shared__ int begin[SORT_ROWS], count[SORT_ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = slots.rows, own = blockIdx.x, mask = (1 << slots.bits) - 1;
  for (int i = threadIdx.x; i < SORT_WARPS * rows; i += blockDim.x) counters[i] = 0;
  grid_dep_wait();
  __syncthreads();

  const int stretch = sort_stretch(n);
  const int lo = min((long long)n, (long long)warp * stretch), hi = min((long long)n, (long long)lo + stretch);
  int* mine = counters + warp * rows;
  uint32_t* notes = reinterpret_cast<uint32_t*>(counters) + SORT_WARPS * rows + warp * room;
  const uint32_t base = (uint32_t)own << 16;
  // Calls f(four codes, place of the first) for the warp's positions, 128 at a time; the next ones are on their way meanwhile. (`codes`
  // begins on 16 bytes and ends on a whole vector.)
  auto walk = [&](auto f) {
    constexpr int SETS = 4;
    uint4 now[SETS], next[SETS];
    auto load = [&](int i0, uint4 (&v)[SETS]) {
#pragma unroll
      for (int h = 0; h < SETS; ++h) {
        const int i = i0 + h * 128 + lane * 4;
        v[h] = i < hi ? *reinterpret_cast<const uint4*>(codes + i) : make_uint4(NO_CODE, NO_CODE, NO_CODE, NO_CODE);
      }
    };
    load(lo, now);
    for (int i0 = lo; i0 < hi; i0 += 128 * SETS) {
      load(i0 + 128 * SETS, next);
#pragma unroll
      for (int h = 0; h < SETS; ++h) {
        const int i = i0 + h * 128 + lane * 4;
        const uint32_t w[4] = {now[h].x, i + 1 < hi ? now[h].y : NO_CODE, i + 2 < hi ? now[h].z : NO_CODE, i + 3 < hi ? now[h].w : NO_CODE};
        f(w, i);
        now[h] = next[h];
      }
    }
  };
  int less = 0, noted = stretch < 1 << 23 ? 0 : room + 1;
  walk([&](const uint32_t (&w)[4], int position) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      less += w[j] < base;
      any |= w[j] - base < 65536u;
    }
    if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = w[j] - base < 65536u;
      const unsigned who = __ballot_sync(0xffffffffu, in);
      const int at = noted + __popc(who & ((1u << lane) - 1));
      if (in) {
        atomicAdd(&mine[w[j] & 0xffffu], 1);
        if (at < room) notes[at] = (w[j] & 0xffffu) << 23 | (uint32_t)(position + j - lo);
      }
      noted = min(noted + __popc(who), room + 1);  // (one more: there was no room)
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) less += __shfl_xor_sync(0xffffffffu, less, o);
  if (lane == 0) below[warp] = less;
  __syncthreads();

  int total = 0, c[SORT_WARPS];
  const int row = threadIdx.x;
  if (row < rows) {
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) c[w] = counters[w * rows + row];
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) total += c[w];
  }
  int upto = total;  // sum over the rows up to this thread's
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  int start = upto - total;
#pragma unroll
  for (int w = 0; w < SORT_WARPS; ++w) start += below[w] + (w < warp ? scan[w] : 0);
  if (row < rows) {
    rowptr[own * rows + row] = start;
    if (own == mask && row == rows - 1) rowptr[(mask + 1) * rows] = start + total;
    begin[row] = start, count[row] = total;
    int at = start;
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) {
      counters[w * rows + row] = at;
      at += c[w];
    }
  }
  __syncthreads();

  // Lanes with `in` put position `i` of row `at` in its place, lanes of the same row in their order.
  auto place = [&](bool in, int at, int i) {
    const unsigned who = __ballot_sync(0xffffffffu, in);
    if (who == 0) return;
    if (in) {
      const unsigned same = (who & (who - 1)) ? __match_any_sync(who, at) : who;
      const int to = mine[at] + __popc(same & ((1u << lane) - 1));
      order[to] = i;
      keys[to] = ((uint32_t)at << slots.bits | (uint32_t)own) | (to == begin[at] ? TOKEN_FIRST : 0u) |
                 (to + 1 == begin[at] + count[at] ? TOKEN_LAST : 0u);
      __syncwarp(same);
      if ((same & ((1u << lane) - 1)) == 0) mine[at] = to + __popc(same);
    }
    __syncwarp();
  };
  if (noted <= room) {
    for (int i = lane; i - lane < noted; i += 32) {
      const uint32_t note = i < noted ? notes[i] : 0u;
      place(i < noted, (int)(note >> 23), lo + (int)(note & 0x7fffffu));
    }
  } else {
    walk([&](const uint32_t (&w)[4], int position) {
#pragma unroll
      for (int j = 0; j < 4; ++j) place(w[j] - base < 65536u, (int)(w[j] & 0xffffu), position + j);
    });
  }
}

// -------------------------------------------------------------------------------------------------------------- sums
// A CTA takes `chunk` consecutive places of the sorted list, whatever tokens they belong to, so that a frequent token's positions are
// spread over many CTAs. A token that lies within the chunk is finished; the sum of one that reaches in from the chunk before (part
// 0) or on into the next (part 1) goes to the workspace, and embed_join_kernel adds those up. The last `fills` CTAs clear the rows
// that nobody names instead: most of the bytes, written while others wait for the rows they gather. (First, and two per SM, they
// held up the sums: 50001 x 1001 fp32 108 and 97 us. None of these kernels lets its successor start early: that put the next one's
// CTAs where room was, not where they belong, 38 and 31 us for 8192 x 768 bf16.)
//
// A thread has COLS vectors of VEC columns, blockDim.x vectors apart (single columns where rows are not aligned: four of them share
// the bookkeeping). Bound by memory, behind four kernels in a row: all of it 31 us for 8192 x 768 bf16 and 50257 rows (90 MB; 21 of them
// without the clearing), 80 us for 50001 x 1001 fp32 and 32003 rows (329 MB, 58 of them here). Clearing beside the sort, which
// needs a mark per row, is no faster (34 and 99 us, as stores or as bulk copies): the sorting CTAs' loads then wait behind the writes.
__device__ __forceinline__ void clear_row(uint8_t* row, long long bytes, int lane) {  // one warp; addresses are even
  const int head = (int)min(bytes, (long long)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15));
  const long long body = (bytes - head) / 16;
  if (lane * 2 < head) *reinterpret_cast<uint16_t*>(row + lane * 2) = 0;
  for (long long i = lane; i < body; i += 32) reinterpret_cast<uint4*>(row + head)[i] = make_uint4(0, 0, 0, 0);
  const long long tail = head + body * 16 + lane * 2;
  if (tail < bytes) *reinterpret_cast<uint16_t*>(row + tail) = 0;
}

// p[j] += v[j] * scale, N of them, by the memory: nobody else adds to them meanwhile, so the order is fixed, and nothing waits for the
// old value (with a load and a store a CTA spent a round trip on every token, 46 us for 32768 x 768 bf16).
template <int N>
__device__ __forceinline__ void add_to(float* p, const float (&v)[N], float scale) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int j = 0; j < N; j += 4)
      asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p + j), "f"(v[j] * scale), "f"(v[j + 1] * scale),
                   "f"(v[j + 2] * scale), "f"(v[j + 3] * scale)
                   : "memory");
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(p + j), "f"(v[j] * scale) : "memory");
  }
}

template <typename TI, typename TO, int VEC, int COLS>
__global__ void __launch_bounds__(256)
embed_sum_kernel(const TI* dy, long long ld, const int* order, const uint32_t* keys, const int* rowptr, long long vocab, Slots slots,
                 TO* out, float* parts, int positions, int width, int chunk, int fills, float scale, int accumulate) {
  extern __shared__ int places[];  // [chunk] positions, [chunk] tokens
  grid_dep_wait();
  const int sums = gridDim.x - fills;
  if ((int)blockIdx.x >= sums) {
    if (accumulate) return;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const long long all = (long long)fills * gridDim.y * warps;
    const long long me = ((long long)blockIdx.y * fills + blockIdx.x - sums) * warps + (threadIdx.x >> 5);
    constexpr int SPAN = 8;  // rows a warp looks at together: few, or a small table keeps a part of the warps busy only
    for (long long r0 = me * SPAN; r0 < vocab; r0 += all * SPAN) {
      const long long r = r0 + lane;
      const bool mine = lane < SPAN && r < vocab;
      const int at = mine ? slot_of(slots, (int)r) : 0;
      unsigned empty = __ballot_sync(0xffffffffu, mine && rowptr[at] == rowptr[at + 1]);
      for (; empty; empty &= empty - 1)
        clear_row(reinterpret_cast<uint8_t*>(out + (r0 + __ffs(empty) - 1) * width), (long long)width * sizeof(TO), lane);
    }
    return;
  }
  const int me = blockIdx.x;
  const long long first = (long long)me * chunk;
  uint32_t* token = reinterpret_cast<uint32_t*>(places + chunk);
  for (int i = threadIdx.x; i < chunk && first + i < positions; i += blockDim.x) {  // (those of padding too: their number is on its way)
    places[i] = order[first + i];
    token[i] = keys[first + i];
  }
  const int count = (int)min((long long)chunk, rowptr[slots.rows << slots.bits] - first);
  __syncthreads();
  if (count <= 0) return;
  const int col0 = (blockIdx.y * COLS * blockDim.x + threadIdx.x) * VEC, step = blockDim.x * VEC;

  using V = Vec<TI, VEC>;
  constexpr int AHEAD = COLS > 1 ? 4 : 8;
  float sum[COLS][VEC];
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[c][j] = 0.f;
  bool from_before = !(token[0] & TOKEN_FIRST);
  for (int i0 = 0; i0 < count; i0 += AHEAD) {
    V v[AHEAD][COLS];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int c = 0; c < COLS; ++c)
        if (i0 + u < count && col0 + c * step < width) v[u][c] = *reinterpret_cast<const V*>(dy + places[i0 + u] * ld + col0 + c * step);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = i0 + u;
      if (i >= count) break;
#pragma unroll
      for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[c][j] += to_f32(v[u][c].v[j]);
      const uint32_t t = token[i];
      if (!(t & TOKEN_LAST) && i + 1 < count) continue;
      if (from_before || !(t & TOKEN_LAST)) {
        float* p = parts + (2 * (long long)me + (from_before ? 0 : 1)) * width;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
          if (col0 + c * step < width) *reinterpret_cast<Vec<float, VEC>*>(p + col0 + c * step) = *reinterpret_cast<Vec<float, VEC>*>(sum[c]);
      } else {
        TO* o = out + (long long)(t & TOKEN_ROW) * width;
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          if (col0 + c * step >= width) continue;
          if constexpr (sizeof(TO) == 4) {
            if (accumulate) {
              add_to<VEC>(reinterpret_cast<float*>(o) + col0 + c * step, sum[c], scale);
              continue;
            }
          }
          Vec<TO, VEC> r;
#pragma unroll
          for (int j = 0; j < VEC; ++j) r.v[j] = from_f32<TO>(sum[c][j] * scale);
          *reinterpret_cast<Vec<TO, VEC>*>(o + col0 + c * step) = r;
        }
      }
      from_before = false;
#pragma unroll
      for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[c][j] = 0.f;
    }
  }
}

// ------------------------------------------------------------------------------------------------- gradient of few positions
// Up to EMBED_FEW positions need no sorted list: a CTA per position looks at all ids, goes if its token occurs before, and adds up
// the token's positions in their order otherwise; the CTAs behind clear the rows that are no id's. One kernel and no workspace, where
// the four others are bound by their launches. Us on the GPU for 128 and (the four kernels) 129 positions of 768 bf16: 1000 rows 4.2, 14.4;
// 50257 rows 16.4, 25.6; one token that fills the batch, which is one CTA's work then and the reason for no more positions, 12.3, 14.4.
static constexpr int EMBED_FEW = 128;  // one per thread

template <typename TI, typename TO, typename ID, int VEC>
__global__ void __launch_bounds__(EMBED_FEW)
embed_few_kernel(const ID* ids, int n, const TI* dy, long long ld, TO* out, int width, long long vocab, long long padding, float scale,
                 int accumulate) {
  __shared__ __align__(16) int rows[EMBED_FEW];  // each position's row, -1 for padding and past the last; then the token's positions
  __shared__ unsigned found[EMBED_FEW / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_dep_wait();
  int row = -1;
  if (tid < n) {
    const long long id = ids[tid];
    const bool pad = id == padding;
    if (!pad && blockIdx.x == 0) (void)TNNB_CHECK(id, vocab);
    row = pad ? -1 : id < 0 || id >= vocab ? 0 : (int)id;
  }
  rows[tid] = row;
  __syncthreads();
  if ((int)blockIdx.x >= n) {
    constexpr int SPAN = 8, SHARE = EMBED_FEW / 4;  // rows of a warp at a time; ids that one of a row's four lanes looks at
    const int fills = gridDim.x - n;
    const long long all = (long long)fills * gridDim.y * (EMBED_FEW / 32);
    const long long me = ((long long)blockIdx.y * fills + blockIdx.x - n) * (EMBED_FEW / 32) + warp;
    for (long long r0 = me * SPAN; r0 < vocab; r0 += all * SPAN) {
      const int r = (int)r0 + lane % SPAN;
      int named = 0;
#pragma unroll 4
      for (int i = lane / SPAN * SHARE; i < (lane / SPAN + 1) * SHARE; i += 4) {
        const int4 o = *reinterpret_cast<const int4*>(rows + i);
        named |= (o.x == r) | (o.y == r) | (o.z == r) | (o.w == r);
      }
      named |= __shfl_xor_sync(0xffffffffu, named, 8);
      named |= __shfl_xor_sync(0xffffffffu, named, 16);
      for (unsigned empty = __ballot_sync(0xffffffffu, !named && lane < SPAN && r < vocab); empty; empty &= empty - 1)
        clear_row(reinterpret_cast<uint8_t*>(out + (r0 + __ffs(empty) - 1) * width), (long long)width * sizeof(TO), lane);
    }
    return;
  }
  const int own = rows[blockIdx.x];
  if (own < 0) return;
  const unsigned same = __ballot_sync(0xffffffffu, row == own);
  if (lane == 0) found[warp] = same;
  __syncthreads();
  int before = 0, count = 0;  // of this token: positions in warps before, positions
#pragma unroll
  for (int w = 0; w < EMBED_FEW / 32; ++w) {
    if (w < warp) before += __popc(found[w]);
    count += __popc(found[w]);
  }
  if (row == own) rows[before + __popc(same & ((1u << lane) - 1))] = tid;
  __syncthreads();
  if (rows[0] != (int)blockIdx.x) return;  // occurs before
  const int col = (blockIdx.y * EMBED_FEW + tid) * VEC;
  if (col >= width) return;
  using V = Vec<TI, VEC>;
  constexpr int AHEAD = 16;
  float sum[VEC] = {};
  for (int i0 = 0; i0 < count; i0 += AHEAD) {
    V v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (i0 + u < count) v[u] = *reinterpret_cast<const V*>(dy + rows[i0 + u] * ld + col);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (i0 + u < count)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] += to_f32(v[u].v[j]);
  }
  TO* o = out + (long long)own * width + col;
  if constexpr (sizeof(TO) == 4) {
    if (accumulate) {
      add_to<VEC>(reinterpret_cast<float*>(o), sum, scale);
      return;
    }
  }
  Vec<TO, VEC> w;
#pragma unroll
  for (int j = 0; j < VEC; ++j) w.v[j] = from_f32<TO>(sum[j] * scale);
  *reinterpret_cast<Vec<TO, VEC>*>(o) = w;
}

// Tokens whose places lie in more than one chunk: the CTAs of the chunk such a token begins in add up its parts, each warp every
// eighth one, then the warps in order. 128 columns per CTA.
static constexpr int JOIN_COLS = 128, JOIN_WARPS = 8;
template <typename TO>
__global__ void __launch_bounds__(32 * JOIN_WARPS)
embed_join_kernel(const float* parts, const uint32_t* keys, const int* rowptr, Slots slots, TO* out, int width, int chunk, float scale,
                  int accumulate) {  // CTA i: the places of chunk i and one more exist
  __shared__ float sums[JOIN_WARPS][JOIN_COLS];
  grid_dep_wait();
  const long long next = ((long long)blockIdx.x + 1) * chunk;
  const int n = rowptr[slots.rows << slots.bits];
  const uint32_t key = keys[next - 1];
  if (next >= n || (key & TOKEN_LAST)) return;
  const uint32_t token = key & TOKEN_ROW;
  const int at = slot_of(slots, (int)token);
  if (rowptr[at] < next - chunk) return;  // begins in an earlier chunk
  const int more = (int)((rowptr[at + 1] - 1) / chunk - blockIdx.x);  // chunks after this one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.y * JOIN_COLS + lane;
  float s[JOIN_COLS / 32] = {};
#pragma unroll 8
  for (int k = warp; k <= more; k += JOIN_WARPS) {
    const float* p = parts + (2 * ((long long)blockIdx.x + k) + (k == 0 ? 1 : 0)) * width + col;
#pragma unroll
    for (int q = 0; q < JOIN_COLS / 32; ++q)
      if (col + q * 32 < width) s[q] += p[q * 32];
  }
#pragma unroll
  for (int q = 0; q < JOIN_COLS / 32; ++q) sums[warp][lane + q * 32] = s[q];
  __syncthreads();
  const int c = blockIdx.y * JOIN_COLS + threadIdx.x;
  if (threadIdx.x >= JOIN_COLS || c >= width) return;
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < JOIN_WARPS; ++w) total += sums[w][threadIdx.x];
  TO* o = out + (long long)token * width + c;
  *o = from_f32<TO>(accumulate ? to_f32(*o) + total * scale : total * scale);
}
template <typename TI, typename TO>
static cudaError_t sum_and_join(const void* dy, long long ld, const int* order, const uint32_t* keys, const int* rowptr, int n,
                                long long vocab, const Slots& slots, void* out, float* parts, int width, int chunk, float scale, int accumulate,
                                cudaStream_t st) {
  const int chunks = (n + chunk - 1) / chunk;
  constexpr int PER16 = 16 / sizeof(TI);
  const bool wide = width % PER16 == 0 && ld % PER16 == 0 && !(((uintptr_t)dy | (uintptr_t)out | (uintptr_t)parts) & 15);
  const int per_thread = wide ? PER16 : 4;
  const int vecs = (width + per_thread - 1) / per_thread;
  const int threads = vecs >= 256 ? 256 : (vecs + 31) / 32 * 32;
  const int fills = accumulate ? 0 : 148 * 4;
  const dim3 grid(fills + chunks, (vecs + threads - 1) / threads);
  const size_t smem = 2 * chunk * sizeof(int);
  cudaError_t e;
  if (wide) {
    auto kern = embed_sum_kernel<TI, TO, PER16, 1>;
    e = launch_dependent(kern, grid, dim3(threads), smem, st, (const TI*)dy, ld, order, keys, rowptr, vocab, slots, (TO*)out, parts, n, width,
                         chunk, fills, scale, accumulate);
  } else {
    auto kern = embed_sum_kernel<TI, TO, 1, 4>;
    e = launch_dependent(kern, grid, dim3(threads), smem, st, (const TI*)dy, ld, order, keys, rowptr, vocab, slots, (TO*)out, parts, n, width,
                         chunk, fills, scale, accumulate);
  }
  if (e != cudaSuccess || chunks == 1) return e;
  auto kern = embed_join_kernel<TO>;
  return launch_dependent(kern, dim3(chunks - 1, (width + JOIN_COLS - 1) / JOIN_COLS), dim3(32 * JOIN_WARPS), 0, st, (const float*)parts, keys,
                          rowptr, slots, (TO*)out, width, chunk, scale, accumulate);
}

template <typename TI, typename TO, typename ID>
static cudaError_t few_tokens(const void* ids, int n, const void* dy, long long ld, void* out, int width, long long vocab, long long padding,
                              float scale, int accumulate, cudaStream_t st) {
  constexpr int PER16 = 16 / sizeof(TI);
  const bool wide = width % PER16 == 0 && ld % PER16 == 0 && !(((uintptr_t)dy | (uintptr_t)out) & 15);
  const int per_block = EMBED_FEW * (wide ? PER16 : 1);
  const long long spans = (vocab + 8 * (EMBED_FEW / 32) - 1) / (8 * (EMBED_FEW / 32));  // CTAs that clear 8 rows per warp
  const int fills = accumulate ? 0 : (int)(spans < 148 * 4 ? spans : 148 * 4);
  auto kern = wide ? embed_few_kernel<TI, TO, ID, PER16> : embed_few_kernel<TI, TO, ID, 1>;
  return launch_dependent(kern, dim3(n + fills, (width + per_block - 1) / per_block), dim3(EMBED_FEW), 0, st, (const ID*)ids, n, (const TI*)dy, ld,
                          (TO*)out, width, vocab, padding, scale, accumulate);
}

template <typename ID>
static cudaError_t sort_tokens(const void* ids, int n, long long vocab, long long padding, const Slots& slots, uint32_t* codes, int* order,
                               uint32_t* keys, int* rowptr, cudaStream_t st) {
  auto code = embed_code_kernel<ID>;
  cudaError_t e = launch_dependent(code, dim3((n + 255) / 256), dim3(256), 0, st, (const ID*)ids, n, vocab, padding, slots, codes);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SORT_WARPS * (SORT_ROWS + SORT_NOTES) * (int)sizeof(int));
  if (e != cudaSuccess) return e;
  const int stretch = sort_stretch(n), room = stretch < SORT_NOTES ? stretch : SORT_NOTES;
  return launch_dependent(embed_sort_kernel, dim3(1u << slots.bits), dim3(SORT_WARPS * 32), (size_t)SORT_WARPS * (slots.rows + room) * sizeof(int), st,
                          (const uint32_t*)codes, n, slots, room, order, keys, rowptr);
}

}  // namespace tnnb

using namespace tnnb;

extern "C" {

// out [n, width] = scale * table[ids], rows of `table` `ld` elements apart; zeros where an id is `padding`.
int tnnb_embed_lookup(const void* ids, int ids64, const void* table, long long ld, void* out, long long n, int width, long long vocab,
                      long long padding, float scale, int type, void* stream) {
  if (n < 0 || width <= 0 || vocab <= 0 || ld < width) return -3;
  if (n == 0) return 0;
  const bool known = with_type(type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    constexpr int PER16 = 16 / sizeof(T);
    const bool wide = width % PER16 == 0 && ld % PER16 == 0 && !(((uintptr_t)table | (uintptr_t)out) & 15);
    const int per_warp = 32 * LOOKUP_VECS * (wide ? PER16 : 1);
    const int slices = (width + per_warp - 1) / per_warp;
    const long long items = n * slices, blocks = (items + 7) / 8;
    const int grid = (int)(blocks < 148 * 8 * 4 ? blocks : 148 * 8 * 4);
    auto run = [&](auto id, auto vec) {
      using ID = typename decltype(id)::type;
      constexpr int VEC = decltype(vec)::value;
      embed_lookup_kernel<T, ID, VEC><<<grid, 256, 0, (cudaStream_t)stream>>>((const ID*)ids, (const T*)table, ld, (T*)out, items, slices,
                                                                              width, vocab, padding, scale);
    };
    using Wide = std::integral_constant<int, PER16>;
    using One = std::integral_constant<int, 1>;
    if (ids64) wide ? run(TypeTag<long long>(), Wide()) : run(TypeTag<long long>(), One());
    else wide ? run(TypeTag<int>(), Wide()) : run(TypeTag<int>(), One());
  });
  if (!known) return -4;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e - 1000;
}

// out [vocab, width] (+)= scale * the sum of the rows of dy [n, width] (rows `ld` apart) per token. `out` has dy's type or is fp32;
// without `accumulate` every row of it is written. Workspaces (none up to 128 positions): `codes` uint32[n rounded up to 4] on 16 bytes, `order` and `keys` int[n],
// `rowptr` int[vocab + vocab / 256 + 129], `parts` float[2 * ceil(n / chunk) * width] on 16 bytes.
int tnnb_embed_grad(const void* ids, int ids64, const void* dy, long long ld, void* out, void* codes, void* order, void* keys, void* rowptr,
                    void* parts, int n, int width, long long vocab, long long padding, float scale, int type, int out_type, int accumulate, int chunk,
                    void* stream) {
  if (n < 0 || width <= 0 || vocab <= 0 || vocab > (1 << 24) || ld < width || chunk < 1 || chunk > 1024) return -3;
  if (out_type != VT_FP32 && (out_type != type || accumulate)) return -4;
  const cudaStream_t st = (cudaStream_t)stream;
  if (n == 0) {
    if (accumulate) return 0;
    const cudaError_t e = cudaMemsetAsync(out, 0, (size_t)vocab * width * value_size(out_type), st);
    return e == cudaSuccess ? 0 : -(int)e - 1000;
  }
  cudaError_t e = cudaSuccess;
  if (n <= EMBED_FEW) {
    const bool known = with_type(type, [&](auto tag) {
      using T = typename decltype(tag)::type;
      auto go = [&](auto to) {
        using TO = typename decltype(to)::type;
        auto few = ids64 ? few_tokens<T, TO, long long> : few_tokens<T, TO, int>;
        return few(ids, n, dy, ld, out, width, vocab, padding, scale, accumulate, st);
      };
      e = out_type == VT_FP32 ? go(TypeTag<float>()) : go(TypeTag<T>());
    });
    if (!known) return -4;
    return e == cudaSuccess ? 0 : -(int)e - 1000;
  }
  const Slots slots = slots_of(vocab);
  e = ids64 ? sort_tokens<long long>(ids, n, vocab, padding, slots, (uint32_t*)codes, (int*)order, (uint32_t*)keys, (int*)rowptr, st)
                        : sort_tokens<int>(ids, n, vocab, padding, slots, (uint32_t*)codes, (int*)order, (uint32_t*)keys, (int*)rowptr, st);
  if (e != cudaSuccess) return -(int)e - 1000;
  const bool known = with_type(type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    auto go = [&](auto to) {
      return sum_and_join<T, typename decltype(to)::type>(dy, ld, (const int*)order, (const uint32_t*)keys, (const int*)rowptr, n, vocab, slots, out,
                                                          (float*)parts, width, chunk, scale, accumulate, st);
    };
    e = out_type == VT_FP32 ? go(TypeTag<float>()) : go(TypeTag<T>());
  });
  if (!known) return -4;
  return e == cudaSuccess ? 0 : -(int)e - 1000;
}

}  // extern "C"
