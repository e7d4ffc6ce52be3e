// Token embedding with scaling, and its gradient by sorted tokens.
//
//   forward   y[t] = scale * W[id[t]]                       (zeros where id[t] is the padding index)
//   gradient  dW[v] = scale * sum over {t : id[t] = v} of dy[t]
//
// bf16, fp16 and fp32, any width; ids of 32 or 64 bits. Products and sums are fp32, rounded once. An id outside the table reads
// (and adds to) row 0 like the layers' embedding kernels (elementwise.cu); the bounds-checked build records it.
//
// The gradient adds up in a fixed order: the positions of each token ascending, in chunks of the sorted list, then the chunks
// ascending. No atomics on values: the same inputs give the same bits, and a row is written once, in the table's own type.
#include "launch.cuh"
#include "ptx.cuh"
#include "values.cuh"

TNNB_BOUNDS_TU(embedding)

namespace tnnb {

// ------------------------------------------------------------------------------------------------------------ lookup
// A warp copies up to LOOKUP_VECS vectors per lane of one row: all of a row's loads are in flight together, and rows are many.
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
// Positions sorted by token, stable, without a pass over global counters: every CTA owns a range of table rows, reads ALL ids
// (they come from L2: 64 KB for 8192 tokens) and picks its own. The number of ids below its range is the place of its part of the
// list, so no CTA waits for another. Within the CTA each warp walks a contiguous stretch of the ids and has a counter per row:
// counts, then starting places (rows ascending, warps ascending within a row), then the places themselves. Rows nobody names are
// cleared here, by the CTA that knows, so that the whole table's gradient is written exactly once.
static constexpr int SORT_WARPS = 32;
static constexpr int SORT_ROWS = 512;  // most rows of a CTA: 64 KB of counters, two CTAs per SM

template <typename ID>
__device__ __forceinline__ long long sort_row(const ID* ids, int i, long long vocab, long long padding) {
  const long long id = ids[i];
  if (id == padding) return -1;
  (void)TNNB_CHECK(id, vocab);
  return id < 0 || id >= vocab ? 0 : id;
}

template <typename ID>
__global__ void __launch_bounds__(SORT_WARPS * 32)
embed_sort_kernel(const ID* ids, int n, long long vocab, long long padding, int rows_each,
                                                                     int* order, int* keys, int* rowptr, uint8_t* clear,
                                                                     long long row_bytes) {
  grid_dep_launch();
  grid_dep_wait();
  extern __shared__ int counters[];  // [SORT_WARPS][rows_each]
  __shared__ int below[SORT_WARPS], scan[SORT_WARPS];
  __shared__ uint8_t empty[SORT_ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long v0 = (long long)blockIdx.x * rows_each;
  const int rows = (int)min((long long)rows_each, vocab - v0);
  for (int i = threadIdx.x; i < SORT_WARPS * rows_each; i += blockDim.x) counters[i] = 0;
  __syncthreads();

  const int stretch = ((n + SORT_WARPS - 1) / SORT_WARPS + 31) / 32 * 32;
  const int lo = min((long long)n, (long long)warp * stretch), hi = min((long long)n, (long long)lo + stretch);
  int* mine = counters + warp * rows_each;
  int less = 0;
  constexpr int AHEAD = 4;
  for (int i0 = lo; i0 < hi; i0 += 32 * AHEAD) {
    long long r[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) r[u] = i0 + u * 32 + lane < hi ? sort_row(ids, i0 + u * 32 + lane, vocab, padding) : -1;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      less += r[u] >= 0 && r[u] < v0;
      const bool in = r[u] >= v0 && r[u] < v0 + rows;
      const unsigned who = __ballot_sync(0xffffffffu, in);
      if (who == 0) continue;
      if (in) {
        const int at = (int)(r[u] - v0);
        const unsigned same = __match_any_sync(who, at);
        if ((same & ((1u << lane) - 1)) == 0) mine[at] += __popc(same);
      }
      __syncwarp();
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) less += __shfl_xor_sync(0xffffffffu, less, o);
  if (lane == 0) below[warp] = less;
  __syncthreads();

  int total = 0;
  if ((int)threadIdx.x < rows)
    for (int w = 0; w < SORT_WARPS; ++w) {
      const int c = counters[w * rows_each + threadIdx.x];
      counters[w * rows_each + threadIdx.x] = total;
      total += c;
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
  for (int w = 0; w < SORT_WARPS; ++w) start += below[w] + (w < warp ? scan[w] : 0);
  if ((int)threadIdx.x < rows) {
    rowptr[v0 + threadIdx.x] = start;
    if (v0 + threadIdx.x == vocab - 1) rowptr[vocab] = start + total;
    for (int w = 0; w < SORT_WARPS; ++w) counters[w * rows_each + threadIdx.x] += start;
    empty[threadIdx.x] = total == 0;
  }
  __syncthreads();

  for (int i0 = lo; i0 < hi; i0 += 32 * AHEAD) {
    long long r[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) r[u] = i0 + u * 32 + lane < hi ? sort_row(ids, i0 + u * 32 + lane, vocab, padding) : -1;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const bool in = r[u] >= v0 && r[u] < v0 + rows;
      const unsigned who = __ballot_sync(0xffffffffu, in);
      if (who == 0) continue;
      int at = 0;
      unsigned same = 0;
      if (in) {
        at = (int)(r[u] - v0);
        same = __match_any_sync(who, at);
        const int to = mine[at] + __popc(same & ((1u << lane) - 1));
        order[to] = i0 + u * 32 + lane;
        keys[to] = (int)r[u];
      }
      __syncwarp();
      if (in && (same & ((1u << lane) - 1)) == 0) mine[at] += __popc(same);
      __syncwarp();
    }
  }
  if (clear == nullptr) return;
  const bool wide = ((reinterpret_cast<uintptr_t>(clear) | row_bytes) & 15) == 0;
  for (int r = warp; r < rows; r += SORT_WARPS) {
    if (!empty[r]) continue;
    uint8_t* row = clear + (v0 + r) * row_bytes;
    if (wide) {
      for (long long b = lane * 16; b < row_bytes; b += 32 * 16) *reinterpret_cast<uint4*>(row + b) = make_uint4(0, 0, 0, 0);
    } else {
      for (long long b = lane * 2; b < row_bytes; b += 32 * 2) *reinterpret_cast<uint16_t*>(row + b) = 0;  // elements have two bytes or four
    }
  }
}

// -------------------------------------------------------------------------------------------------------------- sums
// A CTA takes `chunk` consecutive places of the sorted list, whatever tokens they belong to, so that a frequent token's positions are
// spread over many CTAs. A token that lies within the chunk is finished; the sum of one that reaches in from the chunk before (part
// 0) or on into the next (part 1) goes to the workspace, and embed_join_kernel adds those up.
template <typename TI, typename TO, int VEC>
__global__ void __launch_bounds__(256)
embed_sum_kernel(const TI* dy, long long ld, const int* order, const int* keys, const int* rowptr,
                                                        long long vocab, TO* out, float* parts, int width, int chunk, float scale,
                                                        int accumulate) {
  extern __shared__ int places[];  // [chunk] positions, [chunk + 1] tokens
  grid_dep_launch();
  grid_dep_wait();
  const int n = rowptr[vocab];
  const long long first = (long long)blockIdx.x * chunk;
  if (first >= n) return;
  const int count = (int)min((long long)chunk, n - first);
  int* token = places + chunk;
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    places[i] = order[first + i];
    token[i] = keys[first + i];
  }
  if (threadIdx.x == 0) token[count] = -1;
  __syncthreads();
  const int col = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  if (col >= width) return;
  const bool from_before = rowptr[token[0]] < first;
  const bool goes_on = rowptr[token[count - 1] + 1] > first + count;

  using V = Vec<TI, VEC>;
  constexpr int AHEAD = 8;
  float sum[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
  bool opening = true;  // the chunk's first token
  for (int i0 = 0; i0 < count; i0 += AHEAD) {
    V v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (i0 + u < count) v[u] = *reinterpret_cast<const V*>(dy + places[i0 + u] * ld + col);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = i0 + u;
      if (i >= count) break;
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] += to_f32(v[u].v[j]);
      if (token[i + 1] == token[i]) continue;
      const bool head = opening && from_before, open = head || (i + 1 == count && goes_on);
      opening = false;
      if (open) {
        float* p = parts + (2 * (long long)blockIdx.x + (head ? 0 : 1)) * width + col;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p[j] = sum[j];
      } else {
        TO* o = out + (long long)token[i] * width + col;
        Vec<TO, VEC> r;
        if (accumulate) r = *reinterpret_cast<const Vec<TO, VEC>*>(o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) r.v[j] = from_f32<TO>(accumulate ? to_f32(r.v[j]) + sum[j] * scale : sum[j] * scale);
        *reinterpret_cast<Vec<TO, VEC>*>(o) = r;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
    }
  }
}

// Tokens whose places lie in more than one chunk: the CTAs of the chunk such a token begins in add up its parts, each warp every
// eighth one, then the warps in order. 128 columns per CTA.
static constexpr int JOIN_COLS = 128, JOIN_WARPS = 8;
template <typename TO>
__global__ void __launch_bounds__(32 * JOIN_WARPS)
embed_join_kernel(const float* parts, const int* keys, const int* rowptr, long long vocab,
                                                                     TO* out, int width, int chunk, float scale, int accumulate) {
  __shared__ float sums[JOIN_WARPS][JOIN_COLS];
  grid_dep_launch();
  grid_dep_wait();
  const int n = rowptr[vocab];
  const long long next = ((long long)blockIdx.x + 1) * chunk;
  if (next >= n) return;
  const int token = keys[next];
  if (keys[next - 1] != token || rowptr[token] < next - chunk) return;
  const int more = (int)((rowptr[token + 1] - 1) / chunk - blockIdx.x);  // chunks after this one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.y * JOIN_COLS + lane;
  float s[JOIN_COLS / 32] = {};
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
static cudaError_t sum_and_join(const void* dy, long long ld, const int* order, const int* keys, const int* rowptr, int n, long long vocab,
                                void* out, float* parts, int width, int chunk, float scale, int accumulate, cudaStream_t st) {
  const int chunks = (n + chunk - 1) / chunk;
  constexpr int PER16 = 16 / sizeof(TI);
  const bool wide = width % PER16 == 0 && ld % PER16 == 0 && !(((uintptr_t)dy | (uintptr_t)out | (uintptr_t)parts) & 15);
  const int vecs = wide ? width / PER16 : width;
  const int threads = vecs >= 256 ? 256 : (vecs + 31) / 32 * 32;
  const dim3 grid(chunks, (vecs + threads - 1) / threads);
  const size_t smem = (2 * chunk + 1) * sizeof(int);
  cudaError_t e;
  if (wide) {
    auto kern = embed_sum_kernel<TI, TO, PER16>;
    e = launch_dependent(kern, grid, dim3(threads), smem, st, (const TI*)dy, ld, order, keys, rowptr, vocab, (TO*)out, parts, width, chunk,
                         scale, accumulate);
  } else {
    auto kern = embed_sum_kernel<TI, TO, 1>;
    e = launch_dependent(kern, grid, dim3(threads), smem, st, (const TI*)dy, ld, order, keys, rowptr, vocab, (TO*)out, parts, width, chunk,
                         scale, accumulate);
  }
  if (e != cudaSuccess || chunks == 1) return e;
  auto kern = embed_join_kernel<TO>;
  return launch_dependent(kern, dim3(chunks - 1, (width + JOIN_COLS - 1) / JOIN_COLS), dim3(32 * JOIN_WARPS), 0, st, (const float*)parts, keys,
                          rowptr, vocab, (TO*)out, width, chunk, scale, accumulate);
}

template <typename ID>
static cudaError_t sort_tokens(const void* ids, int n, long long vocab, long long padding, int* order, int* keys, int* rowptr, void* clear,
                               long long row_bytes, cudaStream_t st) {
  // one CTA per SM where the rows per CTA allow it, else two
  const long long one = (vocab + 147) / 148, two = (vocab + 295) / 296;
  const int rows_each = (int)(one <= SORT_ROWS ? one : two <= SORT_ROWS ? two : SORT_ROWS);
  const size_t smem = (size_t)SORT_WARPS * rows_each * sizeof(int);
  auto kern = embed_sort_kernel<ID>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SORT_WARPS * SORT_ROWS * (int)sizeof(int));
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, dim3((unsigned)((vocab + rows_each - 1) / rows_each)), dim3(SORT_WARPS * 32), smem, st, (const ID*)ids, n, vocab,
                          padding, rows_each, order, keys, rowptr, (uint8_t*)clear, row_bytes);
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
// without `accumulate` every row of it is written. Workspaces: `order` and `keys` int[n], `rowptr` int[vocab + 1], `parts`
// float[2 * ceil(n / chunk) * width] on 16 bytes.
int tnnb_embed_grad(const void* ids, int ids64, const void* dy, long long ld, void* out, void* order, void* keys, void* rowptr, void* parts,
                    int n, int width, long long vocab, long long padding, float scale, int type, int out_type, int accumulate, int chunk,
                    void* stream) {
  if (n < 0 || width <= 0 || vocab <= 0 || vocab > 0x7ffffffe || ld < width || chunk < 1 || chunk > 1024) return -3;
  if (out_type != VT_FP32 && (out_type != type || accumulate)) return -4;
  const cudaStream_t st = (cudaStream_t)stream;
  if (n == 0) {
    if (accumulate) return 0;
    const cudaError_t e = cudaMemsetAsync(out, 0, (size_t)vocab * width * value_size(out_type), st);
    return e == cudaSuccess ? 0 : -(int)e - 1000;
  }
  void* clear = accumulate ? nullptr : out;
  const long long row_bytes = (long long)width * value_size(out_type);
  cudaError_t e = ids64 ? sort_tokens<long long>(ids, n, vocab, padding, (int*)order, (int*)keys, (int*)rowptr, clear, row_bytes, st)
                        : sort_tokens<int>(ids, n, vocab, padding, (int*)order, (int*)keys, (int*)rowptr, clear, row_bytes, st);
  if (e != cudaSuccess) return -(int)e - 1000;
  const bool known = with_type(type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    auto go = [&](auto to) {
      return sum_and_join<T, typename decltype(to)::type>(dy, ld, (const int*)order, (const int*)keys, (const int*)rowptr, n, vocab, out,
                                                          (float*)parts, width, chunk, scale, accumulate, st);
    };
    e = out_type == VT_FP32 ? go(TypeTag<float>()) : go(TypeTag<T>());
  });
  if (!known) return -4;
  return e == cudaSuccess ? 0 : -(int)e - 1000;
}

}  // extern "C"
