// The element-wise halves of the Muon optimizer's step around its Newton-Schulz products (newton_schulz.cu), and AdamW for the
// parameters that are no matrices.
//
//   buffer <- mu buffer + (1 - mu) g,   u = mu buffer + (1 - mu) g (Nesterov) or the buffer
//   w <- w - lr (factor o + decay w)    with o = the orthogonalised u, in bf16
//
// Weights and gradients lie in flat buffers at given offsets, equal matrices are one launch; state and updates are packed. One pass
// over the bytes each: bound by memory (24 matrices of 2304 x 768: momentum 120 us, 5.7 TB/s, application 94 us, 5.4 TB/s; AdamW on 80
// million parameters 392 us, 6.1 TB/s). The learning rate and the gradients' scale may come from device memory (`hyper`, as for the
// other optimizers), so that a captured step sees new ones.
#include "ptx.cuh"
#include "values.cuh"

namespace tnnb {

// Four elements per thread where everything is aligned (`wide`), else one.
template <int N>
__global__ void __launch_bounds__(256)
muon_momentum_kernel(const float* __restrict__ grads, const long long* __restrict__ offsets, float* __restrict__ buffer, float* __restrict__ u,
                     long long size, float mu, int nesterov, float gscale, const float* __restrict__ hyper) {
  if (hyper) gscale = hyper[3];
  const float* g = grads + offsets[blockIdx.y];
  buffer += blockIdx.y * size, u += blockIdx.y * size;
  using V = Vec<float, N>;
  for (long long i = (blockIdx.x * 256ll + threadIdx.x) * N; i < size; i += gridDim.x * 256ll * N) {
    const V gv = *reinterpret_cast<const V*>(g + i);
    V b = *reinterpret_cast<const V*>(buffer + i), o;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float add = (1.f - mu) * gv.v[j] * gscale;
      b.v[j] = fmaf(mu, b.v[j], add);
      o.v[j] = nesterov ? fmaf(mu, b.v[j], add) : b.v[j];
    }
    *reinterpret_cast<V*>(buffer + i) = b;
    *reinterpret_cast<V*>(u + i) = o;
  }
}

template <int N>
__global__ void __launch_bounds__(256)
muon_apply_kernel(float* __restrict__ master, __nv_bfloat16* __restrict__ low, const long long* __restrict__ offsets,
                  const __nv_bfloat16* __restrict__ update, long long size, float lr, float factor, float decay,
                  const float* __restrict__ hyper) {
  if (hyper) lr = hyper[0];
  float* w = master + offsets[blockIdx.y];
  __nv_bfloat16* l = low ? low + offsets[blockIdx.y] : nullptr;
  update += blockIdx.y * size;
  for (long long i = (blockIdx.x * 256ll + threadIdx.x) * N; i < size; i += gridDim.x * 256ll * N) {
    Vec<float, N> v = *reinterpret_cast<const Vec<float, N>*>(w + i);
    const Vec<__nv_bfloat16, N> o = *reinterpret_cast<const Vec<__nv_bfloat16, N>*>(update + i);
    Vec<__nv_bfloat16, N> r;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v.v[j] -= lr * fmaf(factor, to_f32(o.v[j]), decay * v.v[j]);
      r.v[j] = from_f32<__nv_bfloat16>(v.v[j]);
    }
    *reinterpret_cast<Vec<float, N>*>(w + i) = v;
    if (l) *reinterpret_cast<Vec<__nv_bfloat16, N>*>(l + i) = r;
  }
}

// Adam (the formula of loss_optim.cu) over pieces of the flat buffers: a block takes piece {offset, length, place of its state}. One that
// does not lie in the buffers (`total` elements, `states` of state) is left out and recorded.
__global__ void __launch_bounds__(256)
adam_pieces_kernel(float* __restrict__ master, __nv_bfloat16* __restrict__ low, const float* __restrict__ grads, float* __restrict__ m,
                   float* __restrict__ v, const long long* __restrict__ pieces, long long total, long long states, float lr, float b1, float b2,
                   float eps, float wd, float bc1, float bc2, float gscale, float lr_ratio, const float* __restrict__ hyper, int* status) {
  if (hyper) lr = hyper[0], bc1 = hyper[1], bc2 = hyper[2], gscale = hyper[3];
  lr *= lr_ratio;
  const long long* p = pieces + 3ll * blockIdx.x;
  const long long at = p[0], n = p[1], st = p[2];
  if (at < 0 || st < 0 || n < 0 || n > total || n > states || at > total - n || st > states - n) {
    if (threadIdx.x == 0 && status) atomicCAS(status, 0, ST_BAD_ARG);
    return;
  }
  const float ib1 = 1.f / bc1, ib2 = 1.f / bc2;
  for (long long i = threadIdx.x; i < n; i += 256) {
    const float g = grads[at + i] * gscale;
    const float mi = b1 * m[st + i] + (1.f - b1) * g, vi = b2 * v[st + i] + (1.f - b2) * g * g;
    float w = master[at + i];
    w = w - lr * (mi * ib1) / (sqrtf(vi * ib2) + eps) - wd * lr * w;
    m[st + i] = mi, v[st + i] = vi, master[at + i] = w;
    if (low) low[at + i] = __float2bfloat16(w);
  }
}

static int muon_grid(long long size, int per_thread, int count) {
  const long long want = (size + 256 * per_thread - 1) / (256 * per_thread), most = (148 * 8 + count - 1) / count;
  return (int)(want < most ? want : most);
}

}  // namespace tnnb

using namespace tnnb;

extern "C" {

// `count` matrices of `size` elements at offsets[i] (device) of the flat fp32 gradients; buffer and u fp32 [count][size]. `wide`: size and every
// offset are multiples of 4.
int tnnb_muon_momentum(const void* grads, const void* offsets, void* buffer, void* u, int count, long long size, float mu, int nesterov,
                       float gscale, const void* hyper, int wide, void* stream) {
  if (count <= 0 || count > 65535 || size <= 0 || (wide && size % 4)) return -3;
  wide = wide && !(((uintptr_t)grads | (uintptr_t)buffer | (uintptr_t)u) & 15);
  const dim3 grid(muon_grid(size, wide ? 4 : 1, count), count);
  (wide ? muon_momentum_kernel<4> : muon_momentum_kernel<1>)<<<grid, 256, 0, (cudaStream_t)stream>>>(
      (const float*)grads, (const long long*)offsets, (float*)buffer, (float*)u, size, mu, nesterov, gscale, (const float*)hyper);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e - 1000;
}

// The same matrices of the flat fp32 weights and, where given, of their bf16 copy; update bf16 [count][size].
int tnnb_muon_apply(void* master, void* low, const void* offsets, const void* update, int count, long long size, float lr, float factor,
                    float decay, const void* hyper, int wide, void* stream) {
  if (count <= 0 || count > 65535 || size <= 0 || (wide && size % 4)) return -3;
  wide = wide && !(((uintptr_t)master | (uintptr_t)update) & 15) && !((uintptr_t)low & 7);
  const dim3 grid(muon_grid(size, wide ? 4 : 1, count), count);
  (wide ? muon_apply_kernel<4> : muon_apply_kernel<1>)<<<grid, 256, 0, (cudaStream_t)stream>>>(
      (float*)master, (__nv_bfloat16*)low, (const long long*)offsets, (const __nv_bfloat16*)update, size, lr, factor, decay,
      (const float*)hyper);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e - 1000;
}

// pieces: int64 [count][3] on the device: offset in the flat buffers (`total` elements), length, place in m and v (`states`).
int tnnb_adam_pieces(void* master, void* low, const void* grads, void* m, void* v, const void* pieces, int count, long long total,
                     long long states, float lr, float b1, float b2, float eps, float wd, float bc1, float bc2, float gscale, float lr_ratio,
                     const void* hyper, int* status, void* stream) {
  if (count < 0 || total < 0 || states < 0) return -3;
  if (count == 0) return 0;
  adam_pieces_kernel<<<count, 256, 0, (cudaStream_t)stream>>>((float*)master, (__nv_bfloat16*)low, (const float*)grads, (float*)m, (float*)v,
                                                             (const long long*)pieces, total, states, lr, b1, b2, eps, wd, bc1, bc2, gscale,
                                                             lr_ratio, (const float*)hyper, status);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -(int)e - 1000;
}

}  // extern "C"
