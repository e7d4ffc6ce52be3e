// Element types of the kernels that take bf16, fp16 and fp32 alike, and vectors of them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace tnnb {

enum ValueType : int { VT_BF16 = 0, VT_FP16 = 1, VT_FP32 = 2 };

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

// N consecutive elements, moved by accesses of up to 16 bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Vec {
  T v[N];
};

// f(type tag) for a ValueType; false for one that does not exist.
template <typename T> struct TypeTag { using type = T; };
template <typename F>
static bool with_type(int vt, F f) {
  if (vt == VT_BF16) f(TypeTag<__nv_bfloat16>());
  else if (vt == VT_FP16) f(TypeTag<__half>());
  else if (vt == VT_FP32) f(TypeTag<float>());
  else return false;
  return true;
}
static inline int value_size(int vt) { return vt == VT_FP32 ? 4 : 2; }

}  // namespace tnnb
