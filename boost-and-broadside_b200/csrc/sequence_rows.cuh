// What the kernels of the recurrent layers outside the trunk share (causal_conv.cu, selective_scan.cu,
// selective_scan_bwd.cu): element types, wide accesses, the scalar functions of a step.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "bnb_trunk.h"

namespace bnb {
namespace seq {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// N neighbouring elements, moved as one access when their bytes are 4, 8 or 16.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack { T v[N]; };
template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = to_f(p.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store(T* at, const float (&f)[N]) {
  Pack<T, N> p;
#pragma unroll
  for (int i = 0; i < N; ++i) p.v[i] = from_f<T>(f[i]);
  *reinterpret_cast<Pack<T, N>*>(at) = p;
}

// 1 / (1 + e^-v).  Results of 16-bit calls are rounded to 11 bits or fewer, where the fast exponential and division
// (2 units in the last place of 24 each, for arguments that matter) are far below the rounding; float32 calls take the exact ones.
template <typename T>
__device__ __forceinline__ float sigmoid(float v) {
  if constexpr (sizeof(T) == 2) return __fdividef(1.0f, 1.0f + __expf(-v));
  return 1.0f / (1.0f + expf(-v));
}
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f;

// Steps of row r that are looked at.
__device__ __forceinline__ int row_steps(const int32_t* lengths, int r, int steps) {
  return lengths ? max(0, min(lengths[r], steps)) : steps;
}

inline size_t elem_bytes(int element) { return element == BNB_ELEM_F32 ? 4 : 2; }
inline size_t round256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace seq
}  // namespace bnb
