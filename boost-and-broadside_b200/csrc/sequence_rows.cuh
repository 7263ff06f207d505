// What the kernels of the recurrent layers outside the trunk share (causal_conv.cu, selective_scan.cu,
// selective_scan_bwd.cu): element types, wide accesses, the scalar functions of a step.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "bnb_trunk.h"
#include "tensor_common.cuh"   // pairs of floats in one instruction, fast exponential and reciprocal

namespace bnb {
namespace seq {

using tensor::F2;
using tensor::f2;
using tensor::halves;
using tensor::mul;
using tensor::add;
using tensor::fma;
using tensor::ex2_fast;
using tensor::rcp_fast;

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

// 1 / (1 + e^-v).  Results of 16-bit calls are rounded to 11 bits or fewer, where the fast exponential and division
// (2 units in the last place of 24 each, for arguments that matter) are far below the rounding; float32 calls take the exact ones.
template <typename T>
__device__ __forceinline__ float sigmoid(float v) {
  if constexpr (sizeof(T) == 2) return __fdividef(1.0f, 1.0f + __expf(-v));
  return 1.0f / (1.0f + expf(-v));
}
constexpr float LOG2E = 1.4426950408889634f;

// N neighbouring elements as pairs of floats, and back.  One element alone has a partner that is never stored.
template <int N> constexpr int PAIRS = (N + 1) / 2;
template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, F2 (&f)[PAIRS<N>]) {
#pragma unroll
  for (int i = 0; i < PAIRS<N>; ++i) f[i] = f2(to_f(p.v[2 * i]), 2 * i + 1 < N ? to_f(p.v[2 * i + 1 < N ? 2 * i + 1 : 0]) : 0.f);
}
template <int N, typename T>
__device__ __forceinline__ void store(T* at, const F2 (&f)[PAIRS<N>]) {
  Pack<T, N> p;
#pragma unroll
  for (int i = 0; i < N; ++i) p.v[i] = from_f<T>(i & 1 ? halves(f[i / 2]).y : halves(f[i / 2]).x);
  *reinterpret_cast<Pack<T, N>*>(at) = p;
}
// sigmoid of a pair
template <typename T>
__device__ __forceinline__ F2 sigmoid(F2 v) {
  if constexpr (sizeof(T) == 4) {
    const float2 s = halves(v);
    return f2(sigmoid<float>(s.x), sigmoid<float>(s.y));
  }
  const float2 m = halves(mul(v, f2(-LOG2E))), den = halves(add(f2(ex2_fast(m.x), ex2_fast(m.y)), f2(1.0f)));
  return f2(rcp_fast(den.x), rcp_fast(den.y));
}

// Steps of row r that are looked at.
__device__ __forceinline__ int row_steps(const int32_t* lengths, int r, int steps) {
  return lengths ? max(0, min(lengths[r], steps)) : steps;
}

inline size_t elem_bytes(int element) { return element == BNB_ELEM_F32 ? 4 : 2; }
inline size_t round256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace seq
}  // namespace bnb
