// What the kernels of the recurrent layers outside the trunk share (causal_conv.cu, selective_scan.cu,
// selective_scan_bwd.cu): element types, wide accesses, the scalar functions of a step.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "bnb_trunk.h"
#include "tensor_common.cuh"   // fast exponential and reciprocal, pairs of floats in one instruction

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

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> __device__ __forceinline__ uint32_t both(float lo, float hi);
template <> __device__ __forceinline__ uint32_t both<__nv_bfloat16>(float lo, float hi) { return tensor::pack_bf16(lo, hi); }
template <> __device__ __forceinline__ uint32_t both<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// N neighbouring elements as they lie in memory, moved as one access of 2, 4, 8 or 16 bytes: words until they are used, so that what is on its
// way takes no more registers than its bytes.
template <int BYTES> struct Words { uint32_t w[BYTES / 4]; };
template <> struct Words<2> { unsigned short w[1]; };
template <typename T, int N> using Raw = Words<sizeof(T) * N>;
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T* at) {
  Raw<T, N> r;
  constexpr int B = sizeof(T) * N;
  if constexpr (B == 2) r.w[0] = *reinterpret_cast<const unsigned short*>(at);
  else if constexpr (B == 4) r.w[0] = *reinterpret_cast<const uint32_t*>(at);
  else if constexpr (B == 8) { const uint2 v = *reinterpret_cast<const uint2*>(at); r.w[0] = v.x, r.w[1] = v.y; }
  else { const uint4 v = *reinterpret_cast<const uint4*>(at); r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w; }
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void unpack(const Raw<T, N>& r, float (&f)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __uint_as_float(r.w[i]);
  } else if constexpr (N == 1) {
    f[0] = to_f(*reinterpret_cast<const T*>(&r.w[0]));
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[2 * i] = tensor::bf16_lo(r.w[i]), f[2 * i + 1] = tensor::bf16_hi(r.w[i]);
      } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      }
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void load(const T* at, float (&f)[N]) { unpack<T, N>(load_raw<T, N>(at), f); }
template <typename T, int N>
__device__ __forceinline__ void store(T* at, const float (&f)[N]) {
  if constexpr (N == 1) {
    *at = from_f<T>(f[0]);
  } else {
    constexpr int W = sizeof(T) * N / 4;
    uint32_t w[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
      else w[i] = both<T>(f[2 * i], f[2 * i + 1]);
    }
    if constexpr (W == 1) *reinterpret_cast<uint32_t*>(at) = w[0];
    else if constexpr (W == 2) *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
    else
#pragma unroll
      for (int i = 0; i < W; i += 4) *reinterpret_cast<uint4*>(at + i * 4 / sizeof(T)) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
}

// 1 / (1 + e^-v).  Results of 16-bit calls are rounded to 11 bits or fewer, where the fast exponential and division
// (2 units in the last place of 24 each, for arguments that matter) are far below the rounding; float32 calls take the exact ones here.  The decays
// and step sizes of the scan (selective_scan.cuh) take the fast ones in every type.
template <typename T>
__device__ __forceinline__ float sigmoid(float v) {
  if constexpr (sizeof(T) == 2) return rcp_fast(1.0f + ex2_fast(v * -LOG2E));
  return 1.0f / (1.0f + expf(-v));
}

// Steps of row r that are looked at.
__device__ __forceinline__ int row_steps(const int32_t* lengths, int r, int steps) {
  return lengths ? max(0, min(lengths[r], steps)) : steps;
}

inline size_t elem_bytes(int element) { return element == BNB_ELEM_F32 ? 4 : 2; }
inline size_t round256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace seq
}  // namespace bnb
