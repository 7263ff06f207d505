// AdamW over many tensors in one launch, with the gradients' global norm in one before it (formulas in include/bnb_trunk.h).
//
// Memory bounds it: 28 bytes an element of float32 with states of 32 bits, 16 with 8 bits; for the some hundred small tensors of a
// policy, launches do, so the list of tensors is an argument of the kernel and nothing is copied to the device.  The tensors are cut into chunks of 2048
// elements; a CTA takes chunks one behind the other, so it looks a tensor up once and then moves on.  A warp takes 256 neighbouring
// elements, eight a lane, which are a block of 8-bit states: its scales are maxima over the warp.
//
// Sums of the norm are 64 bits from 8 elements on and are added in a fixed order by every CTA of the step for itself.  The last CTA of a step moves the
// tensors' counters on, when all have read them.
#include <algorithm>

#include <cuda_fp8.h>

#include "launch_after.h"
#include "sequence_rows.cuh"

namespace bnb {
namespace adamw {
namespace {

using namespace seq;
using tensor::let_next_start;
using tensor::wait_for_previous;

constexpr int SMS = 148, THREADS = 256, CHUNK = THREADS * 8, BLOCK = 256;
constexpr int CTAS = SMS * 8;
static_assert(CTAS == BNB_GRAD_NORM_PARTS, "a part a CTA");

// Arguments of a kernel end at 32 764 bytes, and a longer list takes longer to launch.
template <int MOST> struct Tensors {
  int n;
  uint32_t chunks;
  uint32_t first[MOST + 1];   // chunks before each tensor; all of them behind the last
  BnbAdamTensor t[MOST];
};
constexpr int FEW = 32, SOME = 128, MANY = 360;

// The tensor of a chunk, by all lanes of a warp: two steps where halving takes nine, each of which waits for memory.
template <int MOST>
__device__ __forceinline__ int tensor_of(const Tensors<MOST>& l, uint32_t chunk) {
  constexpr int STRIDE = (MOST + 31) / 32;
  const int lane = threadIdx.x & 31;
  const int part = __popc(__ballot_sync(0xffffffffu, l.first[min(lane * STRIDE, MOST)] <= chunk)) - 1;
  const int i = part * STRIDE + lane;
  const unsigned in = __ballot_sync(0xffffffffu, lane < STRIDE && i < l.n && l.first[min(i, MOST)] <= chunk);
  return part * STRIDE + __popc(in) - 1;
}

// Eight neighbouring elements from `at` on of `n`; `wide`: all there, on their natural boundary of eight.
template <typename T>
__device__ __forceinline__ void take(const T* from, int64_t at, int64_t n, bool wide, float (&f)[8]) {
  if (wide) {
    if constexpr (sizeof(T) == 4) {
      asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]) : "l"(from + at));
    } else {
      load<T, 8>(from + at, f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = at + i < n ? to_f(from[at + i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void put(T* to, int64_t at, int64_t n, bool wide, const float (&f)[8]) {
  if (wide) {
    if constexpr (sizeof(T) == 4) {
      asm volatile("st.global.v8.f32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
                   ::"f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]), "l"(to + at) : "memory");
    } else {
      store<T, 8>(to + at, f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (at + i < n) to[at + i] = from_f<T>(f[i]);
  }
}
__device__ __forceinline__ void take_any(int element, const void* from, int64_t at, int64_t n, bool wide, float (&f)[8]) {
  if (element == BNB_ELEM_F32) take(static_cast<const float*>(from), at, n, wide, f);
  else if (element == BNB_ELEM_BF16) take(static_cast<const __nv_bfloat16*>(from), at, n, wide, f);
  else take(static_cast<const __half*>(from), at, n, wide, f);
}
__device__ __forceinline__ void put_any(int element, void* to, int64_t at, int64_t n, bool wide, const float (&f)[8]) {
  if (element == BNB_ELEM_F32) put(static_cast<float*>(to), at, n, wide, f);
  else if (element == BNB_ELEM_BF16) put(static_cast<__nv_bfloat16*>(to), at, n, wide, f);
  else put(static_cast<__half*>(to), at, n, wide, f);
}
__device__ __forceinline__ bool on(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
__device__ __forceinline__ bool values_lie_well(int element, const void* p) { return on(p, element == BNB_ELEM_F32 ? 32 : 16); }

// Codes of e4m3 as they lie, eight.
__device__ __forceinline__ uint2 take_codes(const uint8_t* from, int64_t at, int64_t n, bool wide) {
  if (wide) return *reinterpret_cast<const uint2*>(from + at);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (at + i < n) w[i / 4] |= (uint32_t)from[at + i] << (8 * (i % 4));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void put_codes(uint8_t* to, int64_t at, int64_t n, bool wide, uint2 v) {
  if (wide) {
    *reinterpret_cast<uint2*>(to + at) = v;
  } else {
    const uint32_t w[2] = {v.x, v.y};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i < n) to[at + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
  }
}
__device__ __forceinline__ void decode(uint2 codes, float scale, float (&f)[8]) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i % 2))), __NV_E4M3));
    const float2 v = __half22float2(h);
    f[2 * i] = v.x * scale;
    f[2 * i + 1] = v.y * scale;
  }
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int by = 16; by; by >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, by));
  return v;
}
// Square root by the instruction, within a unit in the last place; numbers below the normal ones are not taken for 0.
__device__ __forceinline__ float root_of(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// The exponent (in place) of the scale that takes `most` to 128 .. 256.
__device__ __forceinline__ uint32_t scale_exponent(float most) { return (uint32_t)max((int)(__float_as_uint(most) >> 23) - 7, 1); }
__device__ __forceinline__ float power(uint32_t exponent) { return __uint_as_float(exponent << 23); }
// 20 random bits.
__device__ __forceinline__ uint32_t noise(uint64_t position, uint32_t key) {
  uint32_t h = ((uint32_t)position + (uint32_t)(position >> 32) * 0x632BE5ABu) * 0x9E3779B1u + key;
  h ^= h >> 15;
  h *= 0x6C8E944Du;
  h ^= h >> 13;
  h *= 0x5B297A4Du;
  return (h ^ (h >> 16)) >> 12;
}

// ------------------------------------------------------------------ norm

template <int MOST>
__global__ void __launch_bounds__(THREADS) k_norm(const __grid_constant__ Tensors<MOST> l, double* parts, bool add) {
  __shared__ double sums[THREADS / 32];
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t c0 = (uint64_t)l.chunks * blockIdx.x / gridDim.x, c1 = (uint64_t)l.chunks * (blockIdx.x + 1) / gridDim.x;
  double sum = 0;
  int i = c0 < c1 ? tensor_of(l, c0) : 0;
  for (uint32_t c = c0; c < c1; ++c) {
    while (l.first[i + 1] <= c) ++i;
    const BnbAdamTensor& t = l.t[i];
    const int64_t at = (int64_t)(c - l.first[i]) * CHUNK + threadIdx.x * 8;
    if (at >= t.n) continue;
    float g[8];
    take_any(t.element, t.g, at, t.n, values_lie_well(t.element, t.g) && at + 8 <= t.n, g);
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v = fmaf(g[k], g[k], v);
    sum += v;
  }
#pragma unroll
  for (int by = 16; by; by >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, by);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < THREADS / 32; ++w) sum += sums[w];
  if (add) {
    parts[blockIdx.x] += sum;
  } else {
    parts[blockIdx.x] = sum;
    for (int i = blockIdx.x + gridDim.x; i < CTAS; i += gridDim.x) parts[i] = 0;
  }
}

// ------------------------------------------------------------------ step

struct Hyper {
  BnbAdamW c;
  float beta1, rest1, beta2, rest2;   // beta and 1 - beta
  float log1, log2_;                  // natural logarithms of the betas
};

// Eight elements of a lane as they come from memory.
template <bool EIGHT>
struct Piece {
  float p[8], g[8];
  float m[EIGHT ? 1 : 8], v[EIGHT ? 1 : 8];
  uint2 codes_m, codes_v;
  float scale_m, scale_v;
  int64_t at;       // of the lane's first element, behind the tensor's end where the warp has nothing
  int tensor;
  bool whole;
};

// With 8-bit states a chunk's loads are on their way while the one before is rounded and written.
template <int MOST, bool EIGHT>
__global__ void __launch_bounds__(THREADS) k_step(const __grid_constant__ Tensors<MOST> l, const __grid_constant__ Hyper h) {
  __shared__ double sums[THREADS / 32];
  __shared__ bool last;
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t c0 = (uint64_t)l.chunks * blockIdx.x / gridDim.x, c1 = (uint64_t)l.chunks * (blockIdx.x + 1) / gridDim.x;
  int i = c0 < c1 ? tensor_of(l, c0) : 0;
  auto fetch = [&](uint32_t c, Piece<EIGHT>& x) {
    while (l.first[i + 1] <= c) ++i;
    const BnbAdamTensor& t = l.t[i];
    const int64_t start = (int64_t)(c - l.first[i]) * CHUNK + warp * BLOCK;
    x.at = start + lane * 8;
    x.tensor = i;
    x.whole = x.at + 8 <= t.n;
    if (start >= t.n) return;
    take_any(t.element, t.p, x.at, t.n, x.whole && values_lie_well(t.element, t.p), x.p);
    take_any(t.element, t.g, x.at, t.n, x.whole && values_lie_well(t.element, t.g), x.g);
    if constexpr (EIGHT) {
      x.codes_m = take_codes(static_cast<const uint8_t*>(t.m), x.at, t.n, x.whole && on(t.m, 8));
      x.codes_v = take_codes(static_cast<const uint8_t*>(t.v), x.at, t.n, x.whole && on(t.v, 8));
      x.scale_m = t.m_scale[start / BLOCK];
      x.scale_v = t.v_scale[start / BLOCK];
    } else {
      take(static_cast<const float*>(t.m), x.at, t.n, x.whole && on(t.m, 32), x.m);
      take(static_cast<const float*>(t.v), x.at, t.n, x.whole && on(t.v, 32), x.v);
    }
  };
  Piece<EIGHT> x;
  if (c0 < c1) fetch(c0, x);
  const float lr = h.c.lr_device ? *h.c.lr_device : h.c.lr, decay = lr * h.c.weight_decay;
  float clip = 1.f;
  if (h.c.norm_parts) {
    double sum = 0;
    for (int k = threadIdx.x; k < h.c.n_norm_parts; k += THREADS) sum += h.c.norm_parts[k];
#pragma unroll
    for (int by = 16; by; by >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, by);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    sum = sums[0];
    for (int w = 1; w < THREADS / 32; ++w) sum += sums[w];
    const float norm = (float)sqrt(sum);
    if (h.c.norm && blockIdx.x == 0 && threadIdx.x == 0) *h.c.norm = norm;
    if (!isfinite(norm)) return;   // all CTAs do: nobody counts
    clip = fminf(1.f, h.c.max_norm / (norm + 1e-6f));
  }
  int known = -1;
  float rate = 0.f, root = 0.f;
  uint32_t key = 0;
  for (uint32_t c = c0; c < c1; ++c) {
    const BnbAdamTensor& t = l.t[x.tensor];
    if (x.at - lane * 8 >= t.n) {   // the warp's
      if (c + 1 < c1) fetch(c + 1, x);
      continue;
    }
    if (known != x.tensor) {
      known = x.tensor;
      const float steps = *t.step + 1.f;
      rate = lr / -expm1f(steps * h.log1);
      root = 1.f / sqrtf(-expm1f(steps * h.log2_));
      key = h.c.seed * 0x5D2F63B9u + (uint32_t)steps * 0x3C6EF36Bu;
    }
    float m[8], v[8];
    if constexpr (EIGHT) {
      decode(x.codes_m, x.scale_m, m);
      decode(x.codes_v, x.scale_v, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= v[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) m[k] = x.m[k], v[k] = x.v[k];
    }
    float p[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float gk = x.g[k] * clip;
      m[k] = fmaf(m[k], h.beta1, gk * h.rest1);
      v[k] = fmaf(v[k], h.beta2, gk * gk * h.rest2);
      const float r = root_of(v[k]);
      // the quotient by a reciprocal, 2 units in the last place of a change that is a small part of p; 0 for a divisor above 2^126
      p[k] = fmaf(-x.p[k], decay, x.p[k]) - rate * __fdividef(m[k], fmaf(r, root, h.c.eps));
      if constexpr (EIGHT) v[k] = r;
    }
    const int64_t at = x.at;
    const bool whole = x.whole;
    if constexpr (EIGHT)
      if (c + 1 < c1) fetch(c + 1, x);
    put_any(t.element, t.p, at, t.n, whole && values_lie_well(t.element, t.p), p);
    if constexpr (EIGHT) {
      float most_m = 0.f, most_r = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        most_m = fmaxf(most_m, fabsf(m[k]));
        most_r = fmaxf(most_r, v[k]);
      }
      const uint32_t em = scale_exponent(warp_max(most_m)), er = scale_exponent(warp_max(most_r));
      const float by_m = power(254 - em), by_r = power(254 - er);   // exact
      uint32_t cm[2] = {0, 0}, cr[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        const float a = m[k] * by_m, b = m[k + 1] * by_m;
        // an infinity saturates in the conversion: NaN instead
        const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(fmaf(a, 0.f, a), fmaf(b, 0.f, b)), __NV_SATFINITE, __NV_E4M3);
        cm[k / 4] |= two << (8 * (k % 4));
      }
      const uint64_t position = (uint64_t)(t.position + at);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float r = v[k] * by_r;
        // three bits of the mantissa are kept, exponents start at 2^-6; NaN and infinities end beyond the largest code
        const int q = (int)((__float_as_uint(r) + noise(position + k, key)) >> 20) - ((127 - 7) << 3);
        const int code = r == 0.f ? 0 : min(max(q, 8), 0x7F);
        cr[k / 4] |= (uint32_t)code << (8 * (k % 4));
      }
      put_codes(static_cast<uint8_t*>(t.m), at, t.n, whole && on(t.m, 8), make_uint2(cm[0], cm[1]));
      put_codes(static_cast<uint8_t*>(t.v), at, t.n, whole && on(t.v, 8), make_uint2(cr[0], cr[1]));
      if (lane == 0) {
        t.m_scale[at / BLOCK] = power(em);
        t.v_scale[at / BLOCK] = power(er);
      }
    } else {
      put(static_cast<float*>(t.m), at, t.n, whole && on(t.m, 32), m);
      put(static_cast<float*>(t.v), at, t.n, whole && on(t.v, 32), v);
      if (c + 1 < c1) fetch(c + 1, x);
    }
  }
  // the last CTA counts: every other one has read what it needs
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(h.c.control, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  for (int k = threadIdx.x; k < l.n; k += THREADS) *l.t[k].step += 1.f;
  if (threadIdx.x == 0) *h.c.control = 0;
}

// ------------------------------------------------------------------ the calls

int check(const BnbAdamTensor* t, int n) {
  if (n < 0) return BNB_ERR_BAD_ARGUMENT;
  if (n && !t) return BNB_ERR_NULL_POINTER;
  for (int i = 0; i < n; ++i) {
    if (t[i].n < 0 || t[i].element < 0 || t[i].element > 2) return BNB_ERR_BAD_ARGUMENT;
    if (t[i].n > (int64_t)1 << 40) return BNB_ERR_UNSUPPORTED_DIMS;   // chunks of all tensors of a launch in 32 bits
    if (t[i].n && !t[i].g) return BNB_ERR_NULL_POINTER;
  }
  return BNB_OK;
}
template <int MOST>
Tensors<MOST> list_of(const BnbAdamTensor* t, int n) {
  Tensors<MOST> l;
  l.n = n;
  l.chunks = 0;
  for (int i = 0; i < n; ++i) {
    l.t[i] = t[i];
    l.first[i] = l.chunks;
    l.chunks += (uint32_t)((t[i].n + CHUNK - 1) / CHUNK);
  }
  for (int i = n; i <= MOST; ++i) l.first[i] = l.chunks;
  return l;
}
unsigned ctas_of(uint32_t chunks) { return std::max(1u, std::min(chunks, (uint32_t)CTAS)); }

template <int MOST>
int norm(const BnbAdamTensor* t, int n, double* parts, bool add, cudaStream_t st) {
  const Tensors<MOST> l = list_of<MOST>(t, n);
  return launch_after(k_norm<MOST>, dim3(ctas_of(l.chunks)), THREADS, 0, st, l, parts, add);
}
template <int MOST>
int step(const BnbAdamTensor* t, int n, const Hyper& h, cudaStream_t st) {
  const Tensors<MOST> l = list_of<MOST>(t, n);
  return h.c.state_bits == 8 ? launch_after(k_step<MOST, true>, dim3(ctas_of(l.chunks)), THREADS, 0, st, l, h)
                             : launch_after(k_step<MOST, false>, dim3(ctas_of(l.chunks)), THREADS, 0, st, l, h);
}

}  // namespace
}  // namespace adamw
}  // namespace bnb

using namespace bnb;
using namespace bnb::adamw;

extern "C" int bnb_grad_norm(const BnbAdamTensor* t, int n, double* parts, void* stream) {
  if (const int st = check(t, n)) return st;
  if (!parts) return BNB_ERR_NULL_POINTER;
  const auto s = static_cast<cudaStream_t>(stream);
  int i = 0;
  do {
    const int k = std::min(n - i, MANY);
    if (const int r = k <= FEW ? norm<FEW>(t + i, k, parts, i > 0, s) : k <= SOME ? norm<SOME>(t + i, k, parts, i > 0, s) : norm<MANY>(t + i, k, parts, i > 0, s)) return r;
    i += k;
  } while (i < n);
  return BNB_OK;
}

extern "C" int bnb_adamw_step(const BnbAdamTensor* t, int n, const BnbAdamW* c, void* stream) {
  if (const int st = check(t, n)) return st;
  if (!c || !c->control) return BNB_ERR_NULL_POINTER;
  if ((c->state_bits != 8 && c->state_bits != 32) || !(c->beta1 >= 0 && c->beta1 < 1) || !(c->beta2 >= 0 && c->beta2 < 1) || !(c->eps >= 0)) return BNB_ERR_BAD_ARGUMENT;
  if (c->norm_parts && (c->n_norm_parts < 1 || !(c->max_norm >= 0))) return BNB_ERR_BAD_ARGUMENT;
  for (int i = 0; i < n; ++i) {
    if (!t[i].step) return BNB_ERR_NULL_POINTER;
    if (t[i].n && (!t[i].p || !t[i].m || !t[i].v || (c->state_bits == 8 && (!t[i].m_scale || !t[i].v_scale)))) return BNB_ERR_NULL_POINTER;
  }
  Hyper h{};
  h.c = *c;
  h.beta1 = (float)c->beta1, h.rest1 = (float)(1 - c->beta1);
  h.beta2 = (float)c->beta2, h.rest2 = (float)(1 - c->beta2);
  h.log1 = (float)log(c->beta1), h.log2_ = (float)log(c->beta2);
  const auto s = static_cast<cudaStream_t>(stream);
  for (int i = 0; i < n;) {
    const int k = std::min(n - i, MANY);
    if (const int r = k <= FEW ? step<FEW>(t + i, k, h, s) : k <= SOME ? step<SOME>(t + i, k, h, s) : step<MANY>(t + i, k, h, s)) return r;
    i += k;
  }
  return BNB_OK;
}
