// AdamW over many tensors in one launch, with the gradients' global norm in one before it (formulas in include/bnb_trunk.h).
//
// Memory bounds it: 28 bytes an element of float32 with states of 32 bits, 16 with 8 bits; for the some hundred small tensors of a
// policy, launches do, so the list of tensors is an argument of the kernel and nothing is copied to the device.  The tensors are cut into chunks of 2048
// elements, which the CTAs take in turn, so that all of them work in one place of memory at a time: with a range of chunks to each, 8-bit states, whose
// chunks are 2 KB, took 140 us for 40 M elements instead of 108, runs of two chunks 134.  A warp takes 256 neighbouring elements, eight a lane,
// which are a block of 8-bit states: its scales are maxima over the warp.
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

// Arguments of a kernel end at 32 764 bytes, and a longer list takes longer to launch.  (A copy of it in a CTA's shared memory took the norm of
// 99 tensors from 5 to 17 us: arguments are read fast only where all lanes read the same.)
template <int MOST> struct Tensors {
  int n;
  uint32_t chunks;
  uint32_t first[MOST + 2];   // chunks before each tensor; all of them behind the last
  BnbAdamTensor t[MOST];
};
constexpr int MANY = 360;
// The tensor of a CTA's first chunk, by all lanes of a warp: two steps where halving takes nine, each of which waits for memory.  A later chunk's is a few
// tensors on.
template <int MOST>
__device__ __forceinline__ int tensor_of(const Tensors<MOST>& l, uint32_t chunk) {
  constexpr int STRIDE = (MOST + 31) / 32;
  const int lane = threadIdx.x & 31;
  const int part = __popc(__ballot_sync(0xffffffffu, l.first[min(lane * STRIDE, MOST)] <= chunk)) - 1;
  const int i = part * STRIDE + lane;
  const unsigned in = __ballot_sync(0xffffffffu, lane < STRIDE && i < l.n && l.first[min(i, MOST)] <= chunk);
  return part * STRIDE + __popc(in) - 1;
}
template <int MOST>
__device__ __forceinline__ void move_on(const Tensors<MOST>& l, int& i, uint32_t chunk) {
  while (l.first[i + 1] <= chunk) ++i;
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
__device__ __forceinline__ void decode(uint2 codes, F2 (&f)[4]) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i % 2))), __NV_E4M3)));
    f[i] = f2(v.x, v.y);
  }
}
// Maxima over a warp, NaN where any is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int by = 16; by; by >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, by));
  return v;
}
// Square root by the instruction, within a unit in the last place.  For 8-bit states, which are bound by their arithmetic, numbers below 2^-126 are 0;
// taking them as they are is three instructions more.
template <bool FLUSH>
__device__ __forceinline__ float root_of(float v) {
  float r;
  if constexpr (FLUSH) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  else asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// The exponent (in place) of the scale that takes `most` to 128 .. 256.
__device__ __forceinline__ uint32_t scale_exponent(float most) { return (uint32_t)max((int)(__float_as_uint(most) >> 23) - 7, 1); }
__device__ __forceinline__ float power(uint32_t exponent) { return __uint_as_float(exponent << 23); }
// 20 random bits of a position: its product with a constant and the key, mixed.  Eight neighbours from a multiple of eight on share the upper half.
__device__ __forceinline__ uint32_t spread(uint64_t position, uint32_t key) {
  return ((uint32_t)position + (uint32_t)(position >> 32) * 0x632BE5ABu) * 0x9E3779B1u + key;
}
__device__ __forceinline__ uint32_t noise(uint32_t h) {
  h ^= h >> 15;
  h *= 0x6C8E944Du;
  h ^= h >> 13;
  h *= 0x5B297A4Du;
  return (h ^ (h >> 16)) >> 12;
}
// The codes of eight values within 0 .. 256, whose block has no others: m to nearest; r, not negative, at random, 0 alone to 0.  Added to the bits that
// e4m3 has not, the noise carries into the last that it has in proportion; what is left converts exactly.
__device__ __forceinline__ uint2 codes_of(const F2 (&m)[4], F2 by) {
  uint32_t c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) c[k] = __nv_cvt_float2_to_fp8x2(halves(mul(m[k], by)), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
}
__device__ __forceinline__ uint2 random_codes_of(const F2 (&r)[4], F2 by, uint32_t h) {
  uint32_t c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const F2 x = mul(r[k], by);
    const float2 v = halves(x), up = halves(mul(x, f2(0x1p100f)));
    float2 y;
    // no smaller than the least normal number, except 0
    y.x = __uint_as_float((__float_as_uint(fmaxf(v.x, fminf(up.x, 0x1p-6f))) + noise(h + (2 * k) * 0x9E3779B1u)) & 0xFFF00000u);
    y.y = __uint_as_float((__float_as_uint(fmaxf(v.y, fminf(up.y, 0x1p-6f))) + noise(h + (2 * k + 1) * 0x9E3779B1u)) & 0xFFF00000u);
    c[k] = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
}
// ------------------------------------------------------------------ norm

template <int MOST>
__global__ void __launch_bounds__(THREADS) k_norm(const __grid_constant__ Tensors<MOST> l, double* parts, bool add) {
  __shared__ double sums[THREADS / 32];
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum = 0;
  int i = blockIdx.x < l.chunks ? tensor_of(l, blockIdx.x) : 0;
  for (uint32_t c = blockIdx.x; c < l.chunks; c += gridDim.x) {
    move_on(l, i, c);
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

// What a CTA of a step knows before its first chunk: the clipping of the gradients (false: their norm is not finite, and nobody counts).
__device__ __forceinline__ bool clipping(const Hyper& h, double (&sums)[THREADS / 32], float& clip) {
  clip = 1.f;
  if (!h.c.norm_parts) return true;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
  clip = fminf(1.f, h.c.max_norm / (norm + 1e-6f));
  return isfinite(norm);
}
// A tensor's step: the learning rate and the root's factor with their corrections, the key of its random numbers.
struct Rates { float rate, root; uint32_t key; };
__device__ __forceinline__ Rates rates_of(const Hyper& h, float lr, float steps) {
  return {lr / -expm1f(steps * h.log1), 1.f / sqrtf(-expm1f(steps * h.log2_)), h.c.seed * 0x5D2F63B9u + (uint32_t)steps * 0x3C6EF36Bu};
}
// Eight elements: m and v come multiplied by their betas; with EIGHT, v goes back as its root.
template <bool EIGHT>
__device__ __forceinline__ void update(const Hyper& h, const Rates& k, float clip, float decay, const float (&g)[8], float (&p)[8], F2 (&m)[4], F2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const F2 gi = mul(f2(g[2 * i], g[2 * i + 1]), f2(clip)), old = f2(p[2 * i], p[2 * i + 1]);
    m[i] = fma(gi, f2(h.rest1), m[i]);
    v[i] = fma(mul(gi, gi), f2(h.rest2), v[i]);
    const float2 vs = halves(v[i]);
    const F2 r = f2(root_of<EIGHT>(vs.x), root_of<EIGHT>(vs.y));
    // the quotient by a reciprocal, 2 units in the last place of a change that is a small part of p
    const float2 d = halves(fma(r, f2(k.root), f2(h.c.eps)));
    const float2 q = halves(add(fma(old, f2(-decay), old), mul(mul(m[i], f2(-k.rate)), f2(rcp_fast(d.x), rcp_fast(d.y)))));
    p[2 * i] = q.x, p[2 * i + 1] = q.y;
    if constexpr (EIGHT) v[i] = r;
  }
}
__device__ __forceinline__ void flat(const F2 (&f)[4], float (&o)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 s = halves(f[k]);
    o[2 * k] = s.x, o[2 * k + 1] = s.y;
  }
}
// The last CTA counts: every other one has read what it needs.
template <int MOST>
__device__ __forceinline__ void count(const Tensors<MOST>& l, int32_t* control) {
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(control, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  for (int k = threadIdx.x; k < l.n; k += THREADS) *l.t[k].step += 1.f;
  if (threadIdx.x == 0) *control = 0;
}

// Eight elements of a lane as they come from memory.
template <bool EIGHT>
struct Piece {
  float p[8], g[8];
  float m[EIGHT ? 1 : 8], v[EIGHT ? 1 : 8];
  uint2 codes_m, codes_v;
  float scale_m, scale_v;
  float step;       // the tensor's
  int64_t at;       // of the lane's first element
  int tensor;
};

// With 8-bit states a chunk's loads are on their way while the one before is rounded and written.  These are bound by their arithmetic and its latency, 66
// instructions an element at 56 % of the issue slots with 24 warps an SM: one wave of CTAs, 149 us for 40 M elements (eight CTAs an SM 157; four an SM at
// 64 registers 159, two 168).  States of 32 bits are bound by memory, 98 % of the measured copy rate with float32 parameters; 16-bit ones leave fewer bytes
// on their way, 79 % (two CTAs an SM 69 %; four 89 %, but float32 92 %).
constexpr int RESIDENT = 3;
// TYPE: all parameters' element, or MIXED.
constexpr int MIXED = -1;
template <int MOST, bool EIGHT, int TYPE>
__global__ void __launch_bounds__(THREADS, RESIDENT) k_step(const __grid_constant__ Tensors<MOST> l, const __grid_constant__ Hyper h) {
  __shared__ double sums[THREADS / 32];
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t chunks = l.chunks;
  const float lr = h.c.lr_device ? *h.c.lr_device : h.c.lr, decay = lr * h.c.weight_decay;
  int known = -1, i = blockIdx.x < chunks ? tensor_of(l, blockIdx.x) : 0;
  auto element = [](const BnbAdamTensor& t) { return TYPE == MIXED ? t.element : TYPE; };
  auto fetch = [&](uint32_t c, Piece<EIGHT>& x) {
    if (c >= chunks) return;
    move_on(l, i, c);
    const BnbAdamTensor& t = l.t[i];
    const int64_t start = (int64_t)(c - l.first[i]) * CHUNK + warp * BLOCK, at = start + lane * 8;
    x.at = at;
    x.tensor = i;
    if (start >= t.n) return;   // the warp's
    x.step = *t.step;
    const bool whole = at + 8 <= t.n;
    take_any(element(t), t.p, at, t.n, whole && values_lie_well(element(t), t.p), x.p);
    take_any(element(t), t.g, at, t.n, whole && values_lie_well(element(t), t.g), x.g);
    if constexpr (EIGHT) {
      x.codes_m = take_codes(static_cast<const uint8_t*>(t.m), at, t.n, whole && on(t.m, 8));
      x.codes_v = take_codes(static_cast<const uint8_t*>(t.v), at, t.n, whole && on(t.v, 8));
      x.scale_m = t.m_scale[start / BLOCK];
      x.scale_v = t.v_scale[start / BLOCK];
    } else {
      take(static_cast<const float*>(t.m), at, t.n, whole && on(t.m, 32), x.m);
      take(static_cast<const float*>(t.v), at, t.n, whole && on(t.v, 32), x.v);
    }
  };
  Piece<EIGHT> x;
  fetch(blockIdx.x, x);
  float clip;
  if (!clipping(h, sums, clip)) return;   // while the first loads are on their way; all CTAs do: nobody counts
  Rates k{};
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const BnbAdamTensor& t = l.t[x.tensor];
    const int64_t at = x.at, start = at - lane * 8;
    if (start >= t.n) {   // the warp's
      fetch(c + gridDim.x, x);
      continue;
    }
    if (known != x.tensor) {
      known = x.tensor;
      k = rates_of(h, lr, x.step + 1.f);
    }
    const bool whole = at + 8 <= t.n;
    F2 m[4], v[4];
    if constexpr (EIGHT) {
      decode(x.codes_m, m);
      decode(x.codes_v, v);
      // scales are powers of two: beta times a scale is exact
      const F2 bm = f2(h.beta1 * x.scale_m), bv = f2(h.beta2 * fminf(x.scale_v * x.scale_v, 3.4e38f));
#pragma unroll
      for (int j = 0; j < 4; ++j) m[j] = mul(m[j], bm), v[j] = mul(mul(v[j], v[j]), bv);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) m[j] = mul(f2(x.m[2 * j], x.m[2 * j + 1]), f2(h.beta1)), v[j] = mul(f2(x.v[2 * j], x.v[2 * j + 1]), f2(h.beta2));
    }
    update<EIGHT>(h, k, clip, decay, x.g, x.p, m, v);
    put_any(element(t), t.p, at, t.n, whole && values_lie_well(element(t), t.p), x.p);
    float ms[8], vs[8];
    flat(m, ms);
    flat(v, vs);
    if constexpr (EIGHT) {
      fetch(c + gridDim.x, x);
      float most_m = 0.f, most_r = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        most_m = max_nan(most_m, fabsf(ms[j]));
        most_r = max_nan(most_r, vs[j]);
      }
      most_m = warp_max(most_m);
      most_r = warp_max(most_r);
      const bool broken = !(isfinite(most_m) && isfinite(most_r));   // the warp's
      if (broken) {   // the scales are those of what is finite
        most_m = most_r = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (isfinite(ms[j])) most_m = fmaxf(most_m, fabsf(ms[j]));
          if (isfinite(vs[j])) most_r = fmaxf(most_r, vs[j]);
        }
        most_m = warp_max(most_m);
        most_r = warp_max(most_r);
      }
      const uint32_t em = scale_exponent(most_m), er = scale_exponent(most_r);
      uint2 codes_m = codes_of(m, f2(power(254 - em)));   // by powers of two: exact
      uint2 codes_r = random_codes_of(v, f2(power(254 - er)), spread((uint64_t)(t.position + at), k.key));
      if (broken) {   // what is not is NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t nan = 0x7Fu << (8 * (j % 4)), all = 0xFFu << (8 * (j % 4));
          uint32_t &a = j < 4 ? codes_m.x : codes_m.y, &b = j < 4 ? codes_r.x : codes_r.y;
          if (!isfinite(ms[j])) a = (a & ~all) | nan;
          if (!isfinite(vs[j])) b = (b & ~all) | nan;
        }
      }
      put_codes(static_cast<uint8_t*>(t.m), at, t.n, whole && on(t.m, 8), codes_m);
      put_codes(static_cast<uint8_t*>(t.v), at, t.n, whole && on(t.v, 8), codes_r);
      if (lane == 0) {
        t.m_scale[start / BLOCK] = power(em);
        t.v_scale[start / BLOCK] = power(er);
      }
    } else {
      put(static_cast<float*>(t.m), at, t.n, whole && on(t.m, 32), ms);
      put(static_cast<float*>(t.v), at, t.n, whole && on(t.v, 32), vs);
      fetch(c + gridDim.x, x);
    }
  }
  count(l, h.c.control);
}

// ------------------------------------------------------------------ the calls

int check(const BnbAdamTensor* t, int n) {
  if (n < 0) return BNB_ERR_BAD_ARGUMENT;
  if (n && !t) return BNB_ERR_NULL_POINTER;
  for (int i = 0; i < n; ++i) {
    if (t[i].n < 0 || t[i].element < 0 || t[i].element > 2) return BNB_ERR_BAD_ARGUMENT;
    if (t[i].position & (BLOCK - 1)) return BNB_ERR_BAD_ARGUMENT;
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
  for (int i = n; i < MOST + 2; ++i) l.first[i] = l.chunks;
  return l;
}
unsigned ctas_of(uint32_t chunks) { return std::max(1u, std::min(chunks, (uint32_t)CTAS)); }

// f of the shortest list that holds n tensors.
template <class F>
int with_list(int n, F f) {
  if (n <= 32) return f(std::integral_constant<int, 32>());
  if (n <= 112) return f(std::integral_constant<int, 112>());
  if (n <= 192) return f(std::integral_constant<int, 192>());
  return f(std::integral_constant<int, MANY>());
}
template <int MOST>
int norm(const BnbAdamTensor* t, int n, double* parts, bool add, cudaStream_t st) {
  const Tensors<MOST> l = list_of<MOST>(t, n);
  return launch_after(k_norm<MOST>, dim3(ctas_of(l.chunks)), THREADS, 0, st, l, parts, add);
}
template <int MOST>
int step(const BnbAdamTensor* t, int n, const Hyper& h, cudaStream_t st) {
  const Tensors<MOST> l = list_of<MOST>(t, n);
  int type = n ? t[0].element : (int)MIXED;
  for (int i = 1; i < n; ++i) type = t[i].element == type ? type : MIXED;
  const unsigned all = ctas_of(l.chunks), wave = std::min(all, (unsigned)(SMS * RESIDENT));
  auto with = [&](auto kernel, unsigned ctas) { return launch_after(kernel, dim3(ctas), THREADS, 0, st, l, h); };
  if (h.c.state_bits == 8)
    return type == BNB_ELEM_F32 ? with(k_step<MOST, true, BNB_ELEM_F32>, wave) : type == BNB_ELEM_BF16 ? with(k_step<MOST, true, BNB_ELEM_BF16>, wave)
         : type == BNB_ELEM_F16 ? with(k_step<MOST, true, BNB_ELEM_F16>, wave) : with(k_step<MOST, true, MIXED>, wave);
  return type == BNB_ELEM_F32 ? with(k_step<MOST, false, BNB_ELEM_F32>, all) : type == BNB_ELEM_BF16 ? with(k_step<MOST, false, BNB_ELEM_BF16>, all)
       : type == BNB_ELEM_F16 ? with(k_step<MOST, false, BNB_ELEM_F16>, all) : with(k_step<MOST, false, MIXED>, all);
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
    if (const int r = with_list(k, [&](auto most) { return norm<decltype(most)::value>(t + i, k, parts, i > 0, s); })) return r;
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
    if (const int r = with_list(k, [&](auto most) { return step<decltype(most)::value>(t + i, k, h, s); })) return r;
    i += k;
  }
  return BNB_OK;
}
