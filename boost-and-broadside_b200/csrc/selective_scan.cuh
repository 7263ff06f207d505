// What the forward and the backward of the selective state space recurrence share (selective_scan.cu,
// selective_scan_bwd.cu).
//
// Layout of the work.  KL neighbouring lanes own a channel of a row, four states each (KL = states / 4 rounded up to a power of two;
// states behind the last have a = 0 and b = c = 0, so they stay 0, or become NaN where p u is infinite, and y with them).  A CTA walks along time in chunks with a tile of channels of one
// row: what is per channel and step (softplus, gate, p u) is computed once by the CTA's threads together and stands in shared memory,
// and so do the chunk's b and c, which the tile's channels share.  Steps at and behind a row's length get p = 0 and b = c = 0, which
// makes them the identity.
//
// Few rows do not fill the chip.  Then time is cut into splits: a first pass over the splits computes the state each would leave
// from a zero start, and the sum of its p, since the product of a split's decays is exp(a sum p); a short pass along the splits
// turns these into every split's starting state; the last pass is the ordinary one, started there.  That computes the decays twice, so it is
// taken where it at least triples the CTAs at work.
#pragma once

#include <algorithm>

#include "launch_count.h"
#include "sequence_rows.cuh"

namespace bnb {
namespace scan {

using namespace seq;

constexpr int NS = 4;         // states of a thread
constexpr int KEEP = 8;       // steps from one kept state to the next
constexpr int MIN_SPLIT = 64; // steps

struct Splits {
  int steps;   // of a split, a multiple of 16
  int count;
};
// a power of two of lanes with four states each
inline int lanes_of(int states) {
  int k = 1;
  while (NS * k < states) k *= 2;
  return k;
}
inline Splits splits_of(int steps, int64_t ctas_a_split, int ctas_wanted) {
  int64_t count = std::min<int64_t>(ctas_wanted / std::max<int64_t>(1, ctas_a_split), steps / MIN_SPLIT);
  if (count < 3) return {(steps + 15) / 16 * 16, 1};
  const int len = (int)(((steps + count - 1) / count + 15) / 16 * 16);
  return {len, (steps + len - 1) / len};
}

// Sum over the lanes of a warp that differ in the bits [LO, HI) of their number: NV values a lane go in; afterwards v[0] ..
// v[left - 1] hold the totals of the values from `first` on, left = max(1, NV >> (HI - LO)).  A lane passes on half of its values in
// every round, so that NV values take about NV exchanges and not NV log2(lanes).
template <int NV, int LO, int HI>
__device__ __forceinline__ int sum_lanes(float* v) {
  if constexpr (HI == LO) {
    return 0;
  } else {
    const bool up = (threadIdx.x >> (HI - 1)) & 1;
    if constexpr (NV > 1) {
      constexpr int H = NV / 2;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float mine = up ? v[H + i] : v[i], other = up ? v[i] : v[H + i];
        v[i] = mine + __shfl_xor_sync(0xffffffffu, other, 1 << (HI - 1));
      }
      return (up ? H : 0) + sum_lanes<H, LO, HI - 1>(v);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], 1 << (HI - 1));
      return sum_lanes<1, LO, HI - 1>(v);
    }
  }
}
// Whether this lane is the one to write what sum_lanes left of NV values over these bits (others hold the same).
template <int NV, int LO, int HI>
__device__ __forceinline__ bool writes_sum() {
  int left = HI - LO, halvings = 0;
  for (int n = NV; n > 1 && halvings < left; n /= 2) ++halvings;
  return ((threadIdx.x >> LO) & ((1 << (left - halvings)) - 1)) == 0;
}

// |v| up to 128, from where on e^-|v| is 0 in float32; a NaN stays one.
__device__ __forceinline__ float bounded_size(float v) {
  float m;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(v)), "f"(128.0f));
  return m;
}
// Step sizes of a pair: log(1 + e^v) as max(v, 0) + log(1 + x) with x = e^-|v| <= 1, and log(1 + x) = 2 atanh(s), s = x / (2 + x) <= 1/3, by
// its Taylor series: the first term left out, s^14 / 15, is 1.4e-8 of the sum.  e^-|v| = 2^-m with the rounding of m = |v| log2(e) put
// back to first order.  A few units in the last place, which the gradients of a need: they are long sums.  The size of v is
// bounded first: -inf and a type's lowest value, which mask a step, give the step size 0 and not inf - inf.
__device__ __forceinline__ F2 step_size(F2 v, bool with_softplus) {
  if (!with_softplus) return v;
  const float2 vs = halves(v);
  const F2 mag = f2(bounded_size(vs.x), bounded_size(vs.y)), m = mul(mag, f2(LOG2E));
  const F2 rest = fma(mag, f2(-1.925963033e-8f), fma(mag, f2(-LOG2E), m));   // m - |v| log2(e)
  const float2 ms = halves(m);
  const F2 x0 = f2(ex2_fast(-ms.x), ex2_fast(-ms.y)), x = fma(x0, mul(rest, f2(0.6931471805599453f)), x0);
  const float2 den = halves(add(x, f2(2.0f)));
  const F2 t = mul(x, f2(rcp_fast(den.x), rcp_fast(den.y))), q = mul(t, t);
  F2 series = fma(q, f2(1.0f / 13.0f), f2(1.0f / 11.0f));
  series = fma(q, series, f2(1.0f / 9.0f));
  series = fma(q, series, f2(1.0f / 7.0f));
  series = fma(q, series, f2(1.0f / 5.0f));
  series = fma(q, series, f2(1.0f / 3.0f));
  series = fma(q, series, f2(1.0f));
  return fma(add(t, t), series, f2(fmaxf(vs.x, 0.0f), fmaxf(vs.y, 0.0f)));
}
__device__ __forceinline__ float step_size(float v, bool with_softplus) { return halves(step_size(f2(v), with_softplus)).x; }
template <typename T>
__device__ __forceinline__ F2 sigmoid_pair(F2 v) {
  if constexpr (sizeof(T) == 4) {
    const float2 s = halves(v);
    return f2(sigmoid<float>(s.x), sigmoid<float>(s.y));
  }
  const float2 m = halves(mul(v, f2(-LOG2E))), den = halves(add(f2(ex2_fast(m.x), ex2_fast(m.y)), f2(1.0f)));
  return f2(rcp_fast(den.x), rcp_fast(den.y));
}

// Two neighbouring channels of a step: one access where `paired` says that all are on its boundary, else those of `count` that exist.
template <typename T>
__device__ __forceinline__ Raw<T, 2> load_pair(const T* at, int count, bool paired) {
  if (paired && count == 2) return load_raw<T, 2>(at);
  Raw<T, 2> r;
  T* v = reinterpret_cast<T*>(r.w);
  v[0] = count > 0 ? at[0] : from_f<T>(0.f);
  v[1] = count > 1 ? at[1] : from_f<T>(0.f);
  return r;
}
template <typename T>
__device__ __forceinline__ F2 floats_of(const Raw<T, 2>& r) {
  float f[2];
  unpack<T, 2>(r, f);
  return f2(f[0], f[1]);
}
template <typename T>
__device__ __forceinline__ void store_pair(T* at, F2 v, int count, bool paired) {
  const float2 s = halves(v);
  if (paired && count == 2) {
    const float f[2] = {s.x, s.y};
    store(at, f);
  } else {
    if (count > 0) at[0] = from_f<T>(s.x);
    if (count > 1) at[1] = from_f<T>(s.y);
  }
}
// Whether pairs of channels from an even one on lie on their boundary in a view.
inline bool even_view(const BnbView& v, int element) {
  return reinterpret_cast<uintptr_t>(v.data) % (2 * elem_bytes(element)) == 0 && v.step % 2 == 0 && v.row % 2 == 0;
}

// The four states of a lane, n0 .. n0 + 3, of a (.., states) array that may end inside them.
__device__ __forceinline__ void load_states(float (&h)[NS], const float* at, int n0, int states, bool wide) {
  if (wide) {
    const float4 v = *reinterpret_cast<const float4*>(at + n0);
    h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = n0 + i < states ? at[n0 + i] : 0.f;
  }
}
__device__ __forceinline__ void clear_states(float (&h)[NS]) {
#pragma unroll
  for (int i = 0; i < NS; ++i) h[i] = 0.f;
}
__device__ __forceinline__ void store_states(float* at, const float (&h)[NS], int n0, int states, bool wide) {
  if (wide) {
    *reinterpret_cast<float4*>(at + n0) = make_float4(h[0], h[1], h[2], h[3]);
  } else {
#pragma unroll
    for (int i = 0; i < NS; ++i) if (n0 + i < states) at[n0 + i] = h[i];
  }
}

// A state (or adjoint) behind a split's steps whose decays multiply to 2^m.  No step's decay need be beyond float32 where the product is: zero and
// infinity stay what they are, as they do step by step, and the decay is taken in two halves, whose range holds whatever the result's does.
__device__ __forceinline__ float across(float h, float m) {
  if (h == 0.f || isinf(h)) return h;
  const float half = ex2_fast(0.5f * m);
  return h * half * half;
}

// Starting states of the splits from what each leaves of a zero start: local (count, rows, width, 4 KL) holds that on the way in and the
// starting state on the way out.  REVERSE: the same for the adjoint, from the last split to the first.
//   sum_p (count, rows, width); cut (count, rows): the split does not pass on what it starts with
//   start (rows, width, states) or null; end: where the state behind the last split goes (REVERSE: not wanted)
template <bool REVERSE>
__global__ void __launch_bounds__(256) k_join(float* local, const float* sum_p, const uint8_t* cut, const float* a, const float* start,
                                              int count, int rows, int width, int states, int padded) {
  const int64_t cells = (int64_t)rows * width * padded, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= cells) return;
  const int64_t rc = i / padded;
  const int n = (int)(i - rc * padded), r = (int)(rc / width), c = (int)(rc - (int64_t)r * width);
  const bool real = n < states;
  const float rate = real ? a[(int64_t)c * states + n] * LOG2E : 0.f;
  float run = real && start ? start[rc * states + n] : 0.f;
  constexpr int AT_ONCE = 4;   // splits whose loads are on their way together
  for (int k0 = 0; k0 < count; k0 += AT_ONCE) {
    float left[AT_ONCE], sums[AT_ONCE];
    bool passes[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int64_t s = REVERSE ? max(count - 1 - k0 - k, 0) : min(k0 + k, count - 1);
      left[k] = local[s * cells + i];
      sums[k] = sum_p[s * rows * width + rc];
      passes[k] = !cut[s * rows + r];
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      if (k0 + k >= count) break;
      const int64_t s = REVERSE ? count - 1 - k0 - k : k0 + k;
      local[s * cells + i] = run;
      run = (passes[k] ? across(run, rate * sums[k]) : 0.f) + left[k];
    }
  }
}

int check(const BnbSelectiveScan* a);

}  // namespace scan
}  // namespace bnb
