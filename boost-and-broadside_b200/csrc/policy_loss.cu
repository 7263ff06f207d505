// The clipped policy loss of a row's logits (formulas in include/bnb_trunk.h), forward and backward.
//
// A softmax needs its row's maximum and sum: both are carried along one pass over the logits, the sum taken to a new maximum by one
// factor.  The entropy comes from the same pass, u = sum of e^t t with t = z - max:  H = log s - u / s.  The backward needs of a slice only
// lse = max + log s and H:
//
//   p = e^t, t = z - lse;   dz = p (c1 + c2 t) + dl [j is the action],   c2 = g w / W entropy_coef,  c1 = c2 H - dl,
//   dl = g w / W (-A ratio [ratio A <= clip(ratio) A] + kl_coef (1 - e^(ref - l)))
//
// so each pass reads the logits once and the backward writes as much: memory bounds both for wide rows, launches for few.
// A masked logit (-inf, or the type's lowest value, which leaves t = -inf) has e = 0; t is held at -1e4 there, so that e t is 0 and not
// NaN, while NaN passes.  A row's terms are float32, their sums over rows 64 bits: thousands of terms of either sign leave a small mean.
// Sums of CTAs are added in a fixed order by a last launch.
//
// Slices of up to 64 logits: a thread takes a slice, from a tile of rows in shared memory.  Wider ones: 8 to 512 threads take a row.
#include <algorithm>

#include "launch_after.h"
#include "sequence_rows.cuh"

namespace bnb {
namespace policy {
namespace {

using namespace seq;
using tensor::let_next_start;
using tensor::wait_for_previous;

constexpr int SMS = 148, HEAD = 4;          // floats before the rows of `kept`: 1 / W
constexpr int NARROW = 64;                  // logits of a slice that a thread takes
constexpr int TERMS = 5;                    // w surrogate, w k, w H, w clipped, w
constexpr int MAX_CTAS = SMS * 16;

// The larger of two, NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The largest of several pieces; NaN is passed over.
__device__ __forceinline__ uint32_t larger_pair(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t larger_pair(uint32_t a, uint32_t b, __half) {
  const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename E, int N, int B>
__device__ __forceinline__ float top_of(const Raw<E, N> (&raw)[B]) {
  if constexpr (sizeof(E) == 2) {
    uint32_t top = raw[0].w[0];
#pragma unroll
    for (int i = 1; i < 4 * B; ++i) top = larger_pair(top, raw[i / 4].w[i % 4], E{});
    float f[2];
    unpack<E, 2>(Raw<E, 2>{{top}}, f);
    return fmaxf(f[0], f[1]);
  } else {
    float top = __uint_as_float(raw[0].w[0]);
#pragma unroll
    for (int i = 1; i < 4 * B; ++i) top = fmaxf(top, __uint_as_float(raw[i / 4].w[i % 4]));
    return top;
  }
}

// e^t summed, and e^t t, with t = z - m.
struct Soft {
  float m, s, u;
  __device__ __forceinline__ void start() { m = -INFINITY, s = 0.f, u = 0.f; }
  // takes the sums to a maximum that is not below m
  __device__ __forceinline__ void raise(float to) {
    const float d = m == -INFINITY ? 0.f : fmaxf(m - to, -1e4f), f = ex2_fast(d * LOG2E);   // from a type's lowest value up: no 0 times infinity
    u = f * fmaf(d, s, u);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void term(float z, float b) {
    const float t = max_nan(z - b, -1e4f), e = ex2_fast(t * LOG2E);
    s += e;
    u = fmaf(e, t, u);
  }
  __device__ __forceinline__ void add_one(float z) {
    if (z > m) raise(z);
    term(z, base());
  }
  // N values, none above m, two an instruction where there is one; their sums apart until all are there.
  template <int N>
  __device__ __forceinline__ void terms(const float (&z)[N]) {
    const F2 b = f2(-base());
    F2 ss = f2(0.f), us = f2(0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 d = halves(seq::add(f2(z[i], z[i + 1]), b));
      const F2 t = f2(max_nan(d.x, -1e4f), max_nan(d.y, -1e4f));
      const float2 x = halves(mul(t, f2(LOG2E)));
      const F2 e = f2(ex2_fast(x.x), ex2_fast(x.y));
      ss = seq::add(ss, e);
      us = fma(e, t, us);
    }
    const float2 a = halves(ss), c = halves(us);
    s += a.x + a.y;
    u += c.x + c.y;
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&z)[N]) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
    if (top > m) raise(top);
    terms(z);
  }
  // Several pieces together, 16-bit ones compared two an instruction as they lie: one look at the maximum for all of them.
  template <typename E, int N, int B>
  __device__ __forceinline__ void add_pieces(const Raw<E, N> (&raw)[B]) {
    const float top = top_of<E, N, B>(raw);
    if (top > m) raise(top);
#pragma unroll
    for (int k = 0; k < B; ++k) {
      float f[N];
      unpack<E, N>(raw[k], f);
      terms(f);
    }
  }
  __device__ __forceinline__ float lse() const { return m == -INFINITY ? NAN : m + logf(s); }
  __device__ __forceinline__ float entropy() const { return m == -INFINITY ? NAN : logf(s) - u / s; }
};
// The sums of N neighbouring lanes together, in all of them: first to one maximum, so that the sums are plain ones.  ALL: the whole warp holds the
// same N values over and over, and one instruction has their maximum.
template <int N, bool ALL>
__device__ __forceinline__ Soft joined_lanes(Soft v) {
  float top = v.m;
  if constexpr (ALL) {
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(v.m));
  } else {
#pragma unroll
    for (int by = N / 2; by; by >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, by));
  }
  if (top > v.m) v.raise(top);
#pragma unroll
  for (int by = N / 2; by; by >>= 1) {
    v.s += __shfl_xor_sync(0xffffffffu, v.s, by);
    v.u += __shfl_xor_sync(0xffffffffu, v.u, by);
  }
  return v;
}

struct Args {
  BnbPolicyLoss c;
  int width;
  int first[BNB_MAX_SLICES + 1];
  double* part;      // (CTAs, TERMS)
  double* weights;   // sums of weights, n_weights of them; null where there are none
  int n_weights;
  const float* dloss;   // null: 1
  void* dlogits;
  int holds_unit;    // dlogits has the gradient for dloss = 1
};

__device__ __forceinline__ float weight_of(const BnbPolicyLoss& c, int64_t r) {
  return c.weights ? c.weights[r] : c.mask ? (c.mask[r] ? 1.f : 0.f) : 1.f;
}
// The action of slice s, or -1 for one outside of it.
__device__ __forceinline__ int action_of(const BnbPolicyLoss& c, int64_t r, int s) {
  const int64_t a = c.actions[r * c.n_slices + s];
  return a >= 0 && a < c.sizes[s] ? (int)a : -1;
}
// What a row has besides its logits.
struct RowIn { float w, old, advantage, ref; };
__device__ __forceinline__ RowIn row_in(const BnbPolicyLoss& c, int64_t r) {
  return {weight_of(c, r), c.old_logprob[r], c.advantages[r], c.ref_logprob ? c.ref_logprob[r] : 0.f};
}
// How far a row's log-probability is from the old and the reference policy's: from 64 bits, since a rounding of l is many of a difference's.
struct Moved { float old, ref; };   // l - old, ref - l
__device__ __forceinline__ Moved moved(const RowIn& x, double l) { return {(float)(l - x.old), (float)(x.ref - l)}; }
// A row's terms and the loss's slope in l.
struct RowTerms { float surrogate, kl, clipped, slope; };
__device__ __forceinline__ RowTerms row_terms(const BnbPolicyLoss& c, const RowIn& x, Moved by) {
  RowTerms v;
  const float a = x.advantage, ratio = expf(by.old);
  const float lo = 1.f - c.clip_low, hi = 1.f + c.clip_high, held = ratio < lo ? lo : ratio > hi ? hi : ratio;
  const float free_ = ratio * a, bound = held * a;
  v.surrogate = free_ <= bound ? free_ : bound != bound || free_ == free_ ? bound : free_;   // NaN stays NaN
  v.slope = free_ <= bound ? -free_ : free_ != free_ ? free_ : 0.f;
  v.clipped = ratio < lo || ratio > hi ? 1.f : 0.f;
  v.kl = 0.f;
  if (c.ref_logprob) {
    const float d = by.ref, grown = expm1f(d);
    v.kl = grown - d;
    if (c.kl_coef != 0.f) v.slope = fmaf(-c.kl_coef, grown, v.slope);
  }
  return v;
}

struct Sums {
  double v[TERMS];
  __device__ __forceinline__ void start() {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) v[i] = 0;
  }
  __device__ __forceinline__ void add(float w, const RowTerms& t, float h) {
    const double d = w;
    v[0] += d * t.surrogate;
    v[1] += d * t.kl;
    v[2] += d * h;
    v[3] += d * t.clipped;
    v[4] += d;
  }
};
// `parts` sums of a CTA, to the CTA's place.
__device__ __forceinline__ void put_sums(const Args& a, const double (*shared)[TERMS], int parts) {
  __syncthreads();
  if (threadIdx.x < TERMS) {
    double v = 0;
    for (int w = 0; w < parts; ++w) v += shared[w][threadIdx.x];
    a.part[(int64_t)blockIdx.x * TERMS + threadIdx.x] = v;
  }
}

// The sums of all CTAs: loss, means and 1 / W.
__global__ void __launch_bounds__(32 * TERMS) k_finish(const __grid_constant__ Args a, int ctas) {
  __shared__ double total[TERMS];
  const int term = threadIdx.x >> 5, lane = threadIdx.x & 31;
  let_next_start();
  wait_for_previous();
  double v = 0;
#pragma unroll 8
  for (int i = lane; i < ctas; i += 32) v += a.part[(int64_t)i * TERMS + term];
#pragma unroll
  for (int by = 16; by; by >>= 1) v += __shfl_xor_sync(0xffffffffu, v, by);
  if (lane == 0) total[term] = v;
  __syncthreads();
  if (threadIdx.x) return;
  const double by = total[4] != 0 ? 1 / total[4] : 0;
  const double mean[4] = {total[0] * by, total[1] * by, total[2] * by, total[3] * by};
  a.c.loss[0] = (float)(-mean[0] + (a.c.kl_coef != 0.f ? (double)a.c.kl_coef * mean[1] : 0.0) - (double)a.c.entropy_coef * mean[2]);
#pragma unroll
  for (int i = 0; i < 4; ++i) a.c.stats[i] = (float)mean[i];
  a.c.kept[0] = (float)by;
}

// Sums of weights, for a forward that writes gradients: they need 1 / W.
constexpr int WEIGHT_ROWS = 4096;   // of a CTA, at most SMS of them
__global__ void __launch_bounds__(256) k_weights(const __grid_constant__ Args a) {
  __shared__ double sums[8];
  let_next_start();
  wait_for_previous();
  double v = 0;
  for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < a.c.rows; r += (int64_t)gridDim.x * 256) v += weight_of(a.c, r);
#pragma unroll
  for (int by = 16; by; by >>= 1) v += __shfl_xor_sync(0xffffffffu, v, by);
  if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = v;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 8; ++w) v += sums[w];
  a.weights[blockIdx.x] = v;
}
// 1 / W, by every warp for itself.
__device__ __forceinline__ float share_of_rows(const Args& a) {
  double v = 0;
  if (a.weights) {
    for (int i = threadIdx.x & 31; i < a.n_weights; i += 32) v += a.weights[i];
#pragma unroll
    for (int by = 16; by; by >>= 1) v += __shfl_xor_sync(0xffffffffu, v, by);
  } else {
    v = (double)a.c.rows;
  }
  return v != 0 ? (float)(1 / v) : 0.f;
}

// ------------------------------------------------------------------ narrow slices

constexpr int NARROW_WARPS = 16;   // of a CTA, at most
struct Tile { int rows, threads, pitch; size_t bytes; };
// Rows of a tile by how many slices they have; floats in shared memory, rows an odd number of them apart.
Tile tile_of(int slices, int width) {
  Tile t;
  t.rows = slices <= 4 ? 128 : slices <= 8 ? 64 : 32;
  t.threads = t.rows * slices;
  t.pitch = width | 1;
  t.bytes = (size_t)t.rows * t.pitch * 4 + (size_t)t.threads * 8;
  return t;
}
template <typename E>
__global__ void __launch_bounds__(32 * NARROW_WARPS) k_narrow(const __grid_constant__ Args a, int tile_rows, int pitch, uint32_t per_width) {
  extern __shared__ float tile[];
  __shared__ double sums[NARROW_WARPS][TERMS];
  let_next_start();
  wait_for_previous();
  const BnbPolicyLoss& c = a.c;
  const int S = c.n_slices, V = a.width, tid = threadIdx.x, threads = blockDim.x;
  float2* slice_results = reinterpret_cast<float2*>(tile + (size_t)tile_rows * pitch + ((tile_rows * pitch) & 1));   // log-probability, entropy
  const int slice = tid / tile_rows, row = tid - slice * tile_rows;
  const E* logits = static_cast<const E*>(c.logits);
  constexpr int N = 16 / sizeof(E);
  const bool dense = c.logits_row == V && reinterpret_cast<uintptr_t>(logits) % 16 == 0;
  auto row_of = [&](int i) { return V == 1 ? i : (int)__umulhi((uint32_t)i, per_width); };
  Sums s;
  s.start();
  for (int64_t r0 = (int64_t)blockIdx.x * tile_rows; r0 < c.rows; r0 += (int64_t)gridDim.x * tile_rows) {
    const int rows = (int)min((int64_t)tile_rows, c.rows - r0), cells = rows * V;
    __syncthreads();
    int from = 0;
    if (dense) {   // whole pieces of 16 bytes: a tile's first row starts on their boundary
      for (int i = tid * N; i + N <= cells; i += threads * N) {
        float f[N];
        load<E, N>(logits + r0 * V + i, f);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int r = row_of(i + k);
          tile[r * pitch + (i + k - r * V)] = f[k];
        }
      }
      from = cells / N * N;
    }
    for (int i = from + tid; i < cells; i += threads) {
      const int r = row_of(i), j = i - r * V;
      tile[r * pitch + j] = to_f(logits[(r0 + r) * c.logits_row + j]);
    }
    __syncthreads();
    const int64_t r = r0 + row;
    const float w = row < rows ? weight_of(c, r) : 0.f;
    float* kept = c.kept + HEAD + r * (2 * S + 2);
    if (row < rows && w != 0.f) {
      const float* z = tile + row * pitch + a.first[slice];
      const int n = c.sizes[slice];
      Soft v;
      v.start();
      for (int j = 0; j < n; ++j) v.m = fmaxf(v.m, z[j]);
      const float b = v.base();
      for (int j = 0; j < n; ++j) v.term(z[j], b);
      const int at = action_of(c, r, slice);
      const float lse = v.lse(), h = v.entropy();
      kept[2 * slice] = lse;
      kept[2 * slice + 1] = h;
      // z - m first: lse loses digits where the logits are large
      slice_results[tid] = make_float2(at < 0 || v.m == -INFINITY ? NAN : (z[at] - v.m) - logf(v.s), h);
    }
    __syncthreads();
    if (tid < rows) {
      double l = 0;
      float h = 0.f;
      if (w != 0.f) {
        for (int i = 0; i < S; ++i) {
          const float2 v = slice_results[i * tile_rows + tid];
          l += v.x;
          h += v.y;
        }
        const RowIn in = row_in(c, r);
        const Moved by = moved(in, l);
        s.add(w, row_terms(c, in, by), h);
        kept[2 * S] = by.old;
        kept[2 * S + 1] = by.ref;
      }
      c.logprob[r] = (float)l;
    }
  }
#pragma unroll
  for (int i = 0; i < TERMS; ++i)
#pragma unroll
    for (int by = 16; by; by >>= 1) s.v[i] += __shfl_xor_sync(0xffffffffu, s.v[i], by);
  if ((tid & 31) == 0)
#pragma unroll
    for (int i = 0; i < TERMS; ++i) sums[tid >> 5][i] = s.v[i];
  put_sums(a, sums, threads / 32);
}

// ------------------------------------------------------------------ wide slices

// A row of elements from `at` on as a few single ones up to a boundary of 16 bytes, whole pieces and the rest.
struct Span { int head, pieces, tail; };
template <typename E>
__device__ __forceinline__ Span span_of(const E* at, int n) {
  constexpr int N = 16 / sizeof(E);
  Span s;
  s.head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(at) & 15)) & 15) / (int)sizeof(E));
  s.pieces = (n - s.head) / N;
  s.tail = n - s.head - s.pieces * N;
  return s;
}

// What a row's gradients need: dl, and c2 (c1 with each slice's H).
struct Slope { float dl, c2; };
__device__ __forceinline__ Slope slope_of(const BnbPolicyLoss& c, float share, const RowTerms& t) { return {share * t.slope, share * c.entropy_coef}; }
__device__ __forceinline__ float gradient(float z, float lse, float c1, float c2) {
  const float t = max_nan(z - lse, -1e4f);
  return ex2_fast(t * LOG2E) * fmaf(c2, t, c1);
}
// A slice's gradients, T threads along it.  `on`: the row has weight; `at`: the action, or -1.  held: the first HELD pieces of a thread, already in hand.
template <typename E, int T, int HELD>
__device__ __forceinline__ void put_gradients(const E* z, E* to, int n, int t, bool on, int at, float lse, float h, Slope k, const Raw<E, 16 / sizeof(E)>* held) {
  constexpr int N = 16 / sizeof(E);
  const float c1 = on ? fmaf(k.c2, h, -k.dl) : 0.f;
  auto one = [&](int j) { to[j] = on ? from_f<E>(gradient(to_f(z[j]), lse, c1, k.c2) + (j == at ? k.dl : 0.f)) : from_f<E>(0.f); };
  const Span span = span_of(to, n);
  const bool along = (reinterpret_cast<uintptr_t>(z) & 15) == (reinterpret_cast<uintptr_t>(to) & 15);
  if (on && !along) {   // rows that start elsewhere in their 16 bytes than the results
    for (int j = t; j < n; j += T) one(j);
    return;
  }
  if (t < span.head) one(t);
  if (t < span.tail) one(span.head + span.pieces * N + t);
  const F2 by = f2(-lse), c1s = f2(c1), c2s = f2(k.c2);
  auto piece = [&](int i, const Raw<E, N>& raw) {
    const int j = span.head + i * N;
    float f[N];
    unpack<E, N>(raw, f);
#pragma unroll
    for (int q = 0; q < N; q += 2) {
      const float2 d = halves(add(f2(f[q], f[q + 1]), by));
      const F2 v = f2(max_nan(d.x, -1e4f), max_nan(d.y, -1e4f));
      const float2 x = halves(mul(v, f2(LOG2E)));
      const float2 r = halves(mul(f2(ex2_fast(x.x), ex2_fast(x.y)), fma(c2s, v, c1s)));
      f[q] = r.x, f[q + 1] = r.y;
    }
    if ((unsigned)(at - j) < (unsigned)N) {
#pragma unroll
      for (int q = 0; q < N; ++q) f[q] += j + q == at ? k.dl : 0.f;
    }
    store<E, N>(to + j, f);
  };
  if (on) {
    constexpr int UNROLL = 4;
    int i = t;
    if constexpr (HELD > 0) {
#pragma unroll
      for (int q = 0; q < HELD; ++q, i += T)
        if (i < span.pieces) piece(i, held[q]);
    }
    for (; i + (UNROLL - 1) * T < span.pieces; i += UNROLL * T) {
      Raw<E, N> raw[UNROLL];
#pragma unroll
      for (int q = 0; q < UNROLL; ++q) raw[q] = load_raw<E, N>(z + span.head + (int64_t)(i + q * T) * N);
#pragma unroll
      for (int q = 0; q < UNROLL; ++q) piece(i + q * T, raw[q]);
    }
    for (; i < span.pieces; i += T) piece(i, load_raw<E, N>(z + span.head + (int64_t)i * N));
  } else {
    for (int i = t; i < span.pieces; i += T) *reinterpret_cast<uint4*>(to + span.head + (int64_t)i * N) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// T threads a row, of CTAs of THREADS.  GRAD: the gradients for dloss = 1 are written too, from the row's logits once more: the first HELD pieces of
// a thread from its registers, others from L2, so that memory gives and takes every number once.  A row's other numbers are read a row ahead.
template <typename E, int T, int THREADS, bool GRAD>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_wide(const __grid_constant__ Args a) {
  constexpr int N = 16 / sizeof(E), ROWS = THREADS / T, HELD = GRAD && T < 512 ? 4 : 0, UNROLL = 4;   // a row of 512 threads is long: few of its pieces fit
  __shared__ double sums[ROWS][TERMS];
  __shared__ Soft joined[THREADS / 32];
  let_next_start();
  wait_for_previous();
  const BnbPolicyLoss& c = a.c;
  const int S = c.n_slices, t = threadIdx.x % T, group = threadIdx.x / T, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < ROWS * TERMS; i += THREADS) sums[i / TERMS][i % TERMS] = 0;
  __syncthreads();
  const float per_row = GRAD ? share_of_rows(a) : 0.f;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  RowIn next{};
  int next_at = -1;
  auto look = [&](int64_t r) {
    if (r < c.rows) {
      next = row_in(c, r);
      next_at = action_of(c, r, 0);
    }
  };
  look((int64_t)blockIdx.x * ROWS + group);
  for (int64_t first = (int64_t)blockIdx.x * ROWS; first < c.rows; first += step) {
    const int64_t r = first + group;
    const RowIn in = next;
    int at = next_at;
    look(r + step);
    const bool there = r < c.rows, on = there && in.w != 0.f;   // of all threads of a row
    const E* row = static_cast<const E*>(c.logits) + (there ? r : 0) * c.logits_row;
    E* const to = static_cast<E*>(a.dlogits) + (there ? r : 0) * a.width;
    float* kept = c.kept + HEAD + r * (2 * S + 2);
    double l = 0;
    float h = 0.f, lse = 0.f, hs = 0.f;
    Raw<E, N> held[HELD > 0 ? HELD : 1];
    for (int s = 0; s < S; ++s) {
      const E* z = row + a.first[s];
      const Span span = span_of(z, on ? c.sizes[s] : 0);
      const E* body = z + span.head;
      if (s && on) at = action_of(c, r, s);
      const float taken = on && at >= 0 ? to_f(z[at]) : 0.f;
      Soft v;
      v.start();
      int i = t;
#pragma unroll
      for (int k = 0; k < HELD; ++k)
        if (i + k * T < span.pieces) held[k] = load_raw<E, N>(body + (int64_t)(i + k * T) * N);
      if (t < span.head) v.add_one(to_f(z[t]));
      if (t < span.tail) v.add_one(to_f(body[span.pieces * N + t]));
      if (HELD > 0 && span.pieces >= HELD * T) {
        if constexpr (HELD > 0) v.template add_pieces<E, N, HELD>(held);
        i += HELD * T;
      } else {
#pragma unroll
        for (int k = 0; k < HELD; ++k, i += T)
          if (i < span.pieces) {
            float f[N];
            unpack<E, N>(held[k], f);
            v.add(f);
          }
      }
      for (; i + (UNROLL - 1) * T < span.pieces; i += UNROLL * T) {
        Raw<E, N> raw[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) raw[k] = load_raw<E, N>(body + (int64_t)(i + k * T) * N);
        v.template add_pieces<E, N, UNROLL>(raw);
      }
      for (; i < span.pieces; i += T) {
        float f[N];
        load<E, N>(body + (int64_t)i * N, f);
        v.add(f);
      }
      if constexpr (T < 32) __syncwarp();
      v = joined_lanes<(T < 32 ? T : 32), (T >= 32)>(v);
      if constexpr (T > 32) {
        __syncthreads();
        if (lane == 0) joined[warp] = v;
        __syncthreads();
        v = joined_lanes<T / 32, true>(joined[lane % (T / 32)]);
      }
      const float log_s = logf(v.s);
      hs = v.entropy();
      lse = v.lse();
      l += at < 0 || v.m == -INFINITY ? NAN : (taken - v.m) - log_s;
      h += hs;
      if (t == 0 && on) {
        kept[2 * s] = lse;
        kept[2 * s + 1] = hs;
      }
    }
    RowTerms terms{};
    const Moved by = moved(in, l);
    if (on && (GRAD || t == 0)) terms = row_terms(c, in, by);
    if (t == 0 && there) {
      if (on) {
        Sums sum = *reinterpret_cast<const Sums*>(sums[group]);   // its row's, in shared memory: no other thread needs the registers
        sum.add(in.w, terms, h);
        *reinterpret_cast<Sums*>(sums[group]) = sum;
        kept[2 * S] = by.old;
        kept[2 * S + 1] = by.ref;
      }
      c.logprob[r] = on ? (float)l : 0.f;
    }
    if constexpr (GRAD) {
      const Slope k = slope_of(c, in.w * per_row, terms);
      if (S == 1 || !on) {
        if (there) put_gradients<E, T, HELD>(on ? row : to, to, a.width, t, on, at, lse, hs, k, held);
      }
      if (S > 1) {
        if constexpr (T > 32) __syncthreads();   // what thread 0 kept of the slices
        else __syncwarp();
        if (on)
          for (int s = 0; s < S; ++s)
            put_gradients<E, T, 0>(row + a.first[s], to + a.first[s], c.sizes[s], t, true, action_of(c, r, s), kept[2 * s], kept[2 * s + 1], k, nullptr);
      }
    }
    if constexpr (T < 32) __syncwarp();
  }
  put_sums(a, sums, ROWS);
}

// ------------------------------------------------------------------ backward

template <typename E>
__global__ void __launch_bounds__(256) k_narrow_bwd(const __grid_constant__ Args a) {
  let_next_start();
  wait_for_previous();
  const BnbPolicyLoss& c = a.c;
  const int S = c.n_slices, V = a.width;
  E* out = static_cast<E*>(a.dlogits);
  // a thread a slice
  const int64_t total = c.rows * S;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / S;
    const int s = (int)(i - r * S), n = c.sizes[s];
    const float w = weight_of(c, r);
    E* to = out + r * V + a.first[s];
    if (w == 0.f) {
      for (int j = 0; j < n; ++j) to[j] = from_f<E>(0.f);
      continue;
    }
    const float* kept = c.kept + HEAD + r * (2 * S + 2);
    const Slope k = slope_of(c, a.dloss[0] * (w * c.kept[0]), row_terms(c, row_in(c, r), {kept[2 * S], kept[2 * S + 1]}));
    const float lse = kept[2 * s], c1 = fmaf(k.c2, kept[2 * s + 1], -k.dl);
    const int at = action_of(c, r, s);
    const E* z = static_cast<const E*>(c.logits) + r * c.logits_row + a.first[s];
    for (int j = 0; j < n; ++j) to[j] = from_f<E>(gradient(to_f(z[j]), lse, c1, k.c2) + (j == at ? k.dl : 0.f));
  }
}

template <typename E, int T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_wide_bwd(const __grid_constant__ Args a) {
  constexpr int ROWS = THREADS / T;
  let_next_start();
  wait_for_previous();
  const BnbPolicyLoss& c = a.c;
  const int S = c.n_slices, t = threadIdx.x % T;
  const float dloss = a.dloss[0];
  if (a.holds_unit && dloss == 1.f) return;
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / T; r < c.rows; r += (int64_t)gridDim.x * ROWS) {
    const float w = weight_of(c, r);
    const bool on = w != 0.f;
    const float* kept = c.kept + HEAD + r * (2 * S + 2);
    const Slope k = on ? slope_of(c, dloss * (w * c.kept[0]), row_terms(c, row_in(c, r), {kept[2 * S], kept[2 * S + 1]})) : Slope{0.f, 0.f};
    for (int s = 0; s < S; ++s)
      put_gradients<E, T, 0>(static_cast<const E*>(c.logits) + r * c.logits_row + a.first[s], static_cast<E*>(a.dlogits) + r * a.width + a.first[s], c.sizes[s], t, on,
                             on ? action_of(c, r, s) : -1, on ? kept[2 * s] : 0.f, on ? kept[2 * s + 1] : 0.f, k, nullptr);
  }
}

// ------------------------------------------------------------------ the calls

int check_slices(const BnbPolicyLoss* c) {
  if (c->n_slices < 1 || c->n_slices > BNB_MAX_SLICES) return BNB_ERR_UNSUPPORTED_DIMS;
  int64_t width = 0;
  for (int i = 0; i < c->n_slices; ++i) {
    if (c->sizes[i] < 1) return BNB_ERR_UNSUPPORTED_DIMS;
    width += c->sizes[i];
  }
  return width > 1 << 28 ? BNB_ERR_UNSUPPORTED_DIMS : BNB_OK;
}
int check(const BnbPolicyLoss* c) {
  if (!c) return BNB_ERR_NULL_POINTER;
  if (c->rows < 0 || c->element < 0 || c->element > 2) return BNB_ERR_BAD_ARGUMENT;
  if (const int st = check_slices(c)) return st;
  if (c->rows > (int64_t)1 << 40) return BNB_ERR_UNSUPPORTED_DIMS;
  if (c->weights && c->mask) return BNB_ERR_BAD_ARGUMENT;
  if (!(c->clip_low >= 0.f) || !(c->clip_high >= 0.f)) return BNB_ERR_BAD_ARGUMENT;
  if (c->rows && (!c->logits || !c->actions || !c->old_logprob || !c->advantages)) return BNB_ERR_NULL_POINTER;
  if (!c->kept) return BNB_ERR_NULL_POINTER;
  return BNB_OK;
}
Args args_of(const BnbPolicyLoss& c) {
  Args a{};
  a.c = c;
  for (int i = 0; i < c.n_slices; ++i) a.first[i + 1] = a.first[i] + c.sizes[i];
  a.width = a.first[c.n_slices];
  return a;
}
bool narrow(const BnbPolicyLoss& c) { return *std::max_element(c.sizes, c.sizes + c.n_slices) <= NARROW; }
int ctas_of(int64_t units, int most) { return (int)std::max<int64_t>(1, std::min<int64_t>(units, most)); }

// Threads of a row: some 8 to 16 pieces of 16 bytes each, so that what a row takes besides, a chain of some 2 us, is shared by few and many rows are at
// work.  Forward with gradients of 134 M bfloat16 logits (268 MB each way), us by width: 32768 with 256 threads 135 (512: 160), 16384
// with 128 135 (256: 148), 8192 with 64 138 (128: 145, 256: 195), 4096 with 64 149 (32: 171), 2048 with 32 169 (256: 520);
// since then, with one maximum for four pieces, 118, 120, 123 and, 2048 wide, 137.
template <typename E, int T, int THREADS, bool GRAD>
int launch_wide(const Args& a, int& ctas, cudaStream_t st) {
  ctas = ctas_of((a.c.rows + THREADS / T - 1) / (THREADS / T), MAX_CTAS);   // more than there is room for: rows without weight take less
  return launch_after(k_wide<E, T, THREADS, GRAD>, dim3(ctas), THREADS, 0, st, a);
}
template <typename E, bool GRAD>
int wide(const Args& a, int& ctas, cudaStream_t st) {
  const int64_t bytes = (int64_t)a.width * sizeof(E);
  if (bytes <= 1024) return launch_wide<E, 8, 256, GRAD>(a, ctas, st);
  if (bytes <= 2048) return launch_wide<E, 16, 256, GRAD>(a, ctas, st);
  if (bytes <= 4096) return launch_wide<E, 32, 256, GRAD>(a, ctas, st);
  if (bytes <= 16384) return launch_wide<E, 64, 64, GRAD>(a, ctas, st);
  if (bytes <= 32768) return launch_wide<E, 128, 128, GRAD>(a, ctas, st);
  if (bytes <= 131072) return launch_wide<E, 256, 256, GRAD>(a, ctas, st);
  return launch_wide<E, 512, 512, GRAD>(a, ctas, st);
}

template <typename E>
int forward(Args a, cudaStream_t st) {
  const BnbPolicyLoss& c = a.c;
  int ctas, r;
  if (narrow(c)) {
    const Tile t = tile_of(c.n_slices, a.width);
    const size_t bytes = t.bytes + 8;
    if (bytes + NARROW_WARPS * TERMS * sizeof(double) > 48 * 1024 && cudaFuncSetAttribute(k_narrow<E>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return BNB_ERR_LAUNCH;
    ctas = ctas_of((c.rows + t.rows - 1) / t.rows, MAX_CTAS);
    r = launch_after(k_narrow<E>, dim3(ctas), t.threads, bytes, st, a, t.rows, t.pitch, (uint32_t)((((uint64_t)1 << 32) + a.width - 1) / a.width));
  } else {
    const bool grad = a.dlogits != nullptr;
    if (grad && a.weights) {
      a.n_weights = ctas_of((c.rows + WEIGHT_ROWS - 1) / WEIGHT_ROWS, SMS);
      if (r = launch_after(k_weights, dim3(a.n_weights), 256, 0, st, a); r) return r;
    }
    r = grad ? wide<E, true>(a, ctas, st) : wide<E, false>(a, ctas, st);
  }
  return r ? r : launch_after(k_finish, dim3(1), 32 * TERMS, 0, st, a, ctas);
}
template <typename E>
int backward(const Args& a, cudaStream_t st) {
  const BnbPolicyLoss& c = a.c;
  if (narrow(c)) return launch_after(k_narrow_bwd<E>, dim3(ctas_of((c.rows * c.n_slices + 255) / 256, SMS * 32)), 256, 0, st, a);
  const int64_t bytes = (int64_t)a.width * sizeof(E);
  if (bytes <= 1024) return launch_after(k_wide_bwd<E, 8, 256>, dim3(ctas_of((c.rows + 31) / 32, SMS * 8)), 256, 0, st, a);
  if (bytes <= 4096) return launch_after(k_wide_bwd<E, 32, 256>, dim3(ctas_of((c.rows + 7) / 8, SMS * 8)), 256, 0, st, a);
  if (bytes <= 16384) return launch_after(k_wide_bwd<E, 64, 64>, dim3(ctas_of(c.rows, SMS * 32)), 64, 0, st, a);
  return launch_after(k_wide_bwd<E, 256, 256>, dim3(ctas_of(c.rows, SMS * 4)), 256, 0, st, a);
}

}  // namespace
}  // namespace policy
}  // namespace bnb

using namespace bnb;
using namespace bnb::policy;

extern "C" size_t bnb_policy_loss_kept_bytes(const BnbPolicyLoss* c) {
  if (!c || c->n_slices < 1 || c->n_slices > BNB_MAX_SLICES || c->rows < 0) return 0;
  return (HEAD + (size_t)c->rows * (2 * c->n_slices + 2)) * 4;
}

extern "C" size_t bnb_policy_loss_scratch_bytes(const BnbPolicyLoss* c) { return c ? (size_t)(MAX_CTAS * TERMS + SMS) * sizeof(double) : 0; }

extern "C" int bnb_policy_loss_takes_gradients(const BnbPolicyLoss* c) { return c && !check_slices(c) && c->element != BNB_ELEM_F16 && !narrow(*c) ? 1 : 0; }

extern "C" int bnb_policy_loss_fwd(const BnbPolicyLoss* c, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int st = check(c)) return st;
  if (!c->loss || !c->stats || (c->rows && !c->logprob)) return BNB_ERR_NULL_POINTER;
  if (!scratch || scratch_bytes < bnb_policy_loss_scratch_bytes(c)) return BNB_ERR_SCRATCH_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(scratch) & 15) return BNB_ERR_MISALIGNED;
  Args a = args_of(*c);
  a.part = static_cast<double*>(scratch);
  if (c->weights || c->mask) a.weights = a.part + MAX_CTAS * TERMS;
  if (c->dlogits) {
    if (!bnb_policy_loss_takes_gradients(c)) return BNB_ERR_BAD_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(c->dlogits) & 15) return BNB_ERR_MISALIGNED;
    a.dlogits = c->dlogits;
  }
  const auto s = static_cast<cudaStream_t>(stream);
  return c->element == BNB_ELEM_F32 ? forward<float>(a, s) : c->element == BNB_ELEM_BF16 ? forward<__nv_bfloat16>(a, s) : forward<__half>(a, s);
}

extern "C" int bnb_policy_loss_bwd(const BnbPolicyLoss* c, const float* dloss, void* dlogits, int holds_unit, void* stream) {
  if (const int st = check(c)) return st;
  if (c->rows == 0) return BNB_OK;
  if (!dloss || !dlogits) return BNB_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(dlogits) & 15) return BNB_ERR_MISALIGNED;
  Args a = args_of(*c);
  a.dloss = dloss;
  a.dlogits = dlogits;
  a.holds_unit = holds_unit && bnb_policy_loss_takes_gradients(c);
  const auto s = static_cast<cudaStream_t>(stream);
  return c->element == BNB_ELEM_F32 ? backward<float>(a, s) : c->element == BNB_ELEM_BF16 ? backward<__nv_bfloat16>(a, s) : backward<__half>(a, s);
}
