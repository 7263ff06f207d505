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
// Slices of up to 64 logits: a thread takes a slice, from a tile of rows in shared memory.  Wider ones: a warp takes a row, and from 1024 logits
// on a CTA.
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
constexpr int WARP_ROW = 1024;              // logits of a row that a warp takes
constexpr int TERMS = 5;                    // w surrogate, w k, w H, w clipped, w
constexpr int MAX_CTAS = SMS * 8;

// The larger of two, NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
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
  template <int N>
  __device__ __forceinline__ void add(const float (&z)[N]) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, z[i]);
    if (top > m) raise(top);
    const float b = base();
#pragma unroll
    for (int i = 0; i < N; ++i) term(z[i], b);
  }
  __device__ __forceinline__ void join(Soft o) {
    const float to = fmaxf(m, o.m);
    if (to > m) raise(to);
    if (to > o.m) o.raise(to);
    s += o.s;
    u += o.u;
  }
  __device__ __forceinline__ float lse() const { return m == -INFINITY ? NAN : m + logf(s); }
  __device__ __forceinline__ float entropy() const { return m == -INFINITY ? NAN : logf(s) - u / s; }
};
__device__ __forceinline__ Soft shuffle(const Soft& v, int by) {
  return {__shfl_xor_sync(0xffffffffu, v.m, by), __shfl_xor_sync(0xffffffffu, v.s, by), __shfl_xor_sync(0xffffffffu, v.u, by)};
}

struct Args {
  BnbPolicyLoss c;
  int width;
  int first[BNB_MAX_SLICES + 1];
  double* part;      // (CTAs, TERMS)
  const float* dloss;
  void* dlogits;
};

__device__ __forceinline__ float weight_of(const BnbPolicyLoss& c, int64_t r) {
  return c.weights ? c.weights[r] : c.mask ? (c.mask[r] ? 1.f : 0.f) : 1.f;
}
// The action of slice s, or -1 for one outside of it.
__device__ __forceinline__ int action_of(const BnbPolicyLoss& c, int64_t r, int s) {
  const int64_t a = c.actions[r * c.n_slices + s];
  return a >= 0 && a < c.sizes[s] ? (int)a : -1;
}
// A row's terms and, where wanted, the loss's slope in l.
struct RowTerms { float surrogate, kl, clipped, slope; };
__device__ __forceinline__ RowTerms row_terms(const BnbPolicyLoss& c, int64_t r, float l) {
  RowTerms v;
  const float a = c.advantages[r], ratio = expf(l - c.old_logprob[r]);
  const float lo = 1.f - c.clip_low, hi = 1.f + c.clip_high, held = ratio < lo ? lo : ratio > hi ? hi : ratio;
  const float free_ = ratio * a, bound = held * a;
  v.surrogate = free_ <= bound ? free_ : bound != bound || free_ == free_ ? bound : free_;   // NaN stays NaN
  v.slope = free_ <= bound ? -free_ : free_ != free_ ? free_ : 0.f;
  v.clipped = ratio < lo || ratio > hi ? 1.f : 0.f;
  v.kl = 0.f;
  if (c.ref_logprob) {
    const float d = c.ref_logprob[r] - l, grown = expm1f(d);
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
// Sums over a CTA's warps, lane 0 of each holding its own, to the CTA's place.
__device__ __forceinline__ void put_sums(const Args& a, Sums s, double (*shared)[TERMS]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < TERMS; ++i)
#pragma unroll
    for (int by = 16; by; by >>= 1) s.v[i] += __shfl_xor_sync(0xffffffffu, s.v[i], by);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < TERMS; ++i) shared[warp][i] = s.v[i];
  __syncthreads();
  if (threadIdx.x < TERMS) {
    double v = 0;
    for (int w = 0; w < warps; ++w) v += shared[w][threadIdx.x];
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

// ------------------------------------------------------------------ narrow slices

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
__global__ void __launch_bounds__(512) k_narrow(const __grid_constant__ Args a, int tile_rows, int pitch, uint32_t per_width) {
  extern __shared__ float tile[];
  __shared__ double sums[16][TERMS];
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
    float* kept = c.kept + HEAD + r * (2 * S + 1);
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
      float l = 0.f, h = 0.f;
      if (w != 0.f) {
        for (int i = 0; i < S; ++i) {
          const float2 v = slice_results[i * tile_rows + tid];
          l += v.x;
          h += v.y;
        }
        s.add(w, row_terms(c, r, l), h);
        kept[2 * S] = l;
      }
      c.logprob[r] = l;
    }
  }
  put_sums(a, s, sums);
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

// T threads a row, of CTAs of THREADS.
template <typename E, int T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_wide(const __grid_constant__ Args a) {
  constexpr int N = 16 / sizeof(E), ROWS = THREADS / T, UNROLL = 4;
  __shared__ double sums[THREADS / 32][TERMS];
  __shared__ Soft joined[THREADS / 32];
  let_next_start();
  wait_for_previous();
  const BnbPolicyLoss& c = a.c;
  const int S = c.n_slices, t = threadIdx.x % T, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Sums sum;
  sum.start();
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / T; r < c.rows; r += (int64_t)gridDim.x * ROWS) {
    const float w = weight_of(c, r);
    if (w == 0.f) {
      if (t == 0) c.logprob[r] = 0.f;
      continue;
    }
    const E* row = static_cast<const E*>(c.logits) + r * c.logits_row;
    float* kept = c.kept + HEAD + r * (2 * S + 1);
    float l = 0.f, h = 0.f;
    for (int s = 0; s < S; ++s) {
      const E* z = row + a.first[s];
      const Span span = span_of(z, c.sizes[s]);
      const E* body = z + span.head;
      Soft v;
      v.start();
      if (t < span.head) v.add_one(to_f(z[t]));
      if (t < span.tail) v.add_one(to_f(body[span.pieces * N + t]));
      int i = t;
      for (; i + (UNROLL - 1) * T < span.pieces; i += UNROLL * T) {
        Raw<E, N> raw[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) raw[k] = load_raw<E, N>(body + (int64_t)(i + k * T) * N);
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
          float f[N];
          unpack<E, N>(raw[k], f);
          v.add(f);
        }
      }
      for (; i < span.pieces; i += T) {
        float f[N];
        load<E, N>(body + (int64_t)i * N, f);
        v.add(f);
      }
#pragma unroll
      for (int by = 16; by; by >>= 1) v.join(shuffle(v, by));
      if constexpr (T > 32) {
        __syncthreads();
        if (lane == 0) joined[warp] = v;
        __syncthreads();
        v = joined[lane % (T / 32)];
#pragma unroll
        for (int by = T / 64; by; by >>= 1) v.join(shuffle(v, by));
      }
      const int at = action_of(c, r, s);
      const float log_s = logf(v.s), hs = v.entropy();
      l += at < 0 || v.m == -INFINITY ? NAN : (to_f(z[at]) - v.m) - log_s;
      h += hs;
      if (t == 0) {
        kept[2 * s] = v.lse();
        kept[2 * s + 1] = hs;
      }
    }
    if (t == 0) {
      sum.add(w, row_terms(c, r, l), h);
      kept[2 * S] = l;
      c.logprob[r] = l;
    }
  }
  __syncthreads();
  put_sums(a, sum, sums);
}

// ------------------------------------------------------------------ backward

// What a row's gradients need: dl, and c2 (c1 with each slice's H).
struct Slope { float dl, c2; };
__device__ __forceinline__ Slope slope_of(const Args& a, int64_t r, float w) {
  const BnbPolicyLoss& c = a.c;
  const float share = a.dloss[0] * (w * c.kept[0]);
  const float l = c.kept[HEAD + r * (2 * c.n_slices + 1) + 2 * c.n_slices];
  return {share * row_terms(c, r, l).slope, share * c.entropy_coef};
}
__device__ __forceinline__ float gradient(float z, float lse, float c1, float c2) {
  const float t = max_nan(z - lse, -1e4f);
  return ex2_fast(t * LOG2E) * fmaf(c2, t, c1);
}

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
    const Slope k = slope_of(a, r, w);
    const float* kept = c.kept + HEAD + r * (2 * S + 1);
    const float lse = kept[2 * s], c1 = fmaf(k.c2, kept[2 * s + 1], -k.dl);
    const int at = action_of(c, r, s);
    const E* z = static_cast<const E*>(c.logits) + r * c.logits_row + a.first[s];
    for (int j = 0; j < n; ++j) to[j] = from_f<E>(gradient(to_f(z[j]), lse, c1, k.c2) + (j == at ? k.dl : 0.f));
  }
}

template <typename E, int T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_wide_bwd(const __grid_constant__ Args a) {
  constexpr int N = 16 / sizeof(E), ROWS = THREADS / T;
  let_next_start();
  wait_for_previous();
  const BnbPolicyLoss& c = a.c;
  const int S = c.n_slices, t = threadIdx.x % T;
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / T; r < c.rows; r += (int64_t)gridDim.x * ROWS) {
    const float w = weight_of(c, r);
    const bool on = w != 0.f;
    const Slope k = on ? slope_of(a, r, w) : Slope{0.f, 0.f};
    const float* kept = c.kept + HEAD + r * (2 * S + 1);
    for (int s = 0; s < S; ++s) {
      const E* z = static_cast<const E*>(c.logits) + r * c.logits_row + a.first[s];
      E* to = static_cast<E*>(a.dlogits) + r * a.width + a.first[s];
      const int n = c.sizes[s], at = on ? action_of(c, r, s) : -1;
      const float lse = on ? kept[2 * s] : 0.f, c1 = on ? fmaf(k.c2, kept[2 * s + 1], -k.dl) : 0.f;
      auto one = [&](int j) { to[j] = on ? from_f<E>(gradient(to_f(z[j]), lse, c1, k.c2) + (j == at ? k.dl : 0.f)) : from_f<E>(0.f); };
      const Span span = span_of(to, n);
      const bool along = (reinterpret_cast<uintptr_t>(z) & 15) == (reinterpret_cast<uintptr_t>(to) & 15);
      if (on && !along) {   // rows that start elsewhere in their 16 bytes than the results
        for (int j = t; j < n; j += T) one(j);
        continue;
      }
      if (t < span.head) one(t);
      if (t < span.tail) one(span.head + span.pieces * N + t);
      for (int i = t; i < span.pieces; i += T) {
        const int j = span.head + i * N;
        float f[N];
        if (on) {
          load<E, N>(z + j, f);
#pragma unroll
          for (int q = 0; q < N; ++q) f[q] = gradient(f[q], lse, c1, k.c2) + (j + q == at ? k.dl : 0.f);
        } else {
#pragma unroll
          for (int q = 0; q < N; ++q) f[q] = 0.f;
        }
        store<E, N>(to + j, f);
      }
    }
  }
}

// ------------------------------------------------------------------ the calls

int check(const BnbPolicyLoss* c) {
  if (!c) return BNB_ERR_NULL_POINTER;
  if (c->rows < 0 || c->element < 0 || c->element > 2) return BNB_ERR_BAD_ARGUMENT;
  if (c->n_slices < 1 || c->n_slices > BNB_MAX_SLICES) return BNB_ERR_UNSUPPORTED_DIMS;
  int64_t width = 0;
  for (int i = 0; i < c->n_slices; ++i) {
    if (c->sizes[i] < 1) return BNB_ERR_UNSUPPORTED_DIMS;
    width += c->sizes[i];
  }
  if (width > 1 << 28 || c->rows > (int64_t)1 << 40) return BNB_ERR_UNSUPPORTED_DIMS;
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

template <typename E>
int forward(Args a, cudaStream_t st) {
  const BnbPolicyLoss& c = a.c;
  int ctas, r;
  if (narrow(c)) {
    const Tile t = tile_of(c.n_slices, a.width);
    const size_t bytes = t.bytes + 8;
    if (bytes > 48 * 1024 && cudaFuncSetAttribute(k_narrow<E>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return BNB_ERR_LAUNCH;
    ctas = ctas_of((c.rows + t.rows - 1) / t.rows, MAX_CTAS);
    r = launch_after(k_narrow<E>, dim3(ctas), t.threads, bytes, st, a, t.rows, t.pitch, (uint32_t)((((uint64_t)1 << 32) + a.width - 1) / a.width));
  } else if (a.width <= WARP_ROW) {
    ctas = ctas_of((c.rows + 7) / 8, MAX_CTAS);
    r = launch_after(k_wide<E, 32, 256>, dim3(ctas), 256, 0, st, a);
  } else {
    ctas = ctas_of(c.rows, MAX_CTAS);
    r = launch_after(k_wide<E, 256, 256>, dim3(ctas), 256, 0, st, a);
  }
  return r ? r : launch_after(k_finish, dim3(1), 32 * TERMS, 0, st, a, ctas);
}
template <typename E>
int backward(const Args& a, cudaStream_t st) {
  const BnbPolicyLoss& c = a.c;
  if (narrow(c)) return launch_after(k_narrow_bwd<E>, dim3(ctas_of((c.rows * c.n_slices + 255) / 256, SMS * 32)), 256, 0, st, a);
  if (a.width <= WARP_ROW) return launch_after(k_wide_bwd<E, 32, 256>, dim3(ctas_of((c.rows + 7) / 8, MAX_CTAS)), 256, 0, st, a);
  return launch_after(k_wide_bwd<E, 256, 256>, dim3(ctas_of(c.rows, MAX_CTAS)), 256, 0, st, a);
}

}  // namespace
}  // namespace policy
}  // namespace bnb

using namespace bnb;
using namespace bnb::policy;

extern "C" size_t bnb_policy_loss_kept_bytes(const BnbPolicyLoss* c) {
  if (!c || c->n_slices < 1 || c->n_slices > BNB_MAX_SLICES || c->rows < 0) return 0;
  return (HEAD + (size_t)c->rows * (2 * c->n_slices + 1)) * 4;
}

extern "C" size_t bnb_policy_loss_scratch_bytes(const BnbPolicyLoss* c) { return c ? (size_t)MAX_CTAS * TERMS * sizeof(double) : 0; }

extern "C" int bnb_policy_loss_fwd(const BnbPolicyLoss* c, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int st = check(c)) return st;
  if (!c->loss || !c->stats || (c->rows && !c->logprob)) return BNB_ERR_NULL_POINTER;
  if (!scratch || scratch_bytes < bnb_policy_loss_scratch_bytes(c)) return BNB_ERR_SCRATCH_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(scratch) & 15) return BNB_ERR_MISALIGNED;
  Args a = args_of(*c);
  a.part = static_cast<double*>(scratch);
  const auto s = static_cast<cudaStream_t>(stream);
  return c->element == BNB_ELEM_F32 ? forward<float>(a, s) : c->element == BNB_ELEM_BF16 ? forward<__nv_bfloat16>(a, s) : forward<__half>(a, s);
}

extern "C" int bnb_policy_loss_bwd(const BnbPolicyLoss* c, const float* dloss, void* dlogits, void* stream) {
  if (const int st = check(c)) return st;
  if (c->rows == 0) return BNB_OK;
  if (!dloss || !dlogits) return BNB_ERR_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(dlogits) & 15) return BNB_ERR_MISALIGNED;
  Args a = args_of(*c);
  a.dloss = dloss;
  a.dlogits = dlogits;
  const auto s = static_cast<cudaStream_t>(stream);
  return c->element == BNB_ELEM_F32 ? backward<float>(a, s) : c->element == BNB_ELEM_BF16 ? backward<__nv_bfloat16>(a, s) : backward<__half>(a, s);
}
