// The causal depthwise convolution over time with 2 to 4 taps, forward and backward, for sequences and single tokens
// (the conv of griffin.py:96-140 for any width and type, as an operator of its own).
//
//   pre[t] = b + sum_j w[K-1-j] x[t-j],  y = pre or silu(pre);  x[t-j] of an earlier episode counts as 0, before step 0 it is the state
//   dpre = dy act'(pre),  dx[t] = sum_j w[K-1-j] dpre[t+j],  dw[K-1-j] = sum dpre[t] x[t-j],  db = sum dpre
//
// Memory bounds it: x is read and y written once, with about 2 K operations an element in between.  So a thread owns a few
// neighbouring channels of a row (four of them where alignment allows) and walks along time with the window of taps in
// registers; rows are cut into segments of time where there are too few of them to fill the chip, and a segment reads the
// K - 1 steps before it once more.
#include <algorithm>

#include "launch_count.h"
#include "sequence_rows.cuh"

namespace bnb {
namespace {

using namespace seq;

struct Segments {
  int length;   // steps of a segment, a multiple of AHEAD
  int count;
};

constexpr int AHEAD = 4;   // steps whose loads are in flight at once
constexpr int RING = 4;    // the inputs of step t stand in slot t mod 4: no moves, since a group of AHEAD steps goes round it

// The weights of VEC channels, w[j] for lag j, and the bias.
template <int VEC, int K>
__device__ __forceinline__ void parameters(const BnbCausalConv& a, int c, bool in, F2 (&w)[K][PAIRS<VEC>], F2 (&bias)[PAIRS<VEC>]) {
  float v[VEC * K], b[VEC];
#pragma unroll
  for (int i = 0; i < VEC * K; ++i) v[i] = in ? a.weight[(int64_t)c * K + i] : 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) b[i] = in && a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
  for (int i = 0; i < PAIRS<VEC>; ++i) {
    const int x = 2 * i, y = 2 * i + 1 < VEC ? 2 * i + 1 : x;
    bias[i] = f2(b[x], b[y]);
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][i] = f2(v[x * K + K - 1 - j], v[y * K + K - 1 - j]);
  }
}

// The inputs before step t0 into the ring (slots of t0 - 1, t0 - 2, ..: t0 counts as 0) and how many of them are of t0's episode.
template <typename T, int VEC, int K>
__device__ __forceinline__ int window_before(const BnbCausalConv& a, int t0, int r, int c, bool cleared, F2 (&ring)[RING][PAIRS<VEC>]) {
  int valid = 0;
  bool alive = true;
#pragma unroll
  for (int j = 1; j < K; ++j) {
    const int pos = t0 - j;
    F2 (&to)[PAIRS<VEC>] = ring[RING - j];
#pragma unroll
    for (int i = 0; i < PAIRS<VEC>; ++i) to[i] = f2(0.f);
    if (pos >= 0) {
      if (a.done && a.done[(int64_t)pos * a.rows + r]) alive = false;
      if (alive) unpack(*reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.x.data) + pos * a.x.step + r * a.x.row + c), to);
    } else if (alive && a.state_in && !cleared) {
      unpack(*reinterpret_cast<const Pack<float, VEC>*>(a.state_in + ((int64_t)r * (K - 1) + (K - 1 + pos)) * a.width + c), to);
    }
    if (alive) valid = j;
  }
  return valid;
}

// pre of the step whose slot is s
template <int VEC, int K>
__device__ __forceinline__ void convolve(F2 (&pre)[PAIRS<VEC>], const F2 (&ring)[RING][PAIRS<VEC>], const F2 (&w)[K][PAIRS<VEC>], const F2 (&bias)[PAIRS<VEC>], int s) {
#pragma unroll
  for (int i = 0; i < PAIRS<VEC>; ++i) {
    pre[i] = bias[i];
#pragma unroll
    for (int j = K - 1; j >= 0; --j) pre[i] = fma(w[j][i], ring[(s - j + RING) % RING][i], pre[i]);
  }
}
// An episode ended before the step of slot s.  Rare, and the same for a row's threads: worth a branch.
template <int VEC, int K>
__device__ __forceinline__ void forget(F2 (&ring)[RING][PAIRS<VEC>], int s) {
#pragma unroll
  for (int j = 1; j < K; ++j)
#pragma unroll
    for (int i = 0; i < PAIRS<VEC>; ++i) {
      ring[(s - j + RING) % RING][i] = f2(0.f);
      asm volatile("");   // keeps the branch
    }
}

// Units (row, segment) go around the CTAs of a channel tile, so that a thread loads its channels' weights once.
template <typename T, int VEC, int K, bool SILU>
__global__ void __launch_bounds__(256, 3) k_conv(const __grid_constant__ BnbCausalConv a, Segments seg) {
  constexpr int P = PAIRS<VEC>;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  if (c >= a.width) return;
  F2 w[K][P], bias[P];
  parameters<VEC, K>(a, c, true, w, bias);
  const int64_t units = (int64_t)a.rows * seg.count;
  for (int64_t unit = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; unit < units; unit += (int64_t)gridDim.x * blockDim.y) {
    const int s = seg.count == 1 ? 0 : (int)(unit / a.rows), r = (int)(unit - (int64_t)s * a.rows);
    const int n = row_steps(a.lengths, r, a.steps);
    const int t0 = s * seg.length, t1 = min(a.steps, t0 + seg.length), end = min(t1, n);
    T* y = static_cast<T*>(a.y.data) + r * a.y.row + c;
    if (t0 < n || (n == 0 && s == 0)) {
      const T* x = static_cast<const T*>(a.x.data) + r * a.x.row + c;
      F2 ring[RING][P];
#pragma unroll
      for (int i = 0; i < P; ++i) ring[0][i] = f2(0.f);
      window_before<T, VEC, K>(a, t0, r, c, a.reset && a.reset[r], ring);
      for (int t = t0; t < end; t += AHEAD) {
        Pack<T, VEC> raw[AHEAD];
        bool over[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          if (t + k >= end) break;
          raw[k] = *reinterpret_cast<const Pack<T, VEC>*>(x + (t + k) * a.x.step);
          over[k] = a.done && t + k > t0 && a.done[(int64_t)(t + k - 1) * a.rows + r];
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          if (t + k >= end) break;
          if (over[k]) forget<VEC, K>(ring, k);
          unpack(raw[k], ring[k]);
          F2 pre[P];
          convolve<VEC, K>(pre, ring, w, bias, k);
          if (SILU)
#pragma unroll
            for (int i = 0; i < P; ++i) pre[i] = mul(pre[i], sigmoid<T>(pre[i]));
          store<VEC>(y + (t + k) * a.y.step, pre);
        }
      }
      if (n <= t1) {   // the row's last segment: the state is its last taps
#pragma unroll
        for (int q = 0; q < RING; ++q)
          if (((n - t0) & (RING - 1)) == q)
#pragma unroll
            for (int j = 1; j < K; ++j) store<VEC>(a.state_out + ((int64_t)r * (K - 1) + (K - 1 - j)) * a.width + c, ring[(q - j + RING) % RING]);
      }
    }
    F2 zero[P];
#pragma unroll
    for (int i = 0; i < P; ++i) zero[i] = f2(0.f);
    for (int t = max(t0, n); t < t1; ++t) store<VEC>(y + t * a.y.step, zero);
  }
}

struct Plan {
  int bx, by, tiles, blocks;   // channel groups and units of a CTA, channel tiles, CTAs along the units
  Segments seg;
};

// A CTA sums d weight and d bias over its units and leaves them in part (blocks, K + 1, width), so that their order does
// not depend on timing.
template <typename T, int VEC, int K, bool SILU>
__global__ void __launch_bounds__(256, 2) k_conv_bwd(const __grid_constant__ BnbCausalConv a, const __grid_constant__ BnbCausalConvGrads g, Segments seg, float* part) {
  constexpr int P = PAIRS<VEC>;
  extern __shared__ float sums[];   // (by, K + 1, bx * VEC)
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const bool in = c < a.width;
  F2 w[K][P], bias[P], dw[K][P], db[P];
  parameters<VEC, K>(a, c, in, w, bias);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    db[i] = f2(0.f);
#pragma unroll
    for (int j = 0; j < K; ++j) dw[j][i] = f2(0.f);
  }
  const int64_t units = (int64_t)a.rows * seg.count;
  for (int64_t unit = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; in && unit < units; unit += (int64_t)gridDim.x * blockDim.y) {
    const int s = seg.count == 1 ? 0 : (int)(unit / a.rows), r = (int)(unit - (int64_t)s * a.rows);
    const int n = row_steps(a.lengths, r, a.steps);
    const int t0 = s * seg.length, t1 = min(a.steps, t0 + seg.length), own = min(t1, n), end = min(t1 + K - 1, n);
    const T* x = static_cast<const T*>(a.x.data) + r * a.x.row + c;
    const T* dy = static_cast<const T*>(g.dy.data) + r * g.dy.row + c;
    T* dx = static_cast<T*>(g.dx.data) + r * g.dx.row + c;
    float* ds = g.dstate_in ? g.dstate_in + (int64_t)r * (K - 1) * a.width + c : nullptr;
    if (t0 < n || (n == 0 && s == 0)) {
      F2 ring[RING][P], acc[RING][P];   // acc: d x of the step in its slot, so far
#pragma unroll
      for (int j = 0; j < RING; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) acc[j][i] = ring[j][i] = f2(0.f);
      int valid = window_before<T, VEC, K>(a, t0, r, c, false, ring);
      auto emit = [&](int t, const F2 (&v)[P]) {   // the finished gradient of step t, or of the state's tap at t < 0
        if (t >= t0) {
          if (t < t1) store<VEC>(dx + t * g.dx.step, v);
        } else if (t < 0 && s == 0 && ds) {
          store<VEC>(ds + (int64_t)(K - 1 + t) * a.width, v);
        }
      };
      for (int t = t0; t < end; t += AHEAD) {
        Pack<T, VEC> rx[AHEAD], ry[AHEAD];
        bool over[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          if (t + k >= end) break;
          rx[k] = *reinterpret_cast<const Pack<T, VEC>*>(x + (t + k) * a.x.step);
          ry[k] = *reinterpret_cast<const Pack<T, VEC>*>(dy + (t + k) * g.dy.step);
          over[k] = a.done && t + k > t0 && a.done[(int64_t)(t + k - 1) * a.rows + r];
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          if (t + k >= end) break;
          if (t + k > t0) valid = min(valid + 1, K - 1);
          if (over[k]) {
            forget<VEC, K>(ring, k);
            valid = 0;
          }
          unpack(rx[k], ring[k]);
          F2 d[P];
          unpack(ry[k], d);
          if (SILU) {
            F2 pre[P];
            convolve<VEC, K>(pre, ring, w, bias, k);
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const F2 sg = sigmoid<T>(pre[i]);
              d[i] = mul(d[i], mul(sg, fma(pre[i], fma(sg, f2(-1.0f), f2(1.0f)), f2(1.0f))));
            }
          }
          if (t + k < own) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
              db[i] = add(db[i], d[i]);
#pragma unroll
              for (int j = 0; j < K; ++j) dw[j][i] = fma(d[i], ring[(k - j + RING) % RING][i], dw[j][i]);
            }
          }
#pragma unroll
          for (int j = 0; j < K; ++j)
            if (j <= valid) {
#pragma unroll
              for (int i = 0; i < P; ++i) acc[(k - j + RING) % RING][i] = fma(w[j][i], d[i], acc[(k - j + RING) % RING][i]);
            }
          emit(t + k - (K - 1), acc[(k - (K - 1) + RING) % RING]);
#pragma unroll
          for (int i = 0; i < P; ++i) acc[(k - (K - 1) + RING) % RING][i] = f2(0.f);
        }
      }
      if (end == n) {   // the row ends here: its last taps are the state
#pragma unroll
        for (int q = 0; q < RING; ++q)
          if (((n - t0) & (RING - 1)) == q)
#pragma unroll
            for (int j = K - 1; j > 0; --j) {
              F2 (&v)[P] = acc[(q - j + RING) % RING];
              if (g.dstate_out && (j - 1 <= valid || n == 0)) {
                F2 more[P];
                unpack(*reinterpret_cast<const Pack<float, VEC>*>(g.dstate_out + ((int64_t)r * (K - 1) + (K - 1 - j)) * a.width + c), more);
#pragma unroll
                for (int i = 0; i < P; ++i) v[i] = add(v[i], more[i]);
              }
              emit(n - j, v);
            }
      }
    }
    F2 zero[P];
#pragma unroll
    for (int i = 0; i < P; ++i) zero[i] = f2(0.f);
    for (int t = max(t0, n); t < t1; ++t) store<VEC>(dx + t * g.dx.step, zero);
  }
  const int lanes = blockDim.x * VEC;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float* at = sums + (size_t)threadIdx.y * (K + 1) * lanes + threadIdx.x * VEC + i;
    auto half = [&](F2 v) { return i & 1 ? halves(v).y : halves(v).x; };
#pragma unroll
    for (int j = 0; j < K; ++j) at[j * lanes] = half(dw[j][i / 2]);
    at[K * lanes] = half(db[i / 2]);
  }
  __syncthreads();
  for (int e = threadIdx.y * blockDim.x + threadIdx.x; e < (K + 1) * lanes; e += blockDim.x * blockDim.y) {
    const int ch = blockIdx.y * lanes + e % lanes;
    if (ch >= a.width) continue;
    float v = 0.f;
    for (int q = 0; q < (int)blockDim.y; ++q) v += sums[(size_t)q * (K + 1) * lanes + e];
    part[((int64_t)blockIdx.x * (K + 1) + e / lanes) * a.width + ch] = v;
  }
}

// d weight and d bias from the CTAs' sums: 32 warps share the parts of 32 channels of one tap, each in their order, and are added in
// theirs.
__global__ void __launch_bounds__(1024) k_conv_sums(const float* part, int blocks, int width, int taps, float* dweight, float* dbias) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, j = blockIdx.y;
  float v = 0.f;
  if (c < width)
    for (int b = q; b < blocks; b += 32) v += part[((int64_t)b * (taps + 1) + j) * width + c];
  sums[q][lane] = v;
  __syncthreads();
  if (q || c >= width) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) v += sums[k][lane];
  if (j < taps) dweight[(int64_t)c * taps + taps - 1 - j] = v;
  else if (dbias) dbias[c] = v;
}

int check(const BnbCausalConv* a) {
  if (!a) return BNB_ERR_NULL_POINTER;
  if (a->steps < 0 || a->rows < 0 || a->width < 0 || a->element < 0 || a->element > 2 ||
      (a->activation != BNB_ACT_NONE && a->activation != BNB_ACT_SILU)) return BNB_ERR_BAD_ARGUMENT;
  if (a->taps < 2 || a->taps > 4) return BNB_ERR_UNSUPPORTED_DIMS;
  if (a->rows == 0 || a->width == 0) return BNB_OK;
  return !a->weight || (a->steps && !a->x.data) ? BNB_ERR_NULL_POINTER : BNB_OK;
}

// Elements that one access may take: `most` where the width, every stride and every address (of float32 states too) are
// multiples of it, else 1.
int access_width(const BnbCausalConv* a, const BnbCausalConvGrads* g, int most) {
  auto on = [&](const float* p) { return reinterpret_cast<uintptr_t>(p) % (most * 4) == 0; };
  auto fits = [&](const BnbView& v) {
    return reinterpret_cast<uintptr_t>(v.data) % (most * elem_bytes(a->element)) == 0 && v.step % most == 0 && v.row % most == 0;
  };
  bool ok = a->width % most == 0 && fits(a->x) && on(a->state_in);
  ok = ok && (g ? fits(g->dy) && fits(g->dx) && on(g->dstate_in) && on(g->dstate_out) : fits(a->y) && on(a->state_out));
  return ok ? most : 1;
}

// Segments of time such that `threads_a_segment` threads each make about as many threads as the chip holds at half
// occupancy; none shorter than 16 steps, where the three steps read twice are a fifth of the reads.
Segments segments(int steps, int64_t threads_a_segment) {
  const int64_t want = std::max<int64_t>(1, (148 * 1024 + threads_a_segment - 1) / std::max<int64_t>(1, threads_a_segment));
  int length = (int)std::max<int64_t>(16, (steps + want - 1) / want);
  length = (length + AHEAD - 1) / AHEAD * AHEAD;
  int count = std::max(1, (steps + length - 1) / length);
  if (count > 65535) {
    length = (steps + 65534) / 65535;
    count = (steps + length - 1) / length;
  }
  return {length, count};
}

// Channel groups of a CTA: all of a row's in as few equal tiles as 64 threads allow.
int tile_width(int groups) {
  const int tiles = (groups + 63) / 64;
  return (groups + tiles - 1) / tiles;
}

// CTAs: as many as the chip holds at once at `resident` an SM, which then go over the units.
Plan plan(const BnbCausalConv& a, int vec, int resident) {
  Plan p;
  const int groups = (a.width + vec - 1) / vec;
  p.bx = tile_width(groups);
  p.tiles = (groups + p.bx - 1) / p.bx;
  p.seg = segments(a.steps, (int64_t)groups * a.rows);
  const int64_t units = (int64_t)a.rows * p.seg.count;
  p.by = (int)std::max<int64_t>(1, std::min<int64_t>(256 / p.bx, units));
  p.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((units + p.by - 1) / p.by, std::max(1, 148 * resident / p.tiles)));
  return p;
}

// Four elements a thread at most: windows, weights and sums of eight would not stay in registers.
constexpr int FWD_VEC = 4, BWD_VEC = 4, BWD_RESIDENT = 2;

template <typename T, int VEC, int K>
int launch_fwd(const BnbCausalConv& a, cudaStream_t st) {
  const Plan p = plan(a, VEC, 3);
  const dim3 grid(p.blocks, p.tiles), block(p.bx, p.by);
  if (grid.y > 65535) return BNB_ERR_UNSUPPORTED_DIMS;
  count_launch();
  if (a.activation == BNB_ACT_SILU) k_conv<T, VEC, K, true><<<grid, block, 0, st>>>(a, p.seg);
  else k_conv<T, VEC, K, false><<<grid, block, 0, st>>>(a, p.seg);
  return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
}
template <typename T, int VEC>
int fwd_taps(const BnbCausalConv& a, cudaStream_t st) {
  return a.taps == 2 ? launch_fwd<T, VEC, 2>(a, st) : a.taps == 3 ? launch_fwd<T, VEC, 3>(a, st) : launch_fwd<T, VEC, 4>(a, st);
}
template <typename T>
int fwd(const BnbCausalConv& a, cudaStream_t st) {
  return access_width(&a, nullptr, FWD_VEC) > 1 ? fwd_taps<T, FWD_VEC>(a, st) : fwd_taps<T, 1>(a, st);
}

size_t part_bytes(const BnbCausalConv& a, const Plan& p) { return round256((size_t)p.blocks * (a.taps + 1) * a.width * 4); }

template <typename T, int VEC, int K>
int launch_bwd(const BnbCausalConv& a, const BnbCausalConvGrads& g, float* part, cudaStream_t st) {
  const Plan p = plan(a, VEC, BWD_RESIDENT);
  const size_t smem = (size_t)p.by * (K + 1) * p.bx * VEC * 4;   // at most 256 threads x 4 x 5 floats = 20 KB
  const dim3 grid(p.blocks, p.tiles), block(p.bx, p.by);
  count_launch();
  if (a.activation == BNB_ACT_SILU) k_conv_bwd<T, VEC, K, true><<<grid, block, smem, st>>>(a, g, p.seg, part);
  else k_conv_bwd<T, VEC, K, false><<<grid, block, smem, st>>>(a, g, p.seg, part);
  if (cudaGetLastError() != cudaSuccess) return BNB_ERR_LAUNCH;
  count_launch();
  k_conv_sums<<<dim3((a.width + 31) / 32, K + 1), 1024, 0, st>>>(part, p.blocks, a.width, K, g.dweight, g.dbias);
  return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
}
template <typename T, int VEC>
int bwd_taps(const BnbCausalConv& a, const BnbCausalConvGrads& g, float* part, cudaStream_t st) {
  return a.taps == 2 ? launch_bwd<T, VEC, 2>(a, g, part, st)
       : a.taps == 3 ? launch_bwd<T, VEC, 3>(a, g, part, st) : launch_bwd<T, VEC, 4>(a, g, part, st);
}
template <typename T>
int bwd(const BnbCausalConv& a, const BnbCausalConvGrads& g, float* part, cudaStream_t st) {
  return access_width(&a, &g, BWD_VEC) > 1 ? bwd_taps<T, BWD_VEC>(a, g, part, st) : bwd_taps<T, 1>(a, g, part, st);
}

}  // namespace
}  // namespace bnb

using namespace bnb;

extern "C" int bnb_causal_conv_fwd(const BnbCausalConv* a, void* stream) {
  if (const int st = check(a)) return st;
  if (a->rows == 0 || a->width == 0) return BNB_OK;
  if (!a->state_out || (a->steps && !a->y.data)) return BNB_ERR_NULL_POINTER;
  if (a->state_in == a->state_out && a->steps > 1) return BNB_ERR_BAD_ARGUMENT;
  const auto s = static_cast<cudaStream_t>(stream);
  return a->element == BNB_ELEM_F32 ? fwd<float>(*a, s) : a->element == BNB_ELEM_BF16 ? fwd<__nv_bfloat16>(*a, s) : fwd<__half>(*a, s);
}

extern "C" size_t bnb_causal_conv_bwd_scratch_bytes(const BnbCausalConv* a) {
  if (check(a) || a->rows == 0 || a->width == 0) return 0;
  return std::max(part_bytes(*a, plan(*a, 1, BWD_RESIDENT)), part_bytes(*a, plan(*a, BWD_VEC, BWD_RESIDENT)));
}

extern "C" int bnb_causal_conv_bwd(const BnbCausalConv* a, const BnbCausalConvGrads* g, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int st = check(a)) return st;
  if (!g) return BNB_ERR_NULL_POINTER;
  if (a->reset) return BNB_ERR_BAD_ARGUMENT;
  if (a->width == 0) return BNB_OK;
  if (!g->dweight || (a->rows && a->steps && (!g->dy.data || !g->dx.data))) return BNB_ERR_NULL_POINTER;
  const auto s = static_cast<cudaStream_t>(stream);
  if (a->rows == 0) {
    if (cudaMemsetAsync(g->dweight, 0, (size_t)a->width * a->taps * 4, s) != cudaSuccess) return BNB_ERR_LAUNCH;
    return g->dbias && cudaMemsetAsync(g->dbias, 0, (size_t)a->width * 4, s) != cudaSuccess ? BNB_ERR_LAUNCH : BNB_OK;
  }
  if (!scratch || scratch_bytes < bnb_causal_conv_bwd_scratch_bytes(a)) return BNB_ERR_SCRATCH_TOO_SMALL;
  float* part = static_cast<float*>(scratch);
  return a->element == BNB_ELEM_F32 ? bwd<float>(*a, *g, part, s)
       : a->element == BNB_ELEM_BF16 ? bwd<__nv_bfloat16>(*a, *g, part, s) : bwd<__half>(*a, *g, part, s);
}
