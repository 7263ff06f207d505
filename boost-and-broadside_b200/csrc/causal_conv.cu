// The causal depthwise convolution over time with 2 to 4 taps, forward and backward, for sequences and single tokens
// (the conv of griffin.py:96-140 for any width and type, as an operator of its own).
//
//   pre[t] = b + sum_j w[K-1-j] x[t-j],  y = pre or silu(pre);  x[t-j] of an earlier episode counts as 0, before step 0 it is the state
//   dpre = dy act'(pre),  dx[t] = sum_j w[K-1-j] dpre[t+j],  dw[K-1-j] = sum dpre[t] x[t-j],  db = sum dpre
//
// Memory bounds it: x is read and y written once, with about 2 K operations an element in between.  So a thread owns a few
// neighbouring channels of a row (16 bytes of them where alignment allows) and walks along time with the window of taps in
// registers; rows are cut into segments of time where there are too few of them to fill the chip, and a segment reads the
// K - 1 steps before it once more.
#include <algorithm>

#include "launch_count.h"
#include "sequence_rows.cuh"

namespace bnb {
namespace {

using namespace seq;

struct Segments {
  int length;   // steps of a segment
  int count;
};

// Number of valid taps behind step t0 (0..K-1) and their values, newest first: steps since the last episode end.
template <typename T, int VEC, int K>
__device__ __forceinline__ int window_before(const BnbCausalConv& a, int t0, int r, int c, bool cleared, float (&win)[K][VEC]) {
  int valid = 0;
  bool alive = true;
#pragma unroll
  for (int j = 1; j < K; ++j) {
    const int pos = t0 - j;
#pragma unroll
    for (int i = 0; i < VEC; ++i) win[j][i] = 0.f;
    if (pos >= 0) {
      if (a.done && a.done[(int64_t)pos * a.rows + r]) alive = false;
      if (alive) unpack(*reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.x.data) + pos * a.x.step + r * a.x.row + c), win[j]);
    } else if (alive && a.state_in && !cleared) {
      unpack(*reinterpret_cast<const Pack<float, VEC>*>(a.state_in + ((int64_t)r * (K - 1) + (K - 1 + pos)) * a.width + c), win[j]);
    }
    if (alive) valid = j;
  }
  return valid;
}

constexpr int AHEAD = 4;   // steps whose loads are in flight at once

template <typename T, int VEC, int K, bool SILU>
__global__ void __launch_bounds__(256) k_conv(const __grid_constant__ BnbCausalConv a, Segments seg) {
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const int64_t r64 = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (c >= a.width || r64 >= a.rows) return;
  const int r = (int)r64;
  const int n = row_steps(a.lengths, r, a.steps);
  const int t0 = blockIdx.z * seg.length, t1 = min(a.steps, t0 + seg.length), end = min(t1, n);
  T* y = static_cast<T*>(a.y.data) + r * a.y.row + c;
  if (t0 < n || (n == 0 && t0 == 0)) {
    const T* x = static_cast<const T*>(a.x.data) + r * a.x.row + c;
    float w[K][VEC], bias[VEC], win[K][VEC];   // w[j], win[j]: lag j
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      bias[i] = a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) w[j][i] = a.weight[(int64_t)(c + i) * K + K - 1 - j];
    }
    window_before<T, VEC, K>(a, t0, r, c, a.reset && a.reset[r], win);
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
        unpack(raw[k], win[0]);
        float out[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float pre = bias[i];
#pragma unroll
          for (int j = K - 1; j > 0; --j) {
            if (over[k]) win[j][i] = 0.f;
            pre = fmaf(w[j][i], win[j][i], pre);
          }
          pre = fmaf(w[0][i], win[0][i], pre);
          out[i] = SILU ? pre * sigmoid<T>(pre) : pre;
#pragma unroll
          for (int j = K - 1; j > 0; --j) win[j][i] = win[j - 1][i];
        }
        store(y + (t + k) * a.y.step, out);
      }
    }
    if (n <= t1) {   // the row's last segment
#pragma unroll
      for (int j = 1; j < K; ++j) store(a.state_out + ((int64_t)r * (K - 1) + (K - 1 - j)) * a.width + c, win[j]);
    }
  }
  const float zero[VEC] = {};
  for (int t = max(t0, n); t < t1; ++t) store(y + t * a.y.step, zero);
}

struct BwdPlan {
  int bx, by, tiles, blocks;   // channel groups and units of a CTA, channel tiles, CTAs along the units
  Segments seg;
};

// Units (row, segment) go around the CTAs of a channel tile; a CTA sums d weight and d bias over its own and leaves them in
// part (blocks, K + 1, width), so that their order does not depend on timing.
template <typename T, int VEC, int K, bool SILU>
__global__ void __launch_bounds__(256) k_conv_bwd(const __grid_constant__ BnbCausalConv a, const __grid_constant__ BnbCausalConvGrads g, Segments seg, float* part) {
  extern __shared__ float sums[];   // (by, K + 1, bx * VEC)
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const bool in = c < a.width;
  float w[K][VEC], bias[VEC], dw[K][VEC], db[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    bias[i] = in && a.bias ? a.bias[c + i] : 0.f;
    db[i] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      w[j][i] = in ? a.weight[(int64_t)(c + i) * K + K - 1 - j] : 0.f;
      dw[j][i] = 0.f;
    }
  }
  const int64_t units = (int64_t)a.rows * seg.count;
  for (int64_t unit = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; in && unit < units; unit += (int64_t)gridDim.x * blockDim.y) {
    const int s = (int)(unit / a.rows), r = (int)(unit - (int64_t)s * a.rows);
    const int n = row_steps(a.lengths, r, a.steps);
    const int t0 = s * seg.length, t1 = min(a.steps, t0 + seg.length), own = min(t1, n), end = min(t1 + K - 1, n);
    const T* x = static_cast<const T*>(a.x.data) + r * a.x.row + c;
    const T* dy = static_cast<const T*>(g.dy.data) + r * g.dy.row + c;
    T* dx = static_cast<T*>(g.dx.data) + r * g.dx.row + c;
    float* ds = g.dstate_in ? g.dstate_in + (int64_t)r * (K - 1) * a.width + c : nullptr;
    if (t0 < n || (n == 0 && s == 0)) {
      float win[K][VEC], acc[K][VEC];   // acc[j]: d x[t - j] so far
      int valid = window_before<T, VEC, K>(a, t0, r, c, false, win);
#pragma unroll
      for (int j = 0; j < K; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[j][i] = 0.f;
      auto emit = [&](int t, const float (&v)[VEC]) {   // the finished gradient of step t, or of the state's tap at t < 0
        if (t >= t0) {
          if (t < t1) store(dx + t * g.dx.step, v);
        } else if (t < 0 && s == 0 && ds) {
          store(ds + (int64_t)(K - 1 + t) * a.width, v);
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
          if (t + k > t0) valid = over[k] ? 0 : min(valid + 1, K - 1);
          unpack(rx[k], win[0]);
          float d[VEC];
          unpack(ry[k], d);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float pre = bias[i];
#pragma unroll
            for (int j = K - 1; j > 0; --j) {
              if (over[k]) win[j][i] = 0.f;
              pre = fmaf(w[j][i], win[j][i], pre);
            }
            pre = fmaf(w[0][i], win[0][i], pre);
            if (SILU) {
              const float sg = sigmoid<T>(pre);
              d[i] *= sg * fmaf(pre, 1.f - sg, 1.f);
            }
#pragma unroll
            for (int j = 0; j < K; ++j) {
              if (j <= valid) acc[j][i] = fmaf(w[j][i], d[i], acc[j][i]);
              if (t + k < own) dw[j][i] = fmaf(d[i], win[j][i], dw[j][i]);
            }
            if (t + k < own) db[i] += d[i];
          }
          emit(t + k - (K - 1), acc[K - 1]);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
#pragma unroll
            for (int j = K - 1; j > 0; --j) {
              win[j][i] = win[j - 1][i];
              acc[j][i] = acc[j - 1][i];
            }
            acc[0][i] = 0.f;
          }
        }
      }
      if (end == n) {   // the row ends here: its last taps are the state (acc[j], win[j] now stand for step n - j)
#pragma unroll
        for (int j = K - 1; j > 0; --j) {
          if (g.dstate_out && (j - 1 <= valid || n == 0))
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[j][i] += g.dstate_out[((int64_t)r * (K - 1) + (K - 1 - j)) * a.width + c + i];
          emit(n - j, acc[j]);
        }
      }
    }
    const float zero[VEC] = {};
    for (int t = max(t0, n); t < t1; ++t) store(dx + t * g.dx.step, zero);
  }
  const int lanes = blockDim.x * VEC;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float* at = sums + (size_t)threadIdx.y * (K + 1) * lanes + threadIdx.x * VEC + i;
#pragma unroll
    for (int j = 0; j < K; ++j) at[j * lanes] = dw[j][i];
    at[K * lanes] = db[i];
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

// d weight and d bias from the CTAs' sums: a warp per 32 channels of one tap would leave the chip idle, so eight threads share
// a channel's column and add up in a fixed order.
__global__ void __launch_bounds__(256) k_conv_sums(const float* part, int blocks, int width, int taps, float* dweight, float* dbias) {
  __shared__ float sums[8][33];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, j = blockIdx.y;
  float v = 0.f;
  if (c < width)
    for (int b = q; b < blocks; b += 8) v += part[((int64_t)b * (taps + 1) + j) * width + c];
  sums[q][lane] = v;
  __syncthreads();
  if (q || c >= width) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += sums[k][lane];
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
  ok = ok && (g ? fits(g->dy) && fits(g->dx) && on(g->dstate_in) : fits(a->y) && on(a->state_out));
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

template <typename T, int VEC, int K>
int launch_fwd(const BnbCausalConv& a, cudaStream_t st) {
  const int groups = (a.width + VEC - 1) / VEC, bx = tile_width(groups), by = std::max(1, std::min(256 / bx, a.rows));
  const Segments seg = segments(a.steps, (int64_t)groups * a.rows);
  const dim3 grid((a.rows + by - 1) / by, (groups + bx - 1) / bx, seg.count);
  if (grid.y > 65535) return BNB_ERR_UNSUPPORTED_DIMS;
  count_launch();
  if (a.activation == BNB_ACT_SILU) k_conv<T, VEC, K, true><<<grid, dim3(bx, by), 0, st>>>(a, seg);
  else k_conv<T, VEC, K, false><<<grid, dim3(bx, by), 0, st>>>(a, seg);
  return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
}
template <typename T, int VEC>
int fwd_taps(const BnbCausalConv& a, cudaStream_t st) {
  return a.taps == 2 ? launch_fwd<T, VEC, 2>(a, st) : a.taps == 3 ? launch_fwd<T, VEC, 3>(a, st) : launch_fwd<T, VEC, 4>(a, st);
}
template <typename T>
int fwd(const BnbCausalConv& a, cudaStream_t st) {
  constexpr int MOST = 16 / sizeof(T);
  return access_width(&a, nullptr, MOST) > 1 ? fwd_taps<T, MOST>(a, st) : fwd_taps<T, 1>(a, st);
}

// Four elements a thread at most: windows, weights and sums of eight would not stay in registers.
constexpr int BWD_VEC = 4;
BwdPlan bwd_plan(const BnbCausalConv& a, int vec) {
  BwdPlan p;
  const int groups = (a.width + vec - 1) / vec;
  p.bx = tile_width(groups);
  p.by = std::max(1, 256 / p.bx);
  p.tiles = (groups + p.bx - 1) / p.bx;
  p.seg = segments(a.steps, (int64_t)groups * a.rows);
  const int64_t units = ((int64_t)a.rows * p.seg.count + p.by - 1) / p.by;
  p.blocks = (int)std::max<int64_t>(1, std::min<int64_t>(units, std::max(1, 148 * 4 / p.tiles)));
  return p;
}
size_t part_bytes(const BnbCausalConv& a, const BwdPlan& p) { return round256((size_t)p.blocks * (a.taps + 1) * a.width * 4); }

template <typename T, int VEC, int K>
int launch_bwd(const BnbCausalConv& a, const BnbCausalConvGrads& g, float* part, cudaStream_t st) {
  const BwdPlan p = bwd_plan(a, VEC);
  const size_t smem = (size_t)p.by * (K + 1) * p.bx * VEC * 4;   // at most 256 threads x 4 x 5 floats = 20 KB
  const dim3 grid(p.blocks, p.tiles), block(p.bx, p.by);
  count_launch();
  if (a.activation == BNB_ACT_SILU) k_conv_bwd<T, VEC, K, true><<<grid, block, smem, st>>>(a, g, p.seg, part);
  else k_conv_bwd<T, VEC, K, false><<<grid, block, smem, st>>>(a, g, p.seg, part);
  if (cudaGetLastError() != cudaSuccess) return BNB_ERR_LAUNCH;
  count_launch();
  k_conv_sums<<<dim3((a.width + 31) / 32, K + 1), 256, 0, st>>>(part, p.blocks, a.width, K, g.dweight, g.dbias);
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
  return std::max(part_bytes(*a, bwd_plan(*a, 1)), part_bytes(*a, bwd_plan(*a, BWD_VEC)));
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
