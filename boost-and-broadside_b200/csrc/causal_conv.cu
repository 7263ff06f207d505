// The causal depthwise convolution over time with 2 to 4 taps, forward and backward, for sequences and single tokens
// (the conv of griffin.py:96-140 for any width and type, as an operator of its own).
//
//   pre[t] = b + sum_j w[K-1-j] x[t-j],  y = pre or silu(pre);  x[t-j] of an earlier episode counts as 0, before step 0 it is the state
//   dpre = dy act'(pre),  dx[t] = sum_j w[K-1-j] dpre[t+j],  dw[K-1-j] = sum dpre[t] x[t-j],  db = sum dpre
//
// x is read and y written once, so memory is what it could be bound by: 319 MB forward and 478 backward at 32 x 8192 x 256 of bfloat16.
// What it spends beside that are instructions, some 29 a thread and element forward and 63 backward (SiLU and its slope, the taps,
// unpacking), so that neither is full: issue slots 55 and 53 %, DRAM 36 and 25 %.  A thread takes a few neighbouring channels of a
// span of steps of a row, all of whose loads are on their way at once, and goes over them with the taps in registers; the K - 1 steps before (and behind,
// for gradients) are read by the neighbour too, and come from the caches.  Threads that walked along a whole row had a third of the loads in
// flight: 121 us forward and 301 backward, now 91 and 218.
#include <algorithm>

#include "launch_count.h"
#include "sequence_rows.cuh"

namespace bnb {
namespace {

using namespace seq;

constexpr int FWD_SPAN = 8, BWD_SPAN = 16;   // steps of a unit

// The weights of VEC channels, w[j] for lag j, and the bias.
template <int VEC, int K>
__device__ __forceinline__ void parameters(const BnbCausalConv& a, int c, bool in, float (&w)[K][VEC], float (&bias)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    bias[i] = in && a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][i] = in ? a.weight[(int64_t)(c + i) * K + K - 1 - j] : 0.f;
  }
}

template <int N>
__device__ __forceinline__ void clear(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
}

// The inputs before step t0, lag[j] that of step t0 - j, and how many of them are of t0's episode, or of step t0 - 1's (`behind`: the
// taps behind a row's last step).
template <typename T, int VEC, int K>
__device__ __forceinline__ int taps_before(const BnbCausalConv& a, int t0, int r, int c, bool cleared, bool behind, float (&lag)[K][VEC]) {
  int valid = 0;
  bool alive = true;
#pragma unroll
  for (int j = 1; j < K; ++j) {
    const int pos = t0 - j;
    clear(lag[j]);
    if (pos >= 0) {
      if (a.done && !(behind && j == 1) && a.done[(int64_t)pos * a.rows + r]) alive = false;
      if (alive) load(static_cast<const T*>(a.x.data) + pos * a.x.step + r * a.x.row + c, lag[j]);
    } else if (alive && a.state_in && !cleared) {
      load(a.state_in + ((int64_t)r * (K - 1) + (K - 1 + pos)) * a.width + c, lag[j]);
    }
    if (alive) valid = j;
  }
  return valid;
}
// Bit k: an episode ended between steps t0 + k - 1 and t0 + k, for k < N and steps before `end`.
template <int N>
__device__ __forceinline__ unsigned ends(const BnbCausalConv& a, int t0, int end, int r) {
  unsigned over = 0;
  if (a.done) {
    const uint8_t* d = a.done + (int64_t)t0 * a.rows + r;
#pragma unroll
    for (int k = 1; k < N; ++k, d += a.rows)
      if (t0 + k < end && *d) over |= 1u << k;
  }
  return over;
}
// pre of a step: in[j] the input j steps before it
template <int VEC, int K, class In>
__device__ __forceinline__ void convolve(float (&pre)[VEC], const float (&w)[K][VEC], const float (&bias)[VEC], In in) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    pre[i] = bias[i];
#pragma unroll
    for (int j = K - 1; j >= 0; --j) pre[i] = fmaf(w[j][i], in(j)[i], pre[i]);
  }
}

// Units, a row's next to one another, go around the CTAs of a channel tile, so that a thread loads its channels' weights once.
template <typename T, int VEC, int K, bool SILU>
__global__ void __launch_bounds__(256, 4) k_conv(const __grid_constant__ BnbCausalConv a, unsigned units, unsigned spans) {
  constexpr int SPAN = FWD_SPAN;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  if (c >= a.width) return;
  float w[K][VEC], bias[VEC];
  parameters<VEC, K>(a, c, true, w, bias);
  auto act = [](float (&v)[VEC]) {
    if (SILU)
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] *= sigmoid<T>(v[i]);
  };
  for (unsigned unit = blockIdx.x * blockDim.y + threadIdx.y; unit < units; unit += gridDim.x * blockDim.y) {
    const int r = (int)(unit / spans), s = (int)(unit - r * spans);
    const int n = row_steps(a.lengths, r, a.steps);
    const int t0 = s * SPAN, t1 = min(a.steps, t0 + SPAN), end = min(t1, n);
    const bool cleared = a.reset && a.reset[r];
    const T* x = static_cast<const T*>(a.x.data) + r * a.x.row + c + t0 * a.x.step;
    T* y = static_cast<T*>(a.y.data) + r * a.y.row + c + t0 * a.y.step;
    float lag[K][VEC];
    if (t0 + SPAN <= n) {
      Raw<T, VEC> raw[SPAN];
#pragma unroll
      for (int k = 0; k < SPAN; ++k) raw[k] = load_raw<T, VEC>(x + k * a.x.step);
      const unsigned over = ends<SPAN>(a, t0, end, r);
      taps_before<T, VEC, K>(a, t0, r, c, cleared, false, lag);
      float ring[4][VEC];   // the input of step t0 + k in slot k mod 4
      clear(ring[0]);
#pragma unroll
      for (int j = 1; j < K; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) ring[4 - j][i] = lag[j][i];
#pragma unroll
      for (int k = 0; k < SPAN; ++k) {
        if ((over >> k) & 1) {   // rare, and the same for a row's threads: worth a branch
#pragma unroll
          for (int j = 1; j < K; ++j) clear(ring[(k + 4 - j) % 4]);
          asm volatile("");
        }
        unpack<T, VEC>(raw[k], ring[k % 4]);
        float pre[VEC];
        convolve<VEC, K>(pre, w, bias, [&](int j) -> const float (&)[VEC] { return ring[(k + 4 - j) % 4]; });
        act(pre);
        store(y + k * a.y.step, pre);
      }
    } else if (t0 < n) {   // a row's last steps
      taps_before<T, VEC, K>(a, t0, r, c, cleared, false, lag);
#pragma unroll 1
      for (int t = t0; t < end; ++t, x += a.x.step, y += a.y.step) {
        if (a.done && t > t0 && a.done[(int64_t)(t - 1) * a.rows + r]) {
#pragma unroll
          for (int j = 1; j < K; ++j) clear(lag[j]);
        }
        load(x, lag[0]);
        float pre[VEC];
        convolve<VEC, K>(pre, w, bias, [&](int j) -> const float (&)[VEC] { return lag[j]; });
        act(pre);
        store(y, pre);
#pragma unroll
        for (int j = K - 1; j > 0; --j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) lag[j][i] = lag[j - 1][i];
      }
    }
    if (n <= t1 && (t0 < n || s == 0)) {   // the row's last unit: the state is its last taps
      taps_before<T, VEC, K>(a, n, r, c, cleared, true, lag);
#pragma unroll
      for (int j = 1; j < K; ++j) store(a.state_out + ((int64_t)r * (K - 1) + (K - 1 - j)) * a.width + c, lag[j]);
    }
    clear(lag[0]);
    y = static_cast<T*>(a.y.data) + r * a.y.row + c;
    for (int t = max(t0, n); t < t1; ++t) store(y + t * a.y.step, lag[0]);
  }
}

struct Plan {
  int bx, by, tiles, blocks;   // channel groups and units of a CTA, channel tiles, CTAs along the units
  unsigned units, spans;       // of all rows, of a row
};

// A unit computes the gradients of its own steps' inputs, for which it looks at the K - 1 steps behind them too; d weight and d bias it sums over
// its own steps.  A CTA leaves those sums in part (blocks, K + 1, width), so that their order does not depend on timing.
template <typename T, int VEC, int K, bool SILU>
__global__ void __launch_bounds__(256, 2) k_conv_bwd(const __grid_constant__ BnbCausalConv a, const __grid_constant__ BnbCausalConvGrads g, unsigned units, unsigned spans, float* part) {
  constexpr int SPAN = BWD_SPAN;
  extern __shared__ float sums[];   // (by, K + 1, bx * VEC)
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const bool in = c < a.width;
  float w[K][VEC], bias[VEC], dw[K][VEC], db[VEC];
  parameters<VEC, K>(a, c, in, w, bias);
  clear(db);
#pragma unroll
  for (int j = 0; j < K; ++j) clear(dw[j]);
  // d pre from d y
  auto through_act = [](float (&d)[VEC], const float (&pre)[VEC]) {
    if (SILU)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float sg = sigmoid<T>(pre[i]);
        d[i] *= sg * fmaf(pre[i], 1.f - sg, 1.f);
      }
  };
  for (unsigned unit = blockIdx.x * blockDim.y + threadIdx.y; in && unit < units; unit += gridDim.x * blockDim.y) {
    const int r = (int)(unit / spans), s = (int)(unit - r * spans);
    const int n = row_steps(a.lengths, r, a.steps);
    const int t0 = s * SPAN, t1 = min(a.steps, t0 + SPAN);
    const T* x = static_cast<const T*>(a.x.data) + r * a.x.row + c + t0 * a.x.step;
    const T* dy = static_cast<const T*>(g.dy.data) + r * g.dy.row + c + t0 * g.dy.step;
    T* dx = static_cast<T*>(g.dx.data) + r * g.dx.row + c;
    float* ds = g.dstate_in ? g.dstate_in + (int64_t)r * (K - 1) * a.width + c : nullptr;
    // the finished gradient of step t, or of the state's tap at t < 0; the last taps of the row are the state that comes out, of
    // whose entries those of the last step's episode count (`valid` taps before it)
    auto emit = [&](int t, float (&v)[VEC], int valid) {
      if (g.dstate_out && t >= n - (K - 1) && t < n && (n == 0 || n - 1 - t <= valid)) {
        float more[VEC];
        load(g.dstate_out + ((int64_t)r * (K - 1) + (t - (n - (K - 1)))) * a.width + c, more);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] += more[i];
      }
      if (t >= t0) {
        if (t < min(t1, n)) store(dx + t * g.dx.step, v);
      } else if (t < 0 && s == 0 && ds) {
        store(ds + (int64_t)(K - 1 + t) * a.width, v);
      }
    };
    float lag[K][VEC];
    if (t0 + SPAN <= n) {   // all of its own steps are there
      constexpr int N = SPAN + K - 1;
      Raw<T, VEC> rx[N], ry[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int at = k < SPAN ? k : min(k, n - 1 - t0);   // steps behind the row's end count as zero below
        rx[k] = load_raw<T, VEC>(x + at * a.x.step);
        ry[k] = load_raw<T, VEC>(dy + at * g.dy.step);
      }
      const unsigned over = ends<N>(a, t0, n, r);
      taps_before<T, VEC, K>(a, t0, r, c, false, false, lag);
      float ring[4][VEC], acc[4][VEC], before[K][VEC];   // input of step t0 + k, and its gradient so far, in slot k mod 4; of the state's taps
      clear(ring[0]);
#pragma unroll
      for (int j = 0; j < K; ++j) clear(before[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) clear(acc[j]);
#pragma unroll
      for (int j = 1; j < K; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) ring[4 - j][i] = lag[j][i];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if ((over >> k) & 1) {   // earlier steps get nothing from this one: theirs are finished
#pragma unroll
          for (int j = 1; j < K; ++j) clear(ring[(k + 4 - j) % 4]);
          asm volatile("");
        }
        unpack<T, VEC>(rx[k], ring[k % 4]);
        float d[VEC], pre[VEC];
        unpack<T, VEC>(ry[k], d);
        convolve<VEC, K>(pre, w, bias, [&](int j) -> const float (&)[VEC] { return ring[(k + 4 - j) % 4]; });
        through_act(d, pre);
        if (k >= SPAN && t0 + k >= n) clear(d);
        if (k < SPAN) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            db[i] += d[i];
#pragma unroll
            for (int j = 0; j < K; ++j) dw[j][i] = fmaf(d[i], ring[(k + 4 - j) % 4][i], dw[j][i]);
          }
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
          if (k - j >= SPAN) continue;   // not of this unit
          bool same = true;              // no end between the two
#pragma unroll
          for (int q = k - j + 1; q <= k; ++q) same = same && (q < 1 || !((over >> (q < 1 ? 0 : q)) & 1));
          if (k - j < 0) {
            if (s == 0 && same)
#pragma unroll
              for (int i = 0; i < VEC; ++i) before[j - k][i] = fmaf(w[j][i], d[i], before[j - k][i]);
          } else if (same) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[(k - j + 4) % 4][i] = fmaf(w[j][i], d[i], acc[(k - j + 4) % 4][i]);
          }
        }
        if (k >= K - 1) {
          const int q = k - (K - 1);
          float (&v)[VEC] = acc[q % 4];
          if (g.dstate_out && t0 + q >= n - (K - 1) && (over & ((2u << (n - 1 - t0)) - 1) & ~((2u << q) - 1)) == 0) {   // a tap of the state that comes out
            float more[VEC];
            load(g.dstate_out + ((int64_t)r * (K - 1) + (t0 + q - (n - (K - 1)))) * a.width + c, more);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] += more[i];
          }
          store(dx + (t0 + q) * g.dx.step, v);
          clear(v);
        }
      }
      if (s == 0 && ds)
#pragma unroll
        for (int j = 1; j < K; ++j) store(ds + (int64_t)(K - 1 - j) * a.width, before[j]);
    } else if (t0 < n || (n == 0 && s == 0)) {   // a row's last steps
      int valid = taps_before<T, VEC, K>(a, t0, r, c, false, false, lag);
      float acc[K][VEC];   // gradient of the input j steps before, so far
#pragma unroll
      for (int j = 0; j < K; ++j) clear(acc[j]);
      const int stop = min(t1, n) + K - 1;   // behind the row's end, K - 1 steps without inputs finish its last taps
#pragma unroll 1
      for (int t = t0; t < stop; ++t, x += a.x.step, dy += g.dy.step) {
        if (t < n) {
          if (t > t0) valid = min(valid + 1, K - 1);
          if (a.done && t > t0 && a.done[(int64_t)(t - 1) * a.rows + r]) {
            valid = 0;
#pragma unroll
            for (int j = 1; j < K; ++j) clear(lag[j]);
          }
          load(x, lag[0]);
          float d[VEC], pre[VEC];
          load(dy, d);
          convolve<VEC, K>(pre, w, bias, [&](int j) -> const float (&)[VEC] { return lag[j]; });
          through_act(d, pre);
#pragma unroll
          for (int j = 0; j < K; ++j) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              if (t < t1) dw[j][i] = fmaf(d[i], lag[j][i], dw[j][i]);
              if (j <= valid) acc[j][i] = fmaf(w[j][i], d[i], acc[j][i]);
            }
          }
          if (t < t1)
#pragma unroll
            for (int i = 0; i < VEC; ++i) db[i] += d[i];
        }
        emit(t - (K - 1), acc[K - 1], valid);
#pragma unroll
        for (int j = K - 1; j > 0; --j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            lag[j][i] = lag[j - 1][i];
            acc[j][i] = acc[j - 1][i];
          }
        clear(acc[0]);
      }
    }
    clear(lag[0]);
    for (int t = max(t0, n); t < t1; ++t) store(dx + t * g.dx.step, lag[0]);
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
  if (a->taps < 2 || a->taps > 4 || (int64_t)a->rows * (a->steps / std::min(FWD_SPAN, BWD_SPAN) + 1) > INT32_MAX) return BNB_ERR_UNSUPPORTED_DIMS;
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

// Channel groups of a CTA: all of a row's in as few equal tiles as 64 threads allow.
int tile_width(int groups) {
  const int tiles = (groups + 63) / 64;
  return (groups + tiles - 1) / tiles;
}

// CTAs: as many as the chip holds at once at `resident` an SM, which then go over the units.
Plan plan(const BnbCausalConv& a, int vec, int span, int resident) {
  Plan p;
  const int groups = (a.width + vec - 1) / vec;
  p.bx = tile_width(groups);
  p.tiles = (groups + p.bx - 1) / p.bx;
  p.spans = (unsigned)std::max(1, (a.steps + span - 1) / span);
  const int64_t units = (int64_t)a.rows * p.spans;
  p.units = (unsigned)units;
  p.by = (int)std::max<int64_t>(1, std::min<int64_t>(256 / p.bx, units));
  p.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((units + p.by - 1) / p.by, std::max(1, 148 * resident / p.tiles)));
  return p;
}

// Channels of a thread, and CTAs of an SM: what was fastest in bfloat16, with the spans: forward 4 channels, 8 steps, 4 CTAs 90 us, 3 CTAs 95, 16 steps
// 112; backward 2 channels, 16 steps, 2 CTAs 217 us, 4 channels, 8 steps 233, 3 CTAs 261.  With four taps not all of a span's loads, weights
// and sums stay in registers: 16-bit calls spill 52 bytes a thread forward and up to 40 backward, float32 ones, whose loads take
// twice the registers, up to 276 and 64.
constexpr int FWD_VEC = 4, FWD_RESIDENT = 4, BWD_VEC = 2, BWD_RESIDENT = 2;

template <typename T, int VEC, int K>
int launch_fwd(const BnbCausalConv& a, cudaStream_t st) {
  const Plan p = plan(a, VEC, FWD_SPAN, FWD_RESIDENT);
  const dim3 grid(p.blocks, p.tiles), block(p.bx, p.by);
  if (grid.y > 65535) return BNB_ERR_UNSUPPORTED_DIMS;
  count_launch();
  if (a.activation == BNB_ACT_SILU) k_conv<T, VEC, K, true><<<grid, block, 0, st>>>(a, p.units, p.spans);
  else k_conv<T, VEC, K, false><<<grid, block, 0, st>>>(a, p.units, p.spans);
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
  const Plan p = plan(a, VEC, BWD_SPAN, BWD_RESIDENT);
  const size_t smem = (size_t)p.by * (K + 1) * p.bx * VEC * 4;   // at most 256 threads x 2 channels x 5 floats = 10 KB
  const dim3 grid(p.blocks, p.tiles), block(p.bx, p.by);
  count_launch();
  if (a.activation == BNB_ACT_SILU) k_conv_bwd<T, VEC, K, true><<<grid, block, smem, st>>>(a, g, p.units, p.spans, part);
  else k_conv_bwd<T, VEC, K, false><<<grid, block, smem, st>>>(a, g, p.units, p.spans, part);
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
  return std::max(part_bytes(*a, plan(*a, 1, BWD_SPAN, BWD_RESIDENT)), part_bytes(*a, plan(*a, BWD_VEC, BWD_SPAN, BWD_RESIDENT)));
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
