// The selective state space recurrence, forward: whole sequences and single tokens.  For every row, channel and state n
//
//   p = softplus(delta + bias),  h_n = exp(p a_n) h_n + p u b_n,  y = (sum_n c_n h_n + d u) silu(z)
//
// A sequence reads u, delta, z and writes y, eight bytes a channel and step in 16 bits, and computes an exponential for each state: with 16
// states the exponentials (16 a clock and SM) bound it, not memory.  selective_scan.cuh describes how the work is laid out.
// A single token reads and writes the state, eight bytes for each of its elements: memory bounds it.
#include "selective_scan.cuh"

namespace bnb {
namespace scan {

int check(const BnbSelectiveScan* a) {
  if (!a) return BNB_ERR_NULL_POINTER;
  if (a->steps < 0 || a->rows < 0 || a->width < 0 || a->element < 0 || a->element > 2) return BNB_ERR_BAD_ARGUMENT;
  if (a->states < 1 || a->states > 64) return BNB_ERR_UNSUPPORTED_DIMS;
  if (a->groups < 1 || a->width % a->groups) return BNB_ERR_BAD_ARGUMENT;
  if (a->rows == 0 || a->width == 0) return BNB_OK;
  if (!a->a) return BNB_ERR_NULL_POINTER;
  if (a->steps && (!a->u.data || !a->delta.data || !a->b.data || !a->c.data)) return BNB_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(a->state_in) | reinterpret_cast<uintptr_t>(a->state_out) | reinterpret_cast<uintptr_t>(a->a) |
       reinterpret_cast<uintptr_t>(a->kept)) & 15) return BNB_ERR_MISALIGNED;
  if ((int64_t)a->rows * a->width > (int64_t)1 << 40) return BNB_ERR_BAD_ARGUMENT;
  return BNB_OK;
}

namespace {

constexpr int L = 16;    // steps of a chunk
constexpr int CT = 32;   // channels of a CTA

enum Pass : int { WHOLE, LOCAL, JOINED };   // one split; what a split leaves of a zero start; from its starting state

struct Work {
  float* local;       // (splits, rows, width, 4 KL)
  float* sum_p;       // (splits, rows, width)
  uint8_t* cut;       // (splits, rows)
  Splits splits;
  int tiles_a_group;
  bool paired;        // pairs of channels of u, delta, z and y lie on their boundary
};

// 64 registers a thread, so that 32 warps fit on an SM, and the splits that are aimed at all at once: 665 -> 647 us at 32 steps x 8192 rows x 256
// channels x 16 states of bfloat16, 1669 -> 1170 at 128 channels x 64 states, 120 -> 112 for the joined pass over 2 rows x 4093 steps x 1536
// channels; what spills costs a launch of few warps 4 us.  Fewer lanes a channel prepare more steps a thread and are left their registers.
template <typename T, int KL, Pass PASS>
__global__ void __launch_bounds__(CT * KL, KL >= 4 ? 1024 / (CT * KL) : 1) k_scan(const __grid_constant__ BnbSelectiveScan q, const __grid_constant__ Work w) {
  constexpr int THREADS = CT * KL, NP = NS * KL;
  constexpr int BC = (L * NP + THREADS - 1) / THREADS;            // elements of b and c that a thread fetches
  constexpr int PAIRS = CT / 2, AT_ONCE = THREADS / PAIRS < L ? THREADS / PAIRS : L, PER = L / AT_ONCE;   // steps prepared at a time, by a thread
  constexpr int SUMS = KL < 4 ? KL : 4;                           // parts that y is left in
  constexpr bool Y = PASS != LOCAL;
  __shared__ __align__(16) float4 pp_s[L][CT];                    // p, p, p u, p u
  __shared__ __align__(16) float b_s[L][NP], c_s[Y ? L : 1][NP], y_s[Y ? L : 1][CT][SUMS];
  const int tid = threadIdx.x, cl = tid / KL, lane = tid % KL;
  const int tiles = w.tiles_a_group * q.groups, share = q.width / q.groups;
  const int r = blockIdx.x / tiles, tile = blockIdx.x - r * tiles, group = tile / w.tiles_a_group;
  const int c0 = group * share + (tile - group * w.tiles_a_group) * CT, c_end = min((group + 1) * share, c0 + CT);   // channels [c0, c_end)
  const int ch = c0 + cl;
  const bool owns = ch < c_end, wide = q.states % NS == 0;
  const int n = row_steps(q.lengths, r, q.steps);
  const int split = blockIdx.y, first = split * w.splits.steps, last = min(q.steps, first + w.splits.steps), live = min(n, last);
  const int64_t rc = (int64_t)r * q.width + ch;

  F2 rate[2] = {f2(0.f), f2(0.f)}, h[2] = {f2(0.f), f2(0.f)};
  auto state = [&](float (&v)[NS]) {
    const float2 x = halves(h[0]), z = halves(h[1]);
    v[0] = x.x, v[1] = x.y, v[2] = z.x, v[3] = z.y;
  };
  if (owns) {
    float v[NS];
    load_states(v, q.a + (int64_t)ch * q.states, NS * lane, q.states, wide && NS * lane < q.states);
    rate[0] = mul(f2(v[0], v[1]), f2(LOG2E));
    rate[1] = mul(f2(v[2], v[3]), f2(LOG2E));
    clear_states(v);
    if constexpr (PASS == WHOLE) {
      if (q.state_in) load_states(v, q.state_in + rc * q.states, NS * lane, q.states, wide && NS * lane < q.states);
    } else if constexpr (PASS == JOINED) {
      load_states(v, w.local + ((int64_t)split * q.rows * q.width + rc) * NP, NS * lane, NP, true);
    }
    h[0] = f2(v[0], v[1]);
    h[1] = f2(v[2], v[3]);
  }

  // what this thread prepares: channels c0 + 2 pair, + 1 of steps t0 + step + k AT_ONCE
  const int pair = tid % PAIRS, step = tid / PAIRS, count = step < L ? max(0, min(2, c_end - (c0 + 2 * pair))) : 0, pc = c0 + 2 * pair;
  F2 bias = f2(0.f), skip = f2(0.f);
  if (q.delta_bias) bias = f2(count > 0 ? q.delta_bias[pc] : 0.f, count > 1 ? q.delta_bias[pc + 1] : 0.f);
  if (q.d) skip = f2(count > 0 ? q.d[pc] : 0.f, count > 1 ? q.d[pc + 1] : 0.f);
  const T* up = static_cast<const T*>(q.u.data) + r * q.u.row + pc + (first + step) * q.u.step;
  const T* dp = static_cast<const T*>(q.delta.data) + r * q.delta.row + pc + (first + step) * q.delta.step;
  const T* zp = static_cast<const T*>(q.z.data) + r * q.z.row + pc + (first + step) * q.z.step;
  T* yp = static_cast<T*>(q.y.data) + r * q.y.row + pc + (first + step) * q.y.step;
  const T* bp = static_cast<const T*>(q.b.data) + r * q.b.row + group * q.b.group + first * q.b.step;
  const T* cp = static_cast<const T*>(q.c.data) + r * q.c.row + group * q.c.group + first * q.c.step;
  float* kept = q.kept && owns ? q.kept + ((int64_t)(first / KEEP) * q.rows * q.width + rc) * NP : nullptr;
  const int64_t kept_step = (int64_t)q.rows * q.width * NP;
  const bool gated = q.z.data != nullptr;
  const T none = from_f<T>(0.f);
  Raw<T, 2> u_r[PER], d_r[PER], z_r[PER];
  T b_r[BC], c_r[BC];
  unsigned cuts_next = 0;   // bit k: an episode ended before step t0 + k
  auto fetch = [&](int t0) {   // moves the pointers on
    if (q.done) {
      const int t = t0 + (tid & 31) - 1;
      cuts_next = __ballot_sync(0xffffffffu, (tid & 31) < L && t >= 0 && t + 1 < n && q.done[(int64_t)max(t, 0) * q.rows + r]);
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int have = t0 + step + k * AT_ONCE < live ? count : 0;
      u_r[k] = load_pair(up + k * AT_ONCE * q.u.step, have, w.paired);
      d_r[k] = load_pair(dp + k * AT_ONCE * q.delta.step, have, w.paired);
      z_r[k] = load_pair(zp + k * AT_ONCE * q.z.step, Y && gated ? have : 0, w.paired);
    }
#pragma unroll
    for (int k = 0; k < BC; ++k) {
      const int e = tid + k * THREADS, t = e / NP, s = e % NP;
      const bool on = e < L * NP && s < q.states && t0 + t < live;
      b_r[k] = on ? bp[t * q.b.step + s] : none;
      if (Y) c_r[k] = on ? cp[t * q.c.step + s] : none;
    }
    up += L * q.u.step;
    dp += L * q.delta.step;
    zp += L * q.z.step;
    bp += L * q.b.step;
    cp += L * q.c.step;
  };
  float sum_p = 0.f;
  bool any_cut = false;
  if (first < live) fetch(first);
#pragma unroll 1
  for (int t0 = first; t0 < live; t0 += L) {
    F2 u_f[PER], gate[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      u_f[k] = floats_of<T>(u_r[k]);
      const int t = step + k * AT_ONCE;
      F2 p = step_size(add(floats_of<T>(d_r[k]), bias), q.softplus);
      if (t0 + t >= live) p = f2(0.f);
      if (Y) {
        const F2 z = floats_of<T>(z_r[k]);
        gate[k] = gated ? mul(z, sigmoid_pair<T>(z)) : f2(1.0f);
      }
      if (step < L) {
        const float2 ps = halves(p), pu = halves(mul(p, u_f[k]));
        pp_s[t][2 * pair] = make_float4(ps.x, ps.x, pu.x, pu.x);
        pp_s[t][2 * pair + 1] = make_float4(ps.y, ps.y, pu.y, pu.y);
      }
    }
#pragma unroll
    for (int k = 0; k < BC; ++k) {
      const int e = tid + k * THREADS;
      if (e < L * NP) {
        (&b_s[0][0])[e] = to_f(b_r[k]);
        if (Y) (&c_s[0][0])[e] = to_f(c_r[k]);
      }
    }
    const unsigned cuts = cuts_next;
    any_cut |= cuts != 0;
    __syncthreads();
    if (t0 + L < live) fetch(t0 + L);
#pragma unroll 1
    for (int g0 = 0; g0 < L; g0 += KEEP) {
      if (Y && kept && t0 + g0 < live) {
        float v[NS];
        state(v);
        store_states(kept, v, NS * lane, NP, true);
        kept += kept_step;
      }
auto walk = [&](auto with_cuts) {
      constexpr bool cutting = decltype(with_cuts)::value;
#pragma unroll
      for (int k = 0; k < KEEP; ++k) {
        const int t = g0 + k;
        if (cutting && ((cuts >> t) & 1)) h[0] = h[1] = f2(0.f);
        const ulonglong2 pp = *reinterpret_cast<const ulonglong2*>(&pp_s[t][cl]), b = *reinterpret_cast<const ulonglong2*>(&b_s[t][NS * lane]);
        const F2 p{pp.x}, pu{pp.y};
        const float2 m0 = halves(mul(p, rate[0])), m1 = halves(mul(p, rate[1]));
        h[0] = fma(f2(ex2_fast(m0.x), ex2_fast(m0.y)), h[0], mul(pu, F2{b.x}));
        h[1] = fma(f2(ex2_fast(m1.x), ex2_fast(m1.y)), h[1], mul(pu, F2{b.y}));
        if constexpr (!Y) {
          sum_p += halves(p).x;
        } else {
          const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&c_s[t][NS * lane]);
          const float2 both = halves(fma(F2{c.x}, h[0], mul(F2{c.y}, h[1])));
          float y = both.x + both.y;
#pragma unroll
          for (int o = SUMS; o < KL; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
          if (KL <= SUMS || lane < SUMS) y_s[t][cl][lane % SUMS] = y;
        }
      }
      };
      // ends of episodes are rare: without any, the steps are one run of instructions
      if ((cuts >> g0) & ((1u << KEEP) - 1)) walk(std::true_type{});
      else walk(std::false_type{});
    }
    __syncthreads();
    if constexpr (Y) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int t = step + k * AT_ONCE;
        if (t0 + t >= live || step >= L) continue;
        float2 y = make_float2(y_s[t][2 * pair][0], y_s[t][2 * pair + 1][0]);
#pragma unroll
        for (int i = 1; i < SUMS; ++i) y.x += y_s[t][2 * pair][i], y.y += y_s[t][2 * pair + 1][i];
        store_pair(yp + k * AT_ONCE * q.y.step, mul(fma(skip, u_f[k], f2(y.x, y.y)), gate[k]), count, w.paired);
      }
      yp += L * q.y.step;
    }
  }
  float v[NS];
  state(v);
  if constexpr (!Y) {
    if (owns) {
      store_states(w.local + ((int64_t)split * q.rows * q.width + rc) * NP, v, NS * lane, NP, true);
      if (lane == 0) w.sum_p[(int64_t)split * q.rows * q.width + rc] = sum_p;
    }
    if (tid == 0 && tile == 0) w.cut[(int64_t)split * q.rows + r] = any_cut;
  } else {
    yp = static_cast<T*>(q.y.data) + r * q.y.row + pc;
    for (int t = max(first, n) + step; step < L && t < last; t += AT_ONCE) store_pair(yp + t * q.y.step, f2(0.f), count, w.paired);
    // the split that holds the row's last step has its state; a row without steps, the first one
    if (owns && q.state_out && ((first < n && n <= last) || (n == 0 && split == 0)))
      store_states(q.state_out + rc * q.states, v, NS * lane, q.states, wide && NS * lane < q.states);
  }
}

// Four b or c of a lane as they lie: one access where that is on its boundary.
template <typename T>
__device__ __forceinline__ Raw<T, NS> load_shared(const T* at, int n0, int states, bool whole) {
  if (whole) return load_raw<T, NS>(at + n0);
  Raw<T, NS> r;
  T* v = reinterpret_cast<T*>(r.w);
#pragma unroll
  for (int i = 0; i < NS; ++i) v[i] = n0 + i < states ? at[n0 + i] : from_f<T>(0.f);
  return r;
}

// One token a row.  A thread keeps the constants of its channel's states and goes over rows ROWS at a time, whose loads are on their way
// together.  What is per channel and row (step size, gate, output) is computed by one of the channel's lanes for each row and passed on.
template <typename T, int KL, int ROWS, bool WIDE>
__global__ void __launch_bounds__(256, 3) k_step(const __grid_constant__ BnbSelectiveScan q, bool whole) {
  constexpr int BITS = KL == 1 ? 0 : KL == 2 ? 1 : KL == 4 ? 2 : KL == 8 ? 3 : 4;
  constexpr int PER = ROWS > KL ? ROWS / KL : 1, SHARE = KL > ROWS ? KL / ROWS : 1;   // rows of a lane, lanes of a row
  const int lane = threadIdx.x % KL, ch = blockIdx.y * (256 / KL) + threadIdx.x / KL;
  const bool on = ch < q.width;
  const int c = on ? ch : 0, group = c / (q.width / q.groups), n0 = NS * lane;
  float rate_[NS];
  load_states(rate_, q.a + (int64_t)c * q.states, n0, q.states, WIDE && n0 < q.states);
  const F2 rate[2] = {mul(f2(rate_[0], rate_[1]), f2(LOG2E)), mul(f2(rate_[2], rate_[3]), f2(LOG2E))};
  const float bias = q.delta_bias ? q.delta_bias[c] : 0.f, skip = q.d ? q.d[c] : 0.f;
  const bool real = on && n0 < q.states;
  const int first = KL > ROWS ? lane / SHARE : lane * PER;   // this lane's rows among ROWS
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < q.rows; r0 += (int64_t)gridDim.x * ROWS) {
    float h[ROWS][NS];
    Raw<T, NS> b[ROWS], cc[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int64_t r = min(r0 + k, (int64_t)q.rows - 1);
#pragma unroll
      for (int i = 0; i < NS; ++i) h[k][i] = 0.f;
      if (real && q.state_in && !(q.reset && q.reset[r])) load_states(h[k], q.state_in + (r * q.width + c) * q.states, n0, q.states, WIDE);
    }
    float u[PER], p[PER], gate[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int64_t r = min(r0 + first + k, (int64_t)q.rows - 1);
      u[k] = to_f(static_cast<const T*>(q.u.data)[r * q.u.row + c]);
      p[k] = to_f(static_cast<const T*>(q.delta.data)[r * q.delta.row + c]);
      gate[k] = q.z.data ? to_f(static_cast<const T*>(q.z.data)[r * q.z.row + c]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int64_t r = min(r0 + k, (int64_t)q.rows - 1);
      b[k] = load_shared(static_cast<const T*>(q.b.data) + r * q.b.row + group * q.b.group, n0, q.states, whole && n0 < q.states);
      cc[k] = load_shared(static_cast<const T*>(q.c.data) + r * q.c.row + group * q.c.group, n0, q.states, whole && n0 < q.states);
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      p[k] = step_size(p[k] + bias, q.softplus);
      gate[k] = q.z.data ? gate[k] * sigmoid<T>(gate[k]) : 1.f;
    }
    float y[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int from = (threadIdx.x & 31 & ~(KL - 1)) + (KL > ROWS ? k * SHARE : k / PER);
      const float pk = __shfl_sync(0xffffffffu, p[k % PER], from), pu = __shfl_sync(0xffffffffu, p[k % PER] * u[k % PER], from);
      F2 sum = f2(0.f);
      float bf[NS], cf[NS];
      unpack<T, NS>(b[k], bf);
      unpack<T, NS>(cc[k], cf);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 m = halves(mul(f2(pk), rate[i]));
        const F2 v = fma(f2(ex2_fast(m.x), ex2_fast(m.y)), f2(h[k][2 * i], h[k][2 * i + 1]), mul(f2(pu), f2(bf[2 * i], bf[2 * i + 1])));
        sum = fma(f2(cf[2 * i], cf[2 * i + 1]), v, sum);
        const float2 o = halves(v);
        h[k][2 * i] = o.x, h[k][2 * i + 1] = o.y;
      }
      const float2 o = halves(sum);
      y[k] = o.x + o.y;
      if (real && r0 + k < q.rows) store_states(q.state_out + ((r0 + k) * q.width + c) * q.states, h[k], n0, q.states, WIDE);
    }
    sum_lanes<ROWS, 0, BITS>(y);   // this lane's rows' sums stand in front
    if (on && writes_sum<ROWS, 0, BITS>()) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int64_t r = r0 + first + k;
        if (r < q.rows) static_cast<T*>(q.y.data)[r * q.y.row + c] = from_f<T>(fmaf(skip, u[k], y[k]) * gate[k]);
      }
    }
  }
}

// 32 warps of each SM: what the splits aim at.
Splits splits(const BnbSelectiveScan& a, int kl, int tiles) {
  return splits_of(a.steps, (int64_t)tiles * a.rows, 148 * std::max(1, 1024 / (CT * kl)));
}
int tiles_a_group(const BnbSelectiveScan& a) { return (a.width / a.groups + CT - 1) / CT; }

struct Scratch { size_t local, sum_p, cut, total; };
Scratch scratch_of(const BnbSelectiveScan& a, const Splits& s, int kl) {
  Scratch o{};
  if (s.count == 1) return o;
  const size_t cells = (size_t)s.count * a.rows * a.width;
  o.sum_p = round256(cells * NS * kl * 4);
  o.cut = o.sum_p + round256(cells * 4);
  o.total = o.cut + round256((size_t)s.count * a.rows);
  return o;
}

template <typename T, int KL>
int launch(const BnbSelectiveScan& a, uint8_t* scratch, cudaStream_t st) {
  Work w{};
  w.tiles_a_group = tiles_a_group(a);
  const int64_t tiles = (int64_t)w.tiles_a_group * a.groups;
  w.splits = splits(a, KL, (int)tiles);
  w.paired = a.width / a.groups % 2 == 0 && even_view(a.u, a.element) && even_view(a.delta, a.element) && even_view(a.y, a.element) &&
             (!a.z.data || even_view(a.z, a.element));
  if (tiles * a.rows > INT32_MAX || w.splits.count > 65535) return BNB_ERR_UNSUPPORTED_DIMS;
  const dim3 grid((unsigned)(tiles * a.rows), w.splits.count);
  if (w.splits.count == 1) {
    count_launch();
    k_scan<T, KL, WHOLE><<<grid, CT * KL, 0, st>>>(a, w);
  } else {
    const Scratch s = scratch_of(a, w.splits, KL);
    w.local = reinterpret_cast<float*>(scratch);
    w.sum_p = reinterpret_cast<float*>(scratch + s.sum_p);
    w.cut = scratch + s.cut;
    count_launch();
    k_scan<T, KL, LOCAL><<<grid, CT * KL, 0, st>>>(a, w);
    const int64_t cells = (int64_t)a.rows * a.width * NS * KL;
    count_launch();
    k_join<false><<<(unsigned)((cells + 255) / 256), 256, 0, st>>>(w.local, w.sum_p, w.cut, a.a, a.state_in, w.splits.count, a.rows, a.width, a.states, NS * KL);
    count_launch();
    k_scan<T, KL, JOINED><<<grid, CT * KL, 0, st>>>(a, w);
  }
  return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
}

template <typename T, int KL>
int launch_step(const BnbSelectiveScan& a, cudaStream_t st) {
  constexpr int ROWS = 4;
  const int tiles = (a.width * KL + 255) / 256;
  if (tiles > 65535) return BNB_ERR_UNSUPPORTED_DIMS;
  const int64_t groups = (a.rows + ROWS - 1) / ROWS, fit = std::max(1, 148 * 3 / tiles);
  auto on = [&](const BnbView& v) { return reinterpret_cast<uintptr_t>(v.data) % (4 * sizeof(T)) == 0 && v.row % 4 == 0 && v.group % 4 == 0; };
  const bool wide = a.states % NS == 0, whole = wide && on(a.b) && on(a.c);
  count_launch();
  if (groups < fit) {   // fewer rows than it takes to fill the chip: one each
    const dim3 grid((unsigned)a.rows, tiles);
    if (wide) k_step<T, KL, 1, true><<<grid, 256, 0, st>>>(a, whole);
    else k_step<T, KL, 1, false><<<grid, 256, 0, st>>>(a, whole);
  } else {
    const dim3 grid((unsigned)fit, tiles);
    if (wide) k_step<T, KL, ROWS, true><<<grid, 256, 0, st>>>(a, whole);
    else k_step<T, KL, ROWS, false><<<grid, 256, 0, st>>>(a, whole);
  }
  return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
}

template <typename T>
int run(const BnbSelectiveScan& a, uint8_t* scratch, cudaStream_t st) {
  switch (lanes_of(a.states)) {
    case 1: return launch<T, 1>(a, scratch, st);
    case 2: return launch<T, 2>(a, scratch, st);
    case 4: return launch<T, 4>(a, scratch, st);
    case 8: return launch<T, 8>(a, scratch, st);
    default: return launch<T, 16>(a, scratch, st);
  }
}
template <typename T>
int run_step(const BnbSelectiveScan& a, cudaStream_t st) {
  switch (lanes_of(a.states)) {
    case 1: return launch_step<T, 1>(a, st);
    case 2: return launch_step<T, 2>(a, st);
    case 4: return launch_step<T, 4>(a, st);
    case 8: return launch_step<T, 8>(a, st);
    default: return launch_step<T, 16>(a, st);
  }
}

}  // namespace
}  // namespace scan
}  // namespace bnb

using namespace bnb;

extern "C" size_t bnb_selective_scan_kept_bytes(const BnbSelectiveScan* a) {
  if (scan::check(a)) return 0;
  return (size_t)((a->steps + scan::KEEP - 1) / scan::KEEP) * a->rows * a->width * scan::NS * scan::lanes_of(a->states) * 4;
}

extern "C" size_t bnb_selective_scan_scratch_bytes(const BnbSelectiveScan* a) {
  if (scan::check(a) || a->rows == 0 || a->width == 0) return 0;
  const int kl = scan::lanes_of(a->states);
  return scan::scratch_of(*a, scan::splits(*a, kl, scan::tiles_a_group(*a) * a->groups), kl).total;
}

extern "C" int bnb_selective_scan_fwd(const BnbSelectiveScan* a, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int st = scan::check(a)) return st;
  if (a->rows == 0 || a->width == 0) return BNB_OK;
  if (a->reset || (a->state_in && a->state_in == a->state_out)) return BNB_ERR_BAD_ARGUMENT;
  if (!a->state_out || (a->steps && !a->y.data)) return BNB_ERR_NULL_POINTER;
  const size_t need = bnb_selective_scan_scratch_bytes(a);
  if (need && (!scratch || scratch_bytes < need)) return BNB_ERR_SCRATCH_TOO_SMALL;
  const auto s = static_cast<cudaStream_t>(stream);
  auto* at = static_cast<uint8_t*>(scratch);
  return a->element == BNB_ELEM_F32 ? scan::run<float>(*a, at, s)
       : a->element == BNB_ELEM_BF16 ? scan::run<__nv_bfloat16>(*a, at, s) : scan::run<__half>(*a, at, s);
}

extern "C" int bnb_selective_step(const BnbSelectiveScan* a, void* stream) {
  if (const int st = scan::check(a)) return st;
  if (a->rows == 0 || a->width == 0) return BNB_OK;
  if (a->steps != 1 || a->done || a->lengths || a->kept) return BNB_ERR_BAD_ARGUMENT;
  if (!a->state_out || !a->y.data) return BNB_ERR_NULL_POINTER;
  const auto s = static_cast<cudaStream_t>(stream);
  return a->element == BNB_ELEM_F32 ? scan::run_step<float>(*a, s)
       : a->element == BNB_ELEM_BF16 ? scan::run_step<__nv_bfloat16>(*a, s) : scan::run_step<__half>(*a, s);
}
