// The selective state space recurrence, backward.  With dyv = dy silu(z), g_n the gradient of h_n behind a step and h- the state
// before it (after an episode end: 0):
//
//   g_n = carry_n + c_n dyv,   dc_n = sum_ch dyv h_n,   db_n = sum_ch g_n p u,   da_n = sum g_n e_n h-_n p,   carry_n = e_n g_n   (e_n = exp(p a_n))
//   du = p sum_n g_n b_n + d dyv,   dp = sum_n g_n e_n h-_n a_n + u sum_n g_n b_n,   ddelta = dp softplus'(delta + bias)
//   dz = dy (sum_n c_n h_n + d u) silu'(z),   dd = sum dyv u
//
// The forward kept the states of every eighth step.  A CTA takes the chunks of eight steps from the last to the first: the states of
// a chunk are computed forward into registers, with their decays, and the adjoint walks back over them.  Sums over
// the channels (db, dc) go through the lanes of a warp, the warps of the CTA and, where a group has several tiles of channels, a
// short kernel over the tiles; sums over rows and time (da, dd, d bias) stay in registers while a CTA goes over its rows.  No
// atomics, so a result does not depend on timing.
//
// About 35 instructions a state and step bound it, the exponential among them; memory moves some 24 bytes a channel and step.
#include "selective_scan.cuh"

namespace bnb {
namespace scan {
namespace {

constexpr int L = KEEP;

struct Work {
  float* carry;      // (splits, rows, width, 4 KL): the adjoint behind each split, as k_join leaves it
  float* sum_p;      // (splits, rows, width)
  uint8_t* cut;      // (splits, rows)
  float* part_bc;    // (tiles of a group, steps, rows, groups, 8 KL) or null: b and c gradients written directly
  float* part_a;     // (splits * row blocks, width, 4 KL)
  float* part_d;     // (splits * row blocks, 2, width): d d, d bias
  Splits splits;     // steps of a split: a multiple of 16, so of a chunk
  int tiles_a_group;
  int row_blocks;
};

template <int KL> constexpr int CHANNELS = KL <= 4 ? 64 : 256 / KL;   // of a CTA

// LOCAL: only what a split leaves of a zero adjoint behind it, see selective_scan.cuh.
template <typename T, int KL, bool LOCAL>
__global__ void __launch_bounds__(CHANNELS<KL> * KL) k_scan_bwd(const __grid_constant__ BnbSelectiveScan q, const __grid_constant__ BnbSelectiveScanGrads g, Work w) {
  constexpr int CT = CHANNELS<KL>, THREADS = CT * KL, NP = NS * KL, PER = (L + KL - 1) / KL, WARPS = THREADS / 32;
  constexpr int BITS = KL == 1 ? 0 : KL == 2 ? 1 : KL == 4 ? 2 : KL == 8 ? 3 : 4;
  constexpr int BC = (L * NP + THREADS - 1) / THREADS;
  constexpr int GROUP = 4;   // steps whose sums over a channel's lanes are taken together
  __shared__ float p_s[L][CT], pu_s[LOCAL ? 1 : L][CT], dy_s[L][CT], sum_s[LOCAL ? 1 : L][3][CT];
  __shared__ __align__(16) float b_s[LOCAL ? 1 : L][NP], c_s[L][NP];
  extern __shared__ float red[];   // (L, WARPS, 2 NP): sums over a warp's channels
  const int tid = threadIdx.x, cl = tid / KL, lane = tid % KL, warp = tid / 32;
  const int tiles = w.tiles_a_group * q.groups, share = q.width / q.groups;
  const int row_block = blockIdx.x / tiles, tile = blockIdx.x - row_block * tiles, group = tile / w.tiles_a_group, tile_in = tile - group * w.tiles_a_group;
  const int c0 = group * share + tile_in * CT, c_end = min((group + 1) * share, c0 + CT);
  const int ch = c0 + cl;
  const bool owns = ch < c_end, wide = q.states % NS == 0;
  const int split = blockIdx.y, first = split * w.splits.steps, last = min(q.steps, first + w.splits.steps);

  float rate[NS], da[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) rate[i] = da[i] = 0.f;
  if (owns) load_states(rate, q.a + (int64_t)ch * q.states, NS * lane, q.states, wide);
#pragma unroll
  for (int i = 0; i < NS; ++i) rate[i] *= LOG2E;
  const int pc = tid % CT, pt = tid / CT;   // prepares steps pt + k KL of channel c0 + pc
  const bool prepares = c0 + pc < c_end;
  const float bias = prepares && q.delta_bias ? q.delta_bias[c0 + pc] : 0.f, skip = prepares && q.d ? q.d[c0 + pc] : 0.f;
  const bool gated = q.z.data != nullptr;
  const T none = from_f<T>(0.f);
  float dd = 0.f, dbias = 0.f;

  for (int r = row_block; r < q.rows; r += w.row_blocks) {
    const int n = row_steps(q.lengths, r, q.steps), live = min(n, last);
    const int64_t rc = (int64_t)r * q.width + ch;
    const T* up = static_cast<const T*>(q.u.data) + r * q.u.row + c0 + pc;
    const T* dp = static_cast<const T*>(q.delta.data) + r * q.delta.row + c0 + pc;
    const T* zp = static_cast<const T*>(q.z.data) + r * q.z.row + c0 + pc;
    const T* yp = static_cast<const T*>(g.dy.data) + r * g.dy.row + c0 + pc;
    const T* bp = static_cast<const T*>(q.b.data) + r * q.b.row + group * q.b.group;
    const T* cp = static_cast<const T*>(q.c.data) + r * q.c.row + group * q.c.group;
    T* dup = static_cast<T*>(g.du.data) + r * g.du.row + c0 + pc;
    T* ddp = static_cast<T*>(g.ddelta.data) + r * g.ddelta.row + c0 + pc;
    T* dzp = static_cast<T*>(g.dz.data) + r * g.dz.row + c0 + pc;
    T* dbp = static_cast<T*>(g.db.data) + r * g.db.row + group * g.db.group;
    T* dcp = static_cast<T*>(g.dc.data) + r * g.dc.row + group * g.dc.group;
    float* part_bc = w.part_bc ? w.part_bc + (((int64_t)tile_in * q.steps * q.rows + r) * q.groups + group) * 2 * NP : nullptr;
    const int64_t part_step = (int64_t)q.rows * q.groups * 2 * NP;

    // steps behind the row's end
    if constexpr (!LOCAL) {
      if (prepares)
        for (int t = max(first, n) + pt; t < last; t += KL) {
          dup[t * g.du.step] = none;
          ddp[t * g.ddelta.step] = none;
          if (gated) dzp[t * g.dz.step] = none;
        }
      for (int64_t e = tid; e < (int64_t)(last - max(first, n)) * 2 * NP; e += THREADS) {
        const int t = max(first, n) + (int)(e / (2 * NP)), s = (int)(e % (2 * NP));
        if (part_bc) part_bc[t * part_step + s] = 0.f;
        else if (s < NP) { if (s < q.states) dbp[t * g.db.step + s] = none; }
        else if (s - NP < q.states) dcp[t * g.dc.step + s - NP] = none;
      }
    }

    float carry[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) carry[i] = 0.f;
    if (!LOCAL && owns) {
      if (w.splits.count > 1) load_states(carry, w.carry + ((int64_t)split * q.rows * q.width + rc) * NP, NS * lane, NP, true);
      else if (g.dstate_out) load_states(carry, g.dstate_out + rc * q.states, NS * lane, q.states, wide);
    }
    T u_r[PER], d_r[PER], z_r[PER], y_r[PER], b_r[BC], c_r[BC];
    float4 h_r = make_float4(0.f, 0.f, 0.f, 0.f);
    unsigned cuts_next = 0;
    auto fetch = [&](int t0) {
      if (q.done) {
        const int t = t0 + (tid & 31) - 1;
        cuts_next = __ballot_sync(0xffffffffu, (tid & 31) < L && t >= 0 && t + 1 < live && q.done[(int64_t)max(t, 0) * q.rows + r]);
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int t = t0 + pt + k * KL;
        const bool on = prepares && t < live && pt + k * KL < L;
        u_r[k] = on ? up[t * q.u.step] : none;
        d_r[k] = on ? dp[t * q.delta.step] : none;
        z_r[k] = gated && on ? zp[t * q.z.step] : none;
        y_r[k] = on ? yp[t * g.dy.step] : none;
      }
#pragma unroll
      for (int k = 0; k < BC; ++k) {
        const int e = tid + k * THREADS, t = t0 + e / NP, s = e % NP;
        const bool on = e < L * NP && s < q.states && t < live;
        if (!LOCAL) b_r[k] = on ? bp[t * q.b.step + s] : none;
        c_r[k] = on ? cp[t * q.c.step + s] : none;
      }
      if (!LOCAL && owns) h_r = *reinterpret_cast<const float4*>(q.kept + ((int64_t)(t0 / KEEP) * q.rows * q.width + rc) * NP + NS * lane);
    };
    float sum_p = 0.f;
    bool any_cut = false;
    const int begin = live > first ? (live - 1) / L * L : first - L;   // first is a multiple of L
    if (begin >= first) fetch(begin);
#pragma unroll 1
    for (int t0 = begin; t0 >= first; t0 -= L) {
      float u_f[PER], p_f[PER], dyv[PER], raw[PER], dgate[PER];   // dgate: dy silu'(z)
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int t = pt + k * KL;
        u_f[k] = to_f(u_r[k]);
        raw[k] = to_f(d_r[k]) + bias;
        p_f[k] = t0 + t < live ? step_size(raw[k], q.softplus) : 0.f;
        const float dy = to_f(y_r[k]);
        dyv[k] = dy;
        dgate[k] = 0.f;
        if (gated) {
          const float z = to_f(z_r[k]), sg = sigmoid<T>(z);
          dyv[k] = dy * (z * sg);
          dgate[k] = dy * (sg * fmaf(z, 1.f - sg, 1.f));
        }
        if (t < L) {
          p_s[t][pc] = p_f[k];
          dy_s[t][pc] = dyv[k];
          if (!LOCAL) pu_s[t][pc] = p_f[k] * u_f[k];
        }
      }
#pragma unroll
      for (int k = 0; k < BC; ++k) {
        const int e = tid + k * THREADS;
        if (e < L * NP) {
          if (!LOCAL) (&b_s[0][0])[e] = to_f(b_r[k]);
          (&c_s[0][0])[e] = to_f(c_r[k]);
        }
      }
      const float h0[NS] = {h_r.x, h_r.y, h_r.z, h_r.w};
      const unsigned cuts = cuts_next;
      any_cut |= cuts != 0;
      __syncthreads();
      if (t0 - L >= first) fetch(t0 - L);
      if constexpr (LOCAL) {
#pragma unroll
        for (int t = L - 1; t >= 0; --t) {
          const float p = p_s[t][cl], dy = dy_s[t][cl];
          const float4 c4 = *reinterpret_cast<const float4*>(&c_s[t][NS * lane]);
          const float c[NS] = {c4.x, c4.y, c4.z, c4.w};
          sum_p += p;
#pragma unroll
          for (int i = 0; i < NS; ++i) carry[i] = (cuts >> t) & 1 ? 0.f : ex2_fast(p * rate[i]) * fmaf(c[i], dy, carry[i]);
        }
        __syncthreads();
      } else {
        float h[L + 1][NS], e[L][NS];   // h[t]: before step t, episode ends applied; h[t + 1] behind it unless one follows
#pragma unroll
        for (int i = 0; i < NS; ++i) h[0][i] = cuts & 1 ? 0.f : h0[i];
#pragma unroll
        for (int t = 0; t < L; ++t) {
          const float p = p_s[t][cl], pu = pu_s[t][cl];
          const float4 b4 = *reinterpret_cast<const float4*>(&b_s[t][NS * lane]);
          const float b[NS] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            e[t][i] = ex2_fast(p * rate[i]);
            h[t + 1][i] = fmaf(e[t][i], h[t][i], pu * b[i]);
            if (t + 1 < L && ((cuts >> (t + 1)) & 1)) h[t + 1][i] = 0.f;
          }
        }
        float sums[GROUP][3];   // over the states: c h, g b, g e h- a
#pragma unroll
        for (int t = L - 1; t >= 0; --t) {
          const float p = p_s[t][cl], pu = pu_s[t][cl], dy = dy_s[t][cl];
          const float4 b4 = *reinterpret_cast<const float4*>(&b_s[t][NS * lane]), c4 = *reinterpret_cast<const float4*>(&c_s[t][NS * lane]);
          const float b[NS] = {b4.x, b4.y, b4.z, b4.w}, c[NS] = {c4.x, c4.y, c4.z, c4.w};
          const bool ends = t + 1 < L && ((cuts >> (t + 1)) & 1);   // h[t + 1] was cleared for the next step
          float bc[2 * NS], sy = 0.f, sb = 0.f, sa = 0.f;
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            const float eh = e[t][i] * h[t][i];
            const float behind = ends ? fmaf(pu, b[i], eh) : h[t + 1][i];
            const float gh = fmaf(c[i], dy, carry[i]);
            sy = fmaf(c[i], behind, sy);
            sb = fmaf(gh, b[i], sb);
            const float ge = gh * eh;
            sa = fmaf(ge, rate[i], sa);
            da[i] = fmaf(ge, p, da[i]);
            bc[i] = gh * pu;
            bc[NS + i] = behind * dy;
            carry[i] = (cuts >> t) & 1 ? 0.f : gh * e[t][i];
          }
          sums[t % GROUP][0] = sy;
          sums[t % GROUP][1] = sb;
          sums[t % GROUP][2] = sa;
          {   // over the warp's channels
            const int at = sum_lanes<2 * NS, BITS, 5>(bc);
            constexpr int LEFT = (2 * NS) >> (5 - BITS) ? (2 * NS) >> (5 - BITS) : 1;
            if (writes_sum<2 * NS, BITS, 5>()) {
#pragma unroll
              for (int k = 0; k < LEFT; ++k) {
                const int v = at + k;   // 0 .. 3: b, 4 .. 7: c
                red[(t * WARPS + warp) * 2 * NP + (v / NS) * NP + NS * lane + v % NS] = bc[k];
              }
            }
          }
          if (t % GROUP == 0) {   // over the channel's lanes
#pragma unroll
            for (int s = 0; s < 3; ++s) {
              float v[GROUP];
#pragma unroll
              for (int k = 0; k < GROUP; ++k) v[k] = sums[k][s];
              const int at = sum_lanes<GROUP, 0, BITS>(v);
              constexpr int LEFT = GROUP >> BITS ? GROUP >> BITS : 1;
              if (writes_sum<GROUP, 0, BITS>()) {
#pragma unroll
                for (int k = 0; k < LEFT; ++k) sum_s[t + at + k][s][cl] = v[k];
              }
            }
          }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int t = pt + k * KL;
          if (t >= L || !prepares || t0 + t >= live) continue;
          const float sy = sum_s[t][0][pc], sb = sum_s[t][1][pc], sa = sum_s[t][2][pc];
          const float dpt = fmaf(sa, 1.0f / LOG2E, sb * u_f[k]);
          const float draw = q.softplus ? dpt * sigmoid<T>(raw[k]) : dpt;
          dup[(t0 + t) * g.du.step] = from_f<T>(fmaf(sb, p_f[k], skip * dyv[k]));
          ddp[(t0 + t) * g.ddelta.step] = from_f<T>(draw);
          if (gated) dzp[(t0 + t) * g.dz.step] = from_f<T>(dgate[k] * fmaf(skip, u_f[k], sy));
          dd = fmaf(dyv[k], u_f[k], dd);
          dbias += draw;
        }
        for (int x = tid; x < L * 2 * NP; x += THREADS) {
          const int t = x / (2 * NP), s = x % (2 * NP);
          if (t0 + t >= live) break;
          float v = 0.f;
#pragma unroll
          for (int k = 0; k < WARPS; ++k) v += red[(t * WARPS + k) * 2 * NP + s];
          if (part_bc) part_bc[(t0 + t) * part_step + s] = v;
          else if (s < NP) { if (s < q.states) dbp[(t0 + t) * g.db.step + s] = from_f<T>(v); }
          else if (s - NP < q.states) dcp[(t0 + t) * g.dc.step + s - NP] = from_f<T>(v);
        }
        // the next chunk's sums are written behind its first barrier
      }
    }
    if constexpr (LOCAL) {
      if (owns) {
        store_states(w.carry + ((int64_t)split * q.rows * q.width + rc) * NP, carry, NS * lane, NP, true);
        if (lane == 0) w.sum_p[(int64_t)split * q.rows * q.width + rc] = sum_p;
      }
      if (tid == 0 && tile == 0) w.cut[(int64_t)split * q.rows + r] = any_cut;
    } else if (owns && split == 0 && g.dstate_in) {
      store_states(g.dstate_in + rc * q.states, carry, NS * lane, q.states, wide);
    }
  }
  if constexpr (!LOCAL) {
    const int64_t part = (int64_t)blockIdx.y * w.row_blocks + row_block;
    if (owns) store_states(w.part_a + (part * q.width + ch) * NP, da, NS * lane, NP, true);
    __syncthreads();
    float* both = &sum_s[0][0][0];   // (KL, 2, CT) of the threads that prepared a channel
    constexpr int HELD = KL > L ? L : KL;   // threads behind the eighth prepared nothing
    static_assert(sizeof(sum_s) >= HELD * 2 * CT * 4, "room for the sums of a channel");
    if (pt < HELD) {
      both[(pt * 2 + 0) * CT + pc] = dd;
      both[(pt * 2 + 1) * CT + pc] = dbias;
    }
    __syncthreads();
    if (pt < 2 || KL == 1) {
      for (int s = pt; s < 2; s += KL) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < HELD; ++k) v += both[(k * 2 + s) * CT + pc];
        if (prepares) w.part_d[(part * 2 + s) * q.width + c0 + pc] = v;
      }
    }
  }
}

// Gradients of a, d and the bias from the CTAs' sums: item i of `items` sums over `parts`; eight threads share it, in a fixed order.
__global__ void __launch_bounds__(256) k_param_sums(const float* part_a, const float* part_d, int parts, int width, int states, int padded,
                                                    float* da, float* dd, float* dbias) {
  __shared__ float sums[8][33];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t of_a = (int64_t)width * padded, items = of_a + 2 * (int64_t)width, i = (int64_t)blockIdx.x * 32 + lane;
  const float* src = i < of_a ? part_a + i : part_d + (i - of_a);
  const int64_t stride = i < of_a ? of_a : 2 * (int64_t)width;
  float v = 0.f;
  if (i < items)
    for (int k = q; k < parts; k += 8) v += src[k * stride];
  sums[q][lane] = v;
  __syncthreads();
  if (q || i >= items) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += sums[k][lane];
  if (i < of_a) {
    const int64_t c = i / padded;
    if (i - c * padded < states) da[c * states + (i - c * padded)] = v;
  } else if (i - of_a < width) {
    if (dd) dd[i - of_a] = v;
  } else if (dbias) {
    dbias[i - of_a - width] = v;
  }
}

// Gradients of b and c from the tiles of a group's channels.
template <typename T>
__global__ void __launch_bounds__(256) k_bc_sums(const float* part, int tiles, int steps, int rows, int groups, int states, int padded, BnbView db, BnbView dc) {
  const int64_t cells = (int64_t)steps * rows * groups * 2 * padded, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= cells) return;
  float v = 0.f;
  for (int k = 0; k < tiles; ++k) v += part[k * cells + i];
  const int s = (int)(i % (2 * padded)), n = s < padded ? s : s - padded;
  int64_t rest = i / (2 * padded);
  const int gr = (int)(rest % groups);
  rest /= groups;
  const int r = (int)(rest % rows), t = (int)(rest / rows);
  if (n >= states) return;
  const BnbView& o = s < padded ? db : dc;
  static_cast<T*>(o.data)[t * o.step + r * o.row + gr * o.group + n] = from_f<T>(v);
}

struct Plan {
  Splits splits;
  int kl, ct, tiles_a_group, tiles, row_blocks;
  size_t sum_p, cut, part_bc, part_a, part_d, total;   // offsets; the carries stand first
};
Plan plan_of(const BnbSelectiveScan& a) {
  Plan p{};
  p.kl = lanes_of(a.states);
  p.ct = p.kl <= 4 ? 64 : 256 / p.kl;   // CHANNELS
  p.tiles_a_group = (a.width / a.groups + p.ct - 1) / p.ct;
  p.tiles = p.tiles_a_group * a.groups;
  const int fit = 148 * 2;   // CTAs of 256 threads that the chip holds at 128 registers a thread
  p.splits = splits_of(a.steps, (int64_t)p.tiles * a.rows, fit);
  p.row_blocks = (int)std::min<int64_t>(a.rows, std::max<int64_t>(1, fit / ((int64_t)p.tiles * p.splits.count)));
  const size_t cells = (size_t)a.rows * a.width, np = (size_t)NS * p.kl, parts = (size_t)p.splits.count * p.row_blocks;
  size_t at = p.splits.count > 1 ? round256(p.splits.count * cells * np * 4) : 0;
  p.sum_p = at;
  if (p.splits.count > 1) at += round256(p.splits.count * cells * 4);
  p.cut = at;
  if (p.splits.count > 1) at += round256((size_t)p.splits.count * a.rows);
  p.part_bc = at;
  if (p.tiles_a_group > 1) at += round256((size_t)p.tiles_a_group * a.steps * a.rows * a.groups * 2 * np * 4);
  p.part_a = at;
  at += round256(parts * a.width * np * 4);
  p.part_d = at;
  p.total = at + round256(parts * 2 * a.width * 4);
  return p;
}

template <typename T, int KL>
int launch(const BnbSelectiveScan& a, const BnbSelectiveScanGrads& g, const Plan& p, uint8_t* scratch, cudaStream_t st) {
  constexpr int CT = CHANNELS<KL>, NP = NS * KL, WARPS = CT * KL / 32;
  constexpr size_t RED = (size_t)L * WARPS * 2 * NP * 4;   // at most 32 KB beside 17 KB of static shared memory
  Work w{};
  w.splits = p.splits;
  w.tiles_a_group = p.tiles_a_group;
  w.row_blocks = p.row_blocks;
  w.carry = reinterpret_cast<float*>(scratch);
  w.sum_p = reinterpret_cast<float*>(scratch + p.sum_p);
  w.cut = scratch + p.cut;
  w.part_bc = p.tiles_a_group > 1 ? reinterpret_cast<float*>(scratch + p.part_bc) : nullptr;
  w.part_a = reinterpret_cast<float*>(scratch + p.part_a);
  w.part_d = reinterpret_cast<float*>(scratch + p.part_d);
  const int64_t ctas = (int64_t)p.tiles * p.row_blocks;
  if (ctas > INT32_MAX || p.splits.count > 65535) return BNB_ERR_UNSUPPORTED_DIMS;
  const dim3 grid((unsigned)ctas, p.splits.count);
  if (cudaFuncSetAttribute(k_scan_bwd<T, KL, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)RED) != cudaSuccess) return BNB_ERR_LAUNCH;
  if (p.splits.count > 1) {
    count_launch();
    k_scan_bwd<T, KL, true><<<grid, CT * KL, 0, st>>>(a, g, w);
    const int64_t cells = (int64_t)a.rows * a.width * NP;
    count_launch();
    k_join<true><<<(unsigned)((cells + 255) / 256), 256, 0, st>>>(w.carry, w.sum_p, w.cut, a.a, g.dstate_out, p.splits.count, a.rows, a.width, a.states, NP);
  }
  count_launch();
  k_scan_bwd<T, KL, false><<<grid, CT * KL, RED, st>>>(a, g, w);
  count_launch();
  const int64_t items = (int64_t)a.width * NP + 2 * (int64_t)a.width;
  k_param_sums<<<(unsigned)((items + 31) / 32), 256, 0, st>>>(w.part_a, w.part_d, p.splits.count * p.row_blocks, a.width, a.states, NP, g.da, g.dd, g.ddelta_bias);
  if (w.part_bc && a.steps) {
    const int64_t cells = (int64_t)a.steps * a.rows * a.groups * 2 * NP;
    if ((cells + 255) / 256 > INT32_MAX) return BNB_ERR_UNSUPPORTED_DIMS;
    count_launch();
    k_bc_sums<T><<<(unsigned)((cells + 255) / 256), 256, 0, st>>>(w.part_bc, p.tiles_a_group, a.steps, a.rows, a.groups, a.states, NP, g.db, g.dc);
  }
  return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
}
template <typename T>
int run(const BnbSelectiveScan& a, const BnbSelectiveScanGrads& g, const Plan& p, uint8_t* scratch, cudaStream_t st) {
  switch (p.kl) {
    case 1: return launch<T, 1>(a, g, p, scratch, st);
    case 2: return launch<T, 2>(a, g, p, scratch, st);
    case 4: return launch<T, 4>(a, g, p, scratch, st);
    case 8: return launch<T, 8>(a, g, p, scratch, st);
    default: return launch<T, 16>(a, g, p, scratch, st);
  }
}

}  // namespace
}  // namespace scan
}  // namespace bnb

using namespace bnb;

extern "C" size_t bnb_selective_scan_bwd_scratch_bytes(const BnbSelectiveScan* a) {
  if (scan::check(a) || a->rows == 0 || a->width == 0) return 0;
  return scan::plan_of(*a).total;
}

extern "C" int bnb_selective_scan_bwd(const BnbSelectiveScan* a, const BnbSelectiveScanGrads* g, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int st = scan::check(a)) return st;
  if (!g) return BNB_ERR_NULL_POINTER;
  if (a->reset) return BNB_ERR_BAD_ARGUMENT;
  if (a->width == 0) return BNB_OK;
  if (!g->da) return BNB_ERR_NULL_POINTER;
  const auto s = static_cast<cudaStream_t>(stream);
  if (a->rows == 0) {
    bool ok = cudaMemsetAsync(g->da, 0, (size_t)a->width * a->states * 4, s) == cudaSuccess;
    if (g->dd) ok = ok && cudaMemsetAsync(g->dd, 0, (size_t)a->width * 4, s) == cudaSuccess;
    if (g->ddelta_bias) ok = ok && cudaMemsetAsync(g->ddelta_bias, 0, (size_t)a->width * 4, s) == cudaSuccess;
    return ok ? BNB_OK : BNB_ERR_LAUNCH;
  }
  if (a->steps && (!g->dy.data || !g->du.data || !g->ddelta.data || !g->db.data || !g->dc.data || (a->z.data && !g->dz.data) || !a->kept))
    return BNB_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(g->dstate_out) | reinterpret_cast<uintptr_t>(g->dstate_in)) & 15) return BNB_ERR_MISALIGNED;
  const scan::Plan p = scan::plan_of(*a);
  if (!scratch || scratch_bytes < p.total) return BNB_ERR_SCRATCH_TOO_SMALL;
  auto* at = static_cast<uint8_t*>(scratch);
  return a->element == BNB_ELEM_F32 ? scan::run<float>(*a, *g, p, at, s)
       : a->element == BNB_ELEM_BF16 ? scan::run<__nv_bfloat16>(*a, *g, p, at, s) : scan::run<__half>(*a, *g, p, at, s);
}
