// The selective state space recurrence, backward.  With dyv = dy silu(z), g_n the gradient of h_n behind a step and h- the state
// before it (after an episode end: 0):
//
//   g_n = carry_n + c_n dyv,   dc_n = sum_ch dyv h_n,   db_n = sum_ch g_n p u,   da_n = sum g_n e_n h-_n p,   carry_n = e_n g_n   (e_n = exp(p a_n))
//   du = p sum_n g_n b_n + d dyv,   dp = sum_n g_n e_n h-_n a_n + u sum_n g_n b_n,   ddelta = dp softplus'(delta + bias)
//   dz = dy (sum_n c_n h_n + d u) silu'(z),   dd = sum dyv u
//
// The forward kept the states of every eighth step.  A CTA takes the chunks of eight steps from the last to the first: the states of
// a chunk are computed forward into registers, and the adjoint walks back over them, with the decays once more.
//
// Sums over the channels (db, dc), 2 NS values a thread and step, are the most work of all if they go through shuffles: four instructions for
// each halving.  They are matrix products instead: D (16 x 8) += A (16 x 8) B (8 x 8) on mma.sync, where a warp's lanes hold four channels as the
// depth and (state lane, other channels) as the rows of A just as they are, db's values in its upper half and dc's in its lower, one
// state in the depths 0 .. 3 and a second one in 4 .. 7.  B has ones in a step's two columns, so that the accumulators of four steps are
// filled two columns after two.  (With the values in B, which holds half of what A does, twice the products were needed: 2030 us against
// 2020 at 32 steps x 8192 rows x 256 channels x 16 states in bfloat16, and more in float32, where there are twice as many.)
// The operands are pieces of the float32 values.  bfloat16 calls: two bfloat16 pieces, 2^-15 of a value at most from it, side by side in the depth of
// a 16 x 8 x 16 product.  Others: 11 bits and, in a product of its own, the 11 that follow.  (Rounded to 11 bits alone, a bfloat16 call
// took 2020 us, lost NaN, and was off by 2^-11 of a term where few channels share b and c; two products of 11 bits took 2190.)  An infinity
// becomes NaN: inf - inf remains of it, and it meets the zeros of the other columns.
//
// What is left of the sums over channels goes through the warps of the CTA and, where a group has several tiles of channels, a
// short kernel over the tiles; sums over rows and time (da, dd, d bias) stay in registers while a CTA goes over its rows.  No
// atomics, so a result does not depend on timing.
//
// Some 156 instructions for a warp's step of 8 channels x 16 states bound it (8 exponentials, 60 for the recurrence and its adjoint, 30 for db
// and dc, 12 for the sums over a channel's lanes, the rest per chunk), issued in 57 % of the cycles: at 128 registers a thread 16 warps fit on an
// SM.  2117 us at 32 steps x 8192 rows x 256 channels of bfloat16.  Registers decide what else may be tried: a version with 20 more values alive in
// the walk spilled, and took 2460 us when this one took 2020.
// Memory moves some 24 bytes a channel and step, 20 % of what it could.  The next chunk's operands therefore come by asynchronous
// copies into shared memory, which hold no register (2220 -> 2150 us).
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
  bool paired;       // pairs of channels of u, delta, z, dy and their gradients lie on their boundary
  bool paired_bc;    // and pairs of states of b and c
};

template <int KL> constexpr int CHANNELS = KL <= 4 ? 64 : 256 / KL;   // of a CTA

// d += what a lane holds of two states for db and for dc, in a step's columns; see above for what is where.  KEPT: the bits of a float's first piece.
template <uint32_t KEPT>
__device__ __forceinline__ F2 first_piece(F2 v) {
  const float2 s = halves(v);
  return f2(__uint_as_float(__float_as_uint(s.x) & KEPT), __uint_as_float(__float_as_uint(s.y) & KEPT));
}
__device__ __forceinline__ uint32_t pieces(float first, float rest) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(first), "f"(rest));
  return r;
}
__device__ __forceinline__ void mma_rows(float (&d)[4], float2 b, float2 c, const uint32_t (&one)[2]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(b.x)), "r"(__float_as_uint(c.x)), "r"(__float_as_uint(b.y)), "r"(__float_as_uint(c.y)), "r"(one[0]), "r"(one[1]));
}
template <typename T>
__device__ __forceinline__ void add_rows(float (&d)[4], F2 b, F2 c, const uint32_t (&one)[2]) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t KEPT = BF16 ? 0xffff0000u : 0xffffe000u;
  const F2 bh = first_piece<KEPT>(b), ch = first_piece<KEPT>(c);
  const float2 b1 = halves(bh), c1 = halves(ch), b2 = halves(fma(bh, f2(-1.0f), b)), c2 = halves(fma(ch, f2(-1.0f), c));
  if constexpr (BF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(pieces(b1.x, b2.x)), "r"(pieces(c1.x, c2.x)), "r"(pieces(b1.y, b2.y)), "r"(pieces(c1.y, c2.y)), "r"(one[0]), "r"(one[1]));
  } else {
    mma_rows(d, b2, c2, one);
    mma_rows(d, b1, c1, one);
  }
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(BYTES) : "memory");
}
// Two neighbouring elements, or those of `count` that exist and zeros: under way with one access where they lie on their boundary.
template <typename T>
__device__ __forceinline__ void copy_pair(Raw<T, 2>* to, const T* from, int count, bool paired) {
  if (paired && count == 2) copy_async<2 * sizeof(T)>(to, from);
  else *to = load_pair<T>(from, count, false);
}

// LOCAL: only what a split leaves of a zero adjoint behind it, see selective_scan.cuh.
template <typename T, int KL, bool LOCAL>
__global__ void __launch_bounds__(CHANNELS<KL> * KL, KL <= 4 ? 512 / (CHANNELS<KL> * KL) : 2) k_scan_bwd(const __grid_constant__ BnbSelectiveScan q, const __grid_constant__ BnbSelectiveScanGrads g, const __grid_constant__ Work w) {
  constexpr int CT = CHANNELS<KL>, THREADS = CT * KL, NP = NS * KL, WARPS = THREADS / 32;
  constexpr int BITS = KL == 1 ? 0 : KL == 2 ? 1 : KL == 4 ? 2 : KL == 8 ? 3 : 4, CB = 5 - BITS;   // lane: channel in the low CB bits, state lane above
  constexpr int PAIRS = CT / 2, AT_ONCE = THREADS / PAIRS < L ? THREADS / PAIRS : L, PER = L / AT_ONCE;   // steps prepared at a time, by a thread
  constexpr int GROUP = 2;         // steps whose sums over a channel's lanes are taken together: with 4, 6 more values live and spill
  constexpr bool MMA = KL <= 8;    // with 16 lanes a channel, four neighbouring lanes are not four channels
  constexpr int PARTS = MMA ? 8 / KL : 1, RED = PARTS * 2 * NP;   // sums over a part of a warp's channels, a step's of a warp
  __shared__ __align__(16) float4 pp_s[L][CT];                        // p, p, p u, p u
  __shared__ __align__(16) float2 dy_s[L][CT];                        // dyv twice
  __shared__ __align__(16) float b_s[LOCAL ? 1 : L][NP], c_s[L][NP];
  __shared__ __align__(16) float sum_s[LOCAL ? 1 : L][3][CT];
  __shared__ __align__(16) float held_s[LOCAL ? 1 : L][3][CT];        // u, softplus', dy silu'(z)
  // the next chunk, on its way while this one is computed: a thread copies what it reads itself
  constexpr int PREPARE = PAIRS * AT_ONCE, BC = (LOCAL ? 1 : 2) * L * NP / 2, BC_PER = (BC + THREADS - 1) / THREADS;
  __shared__ __align__(16) Raw<T, 2> next_s[PER][4][PREPARE], next_bc_s[BC_PER][THREADS];   // u, delta, z, dy; pairs of c, then of b
  __shared__ __align__(16) float4 next_h_s[LOCAL ? 1 : THREADS];
  extern __shared__ __align__(16) float red[];   // (L, WARPS, 2, PARTS, NP): sums over channels
  const int tid = threadIdx.x, warp = tid / 32, wl = tid & 31, lane = wl >> CB, cl = warp * (32 / KL) + (wl & ((1 << CB) - 1));
  const int tiles = w.tiles_a_group * q.groups, share = q.width / q.groups;
  const int row_block = blockIdx.x / tiles, tile = blockIdx.x - row_block * tiles, group = tile / w.tiles_a_group, tile_in = tile - group * w.tiles_a_group;
  const int c0 = group * share + tile_in * CT, c_end = min((group + 1) * share, c0 + CT);
  const int ch = c0 + cl;
  const bool owns = ch < c_end, wide = q.states % NS == 0;
  const int split = blockIdx.y, first = split * w.splits.steps, last = min(q.steps, first + w.splits.steps);

  F2 rate[2] = {f2(0.f), f2(0.f)}, da[2] = {f2(0.f), f2(0.f)};
  auto put = [](float (&v)[NS], const F2 (&x)[2]) {
    const float2 a = halves(x[0]), b = halves(x[1]);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  };
  auto get = [](F2 (&x)[2], const float (&v)[NS]) {
    x[0] = f2(v[0], v[1]);
    x[1] = f2(v[2], v[3]);
  };
  if (owns) {
    float v[NS];
    load_states(v, q.a + (int64_t)ch * q.states, NS * lane, q.states, wide && NS * lane < q.states);
    get(rate, v);
    rate[0] = mul(rate[0], f2(LOG2E));
    rate[1] = mul(rate[1], f2(LOG2E));
  }
  // what this thread prepares: channels c0 + 2 pair, + 1 of steps t0 + step + k AT_ONCE
  const int pair = tid % PAIRS, step = tid / PAIRS, pc = c0 + 2 * pair, count = step < L ? max(0, min(2, c_end - pc)) : 0;
  F2 bias = f2(0.f), skip = f2(0.f), dd = f2(0.f), dbias = f2(0.f);
  if (q.delta_bias) bias = f2(count > 0 ? q.delta_bias[pc] : 0.f, count > 1 ? q.delta_bias[pc + 1] : 0.f);
  if (q.d) skip = f2(count > 0 ? q.d[pc] : 0.f, count > 1 ? q.d[pc + 1] : 0.f);
  const bool gated = q.z.data != nullptr;
  const T none = from_f<T>(0.f);
  auto place = [&](const BnbView& v) { return step * v.step + pc; };
  // starts the copies of row r's chunk at t0, of which the steps before `live` exist
  auto fetch = [&](int r, int t0, int live) {
    auto at = [&](const BnbView& v, int t) { return static_cast<const T*>(v.data) + r * v.row + t * v.step; };
    if (step < AT_ONCE) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int tu = t0 + k * AT_ONCE, have = tu + step < live ? count : 0;
        if (!LOCAL) copy_pair(&next_s[k][0][tid], at(q.u, tu) + place(q.u), have, w.paired);
        copy_pair(&next_s[k][1][tid], at(q.delta, tu) + place(q.delta), have, w.paired);
        copy_pair(&next_s[k][2][tid], at(q.z, tu) + place(q.z), gated ? have : 0, w.paired);
        copy_pair(&next_s[k][3][tid], at(g.dy, tu) + place(g.dy), have, w.paired);
      }
    }
#pragma unroll
    for (int k = 0; k < BC_PER; ++k) {
      const int x = tid + k * THREADS, e = x % (L * NP / 2), t = e / (NP / 2), s = e % (NP / 2) * 2;
      const BnbView& v = x < L * NP / 2 ? q.c : q.b;
      if (x < BC) copy_pair(&next_bc_s[k][tid], at(v, t0 + t) + group * v.group + s, t0 + t < live ? max(0, min(2, q.states - s)) : 0, w.paired_bc);
    }
    if (!LOCAL && owns) copy_async<16>(&next_h_s[tid], q.kept + ((int64_t)(t0 / KEEP) * q.rows * q.width + (int64_t)r * q.width + ch) * NP + NS * lane);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // whether an episode ended before this lane's step of a chunk
  auto ended = [&](int r, int t0, int live) -> uint8_t {
    const int t = t0 + wl - 1;
    return q.done && wl < L && t >= 0 && t + 1 < live ? q.done[(int64_t)t * q.rows + r] : 0;
  };
  auto last_chunk = [&](int live) { return live > first ? (live - 1) / L * L : first - L; };   // first is a multiple of L
  if (!LOCAL && !owns) next_h_s[tid] = make_float4(0.f, 0.f, 0.f, 0.f);
  bool fetched = false;
  uint8_t ended_next = 0;
  int n_next = row_block < q.rows ? row_steps(q.lengths, row_block, q.steps) : 0;

  for (int r = row_block; r < q.rows; r += w.row_blocks) {
    const int n = n_next, live = min(n, last), r_next = r + w.row_blocks;
    if (r_next < q.rows) n_next = row_steps(q.lengths, r_next, q.steps);
    const int64_t rc = (int64_t)r * q.width + ch;
    const int begin = last_chunk(live);
    // A row's step: the same address for the whole CTA.  A thread's place from there is the same for every chunk.
    auto at = [&](const BnbView& v, int t) { return static_cast<T*>(v.data) + r * v.row + t * v.step; };
    auto db_at = [&](int t) { return at(g.db, t) + group * g.db.group; };
    auto dc_at = [&](int t) { return at(g.dc, t) + group * g.dc.group; };
    float* part_bc = w.part_bc ? w.part_bc + (((int64_t)tile_in * q.steps * q.rows + r) * q.groups + group) * 2 * NP : nullptr;
    const int64_t part_step = (int64_t)q.rows * q.groups * 2 * NP;

    // steps behind the row's end
    if constexpr (!LOCAL) {
      for (int t = max(first, n) + step; step < L && t < last; t += AT_ONCE) {
        store_pair(at(g.du, t) + pc, f2(0.f), count, w.paired);
        store_pair(at(g.ddelta, t) + pc, f2(0.f), count, w.paired);
        if (gated) store_pair(at(g.dz, t) + pc, f2(0.f), count, w.paired);
      }
      for (int64_t e = tid; e < (int64_t)(last - max(first, n)) * 2 * NP; e += THREADS) {
        const int t = max(first, n) + (int)(e / (2 * NP)), s = (int)(e % (2 * NP));
        if (part_bc) part_bc[t * part_step + s] = 0.f;
        else if (s < NP) { if (s < q.states) db_at(t)[s] = none; }
        else if (s - NP < q.states) dc_at(t)[s - NP] = none;
      }
    }

    F2 carry[2] = {f2(0.f), f2(0.f)};
    if (!LOCAL && owns) {
      float v[NS];
      clear_states(v);
      if (w.splits.count > 1) load_states(v, w.carry + ((int64_t)split * q.rows * q.width + rc) * NP, NS * lane, NP, true);
      else if (g.dstate_out) load_states(v, g.dstate_out + rc * q.states, NS * lane, q.states, wide && NS * lane < q.states);
      get(carry, v);
    }
    float sum_p = 0.f;
    bool any_cut = false;
    if (!fetched && begin >= first) {
      fetch(r, begin, live);
      ended_next = ended(r, begin, live);
    }
    fetched = false;
#pragma unroll 1
    for (int t0 = begin; t0 >= first; t0 -= L) {
      const unsigned cuts = __ballot_sync(0xffffffffu, ended_next != 0);   // bit k: an episode ended before step t0 + k
      asm volatile("cp.async.wait_all;" ::: "memory");
      const float4 h_r = LOCAL ? make_float4(0.f, 0.f, 0.f, 0.f) : next_h_s[LOCAL ? 0 : tid];
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        if (step >= AT_ONCE) continue;
        const int ts = step + k * AT_ONCE, t = t0 + ts;
        const Raw<T, 2> u_r = next_s[k][0][tid], d_r = next_s[k][1][tid], z_r = next_s[k][2][tid], y_r = next_s[k][3][tid];
        const F2 u = floats_of<T>(u_r), raw = add(floats_of<T>(d_r), bias), dy = floats_of<T>(y_r);
        const F2 p = t < live ? step_size(raw, q.softplus) : f2(0.f);
        F2 dyv = dy, dgate = f2(0.f);   // dgate: dy silu'(z)
        if (gated) {
          const F2 z = floats_of<T>(z_r), sg = sigmoid_pair<T>(z);
          dyv = mul(dy, mul(z, sg));
          dgate = mul(dy, mul(sg, fma(z, fma(sg, f2(-1.0f), f2(1.0f)), f2(1.0f))));
        }
        {
          const float2 ps = halves(p), pu = halves(mul(p, u)), ds = halves(dyv);
          pp_s[ts][2 * pair] = make_float4(ps.x, ps.x, pu.x, pu.x);
          pp_s[ts][2 * pair + 1] = make_float4(ps.y, ps.y, pu.y, pu.y);
          *reinterpret_cast<float4*>(&dy_s[ts][2 * pair]) = make_float4(ds.x, ds.x, ds.y, ds.y);
          if (!LOCAL) {   // for this thread's own use behind the walk
            const F2 slope = q.softplus ? sigmoid_pair<T>(raw) : f2(1.0f);
            *reinterpret_cast<float2*>(&held_s[ts][0][2 * pair]) = halves(u);
            *reinterpret_cast<float2*>(&held_s[ts][1][2 * pair]) = halves(slope);
            *reinterpret_cast<float2*>(&held_s[ts][2][2 * pair]) = halves(dgate);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < BC_PER; ++k) {
        const int x = tid + k * THREADS;
        if (x < BC) *reinterpret_cast<float2*>(x < L * NP / 2 ? &c_s[0][0] + 2 * x : &b_s[0][0] + 2 * x - L * NP) = halves(floats_of<T>(next_bc_s[k][tid]));
      }
      const F2 h0[2] = {f2(h_r.x, h_r.y), f2(h_r.z, h_r.w)};
      any_cut |= cuts != 0;
      __syncthreads();
      if (t0 > first) {
        fetch(r, t0 - L, live);
        ended_next = ended(r, t0 - L, live);
      } else if (r_next < q.rows) {
        const int of = min(n_next, last), begins = last_chunk(of);
        fetched = begins >= first;
        if (fetched) {
          fetch(r_next, begins, of);
          ended_next = ended(r_next, begins, of);
        }
      }
      if constexpr (LOCAL) {
#pragma unroll
        for (int t = L - 1; t >= 0; --t) {
          const F2 p{*reinterpret_cast<const unsigned long long*>(&pp_s[t][cl])}, dy{*reinterpret_cast<const unsigned long long*>(&dy_s[t][cl])};
          const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&c_s[t][NS * lane]);
          sum_p += halves(p).x;
          const float2 m0 = halves(mul(p, rate[0])), m1 = halves(mul(p, rate[1]));
          carry[0] = mul(f2(ex2_fast(m0.x), ex2_fast(m0.y)), fma(F2{c.x}, dy, carry[0]));
          carry[1] = mul(f2(ex2_fast(m1.x), ex2_fast(m1.y)), fma(F2{c.y}, dy, carry[1]));
          if ((cuts >> t) & 1) carry[0] = carry[1] = f2(0.f);
        }
        __syncthreads();
      } else {
        auto walk = [&](auto with_cuts) {
      constexpr bool cutting = decltype(with_cuts)::value;
        F2 h[L + 1][2];   // behind step t - 1
        h[0][0] = h0[0];
        h[0][1] = h0[1];
#pragma unroll
        for (int t = 0; t < L; ++t) {
          asm volatile("" ::: "memory");   // a step's loads stay in their step: with all in front, registers spill
          const ulonglong2 pp = *reinterpret_cast<const ulonglong2*>(&pp_s[t][cl]), b = *reinterpret_cast<const ulonglong2*>(&b_s[t][NS * lane]);
          const F2 bs[2] = {F2{b.x}, F2{b.y}};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 m = halves(mul(F2{pp.x}, rate[i]));
            h[t + 1][i] = fma(f2(ex2_fast(m.x), ex2_fast(m.y)), cutting && ((cuts >> t) & 1) ? f2(0.f) : h[t][i], mul(F2{pp.y}, bs[i]));
          }
        }
        struct Step { ulonglong2 pp, b, c; unsigned long long dy; };
        auto operands = [&](int t) -> Step {
          return {*reinterpret_cast<const ulonglong2*>(&pp_s[t][cl]), *reinterpret_cast<const ulonglong2*>(&b_s[t][NS * lane]),
                  *reinterpret_cast<const ulonglong2*>(&c_s[t][NS * lane]), *reinterpret_cast<const unsigned long long*>(&dy_s[t][cl])};
        };
        Step next = operands(L - 1);
        F2 da_chunk[2];         // summed by chunks first: one long sum of float32 loses a digit
        float rows[2][4], sums[GROUP][3];   // over the states: c h, g b, g e h- a
#pragma unroll
        for (int t = L - 1; t >= 0; --t) {
          asm volatile("" ::: "memory");
          const Step now = next;   // the step's operands came while the one behind it was computed
          if (t) next = operands(t - 1);
          const F2 p{now.pp.x}, pu{now.pp.y}, dy{now.dy};
          const F2 bs[2] = {F2{now.b.x}, F2{now.b.y}}, cs[2] = {F2{now.c.x}, F2{now.c.y}};
          F2 sy = f2(0.f), sb = f2(0.f), sa = f2(0.f);
          F2 of_b[2], of_c[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 m = halves(mul(p, rate[i]));
            const F2 e = f2(ex2_fast(m.x), ex2_fast(m.y)), eh = mul(e, cutting && ((cuts >> t) & 1) ? f2(0.f) : h[t][i]), behind = h[t + 1][i];
            const F2 gh = fma(cs[i], dy, carry[i]), ge = mul(gh, eh);
            sy = i ? fma(cs[i], behind, sy) : mul(cs[i], behind);
            sb = i ? fma(gh, bs[i], sb) : mul(gh, bs[i]);
            sa = i ? fma(ge, rate[i], sa) : mul(ge, rate[i]);
            da_chunk[i] = t == L - 1 ? mul(ge, p) : fma(ge, p, da_chunk[i]);
            of_b[i] = mul(gh, pu);
            of_c[i] = mul(behind, dy);
            carry[i] = mul(gh, e);
          }
          if (cutting && ((cuts >> t) & 1)) carry[0] = carry[1] = f2(0.f);
          const float2 y2 = halves(sy), b2 = halves(sb), a2 = halves(sa);
          sums[t % GROUP][0] = y2.x + y2.y;
          sums[t % GROUP][1] = b2.x + b2.y;
          sums[t % GROUP][2] = a2.x + a2.y;
          if (t % GROUP == 0) {   // over the channel's lanes
#pragma unroll
            for (int s = 0; s < 3; ++s) {
              float v[GROUP];
#pragma unroll
              for (int k = 0; k < GROUP; ++k) v[k] = sums[k][s];
              const int at = sum_lanes<GROUP, CB, 5>(v);
              constexpr int LEFT = GROUP >> BITS ? GROUP >> BITS : 1;
              if (writes_sum<GROUP, CB, 5>()) {
#pragma unroll
                for (int k = 0; k < LEFT; ++k) sum_s[t + at + k][s][cl] = v[k];
              }
            }
          }
          if constexpr (MMA) {
            constexpr uint32_t ONE = std::is_same<T, __nv_bfloat16>::value ? 0x3f803f80u : 0x3f800000u;   // for both pieces, or the one
            const uint32_t one[2] = {(wl >> 2) == 2 * (t % 4) ? ONE : 0u, (wl >> 2) == 2 * (t % 4) + 1 ? ONE : 0u};
            if (t % 4 == 3)
#pragma unroll
              for (int i = 0; i < 2; ++i) rows[i][0] = rows[i][1] = rows[i][2] = rows[i][3] = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) add_rows<T>(rows[i], of_b[i], of_c[i], one);
            if (t % 4 == 0) {   // this lane's sums are of step t + wl % 4 and of all four states of the state lane of row wl / 4
              const int g8 = wl >> 2;
              float* to = &red[((t + (wl & 3)) * WARPS + warp) * RED + (g8 % PARTS) * NP + g8 / PARTS * NS];
              *reinterpret_cast<float4*>(to) = make_float4(rows[0][0], rows[0][1], rows[1][0], rows[1][1]);
              *reinterpret_cast<float4*>(to + PARTS * NP) = make_float4(rows[0][2], rows[0][3], rows[1][2], rows[1][3]);
            }
          } else {   // over the warp's channels by shuffles
            float bc[2 * NS];
            put(*reinterpret_cast<float(*)[NS]>(&bc[0]), of_b);
            put(*reinterpret_cast<float(*)[NS]>(&bc[NS]), of_c);
            const int at = sum_lanes<2 * NS, 0, CB>(bc);
            constexpr int LEFT = (2 * NS) >> CB ? (2 * NS) >> CB : 1;
            if (writes_sum<2 * NS, 0, CB>()) {
#pragma unroll
              for (int k = 0; k < LEFT; ++k) {
                const int v = at + k;   // 0 .. 3: b, 4 .. 7: c
                red[(t * WARPS + warp) * RED + (v / NS) * NP + NS * lane + v % NS] = bc[k];
              }
            }
          }
        }
        da[0] = add(da[0], da_chunk[0]);
        da[1] = add(da[1], da_chunk[1]);
        };
        // ends of episodes are rare: without any, the steps are one run of instructions
        if (cuts) walk(std::true_type{});
        else walk(std::false_type{});
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int t = step + k * AT_ONCE;
          if (step >= L || t0 + t >= live) continue;
          auto pair_of = [&](const float* at) { const float2 v = *reinterpret_cast<const float2*>(at); return f2(v.x, v.y); };
          const F2 sy = pair_of(&sum_s[t][0][2 * pair]), sb = pair_of(&sum_s[t][1][2 * pair]), sa = pair_of(&sum_s[t][2][2 * pair]);
          const F2 u = pair_of(&held_s[t][0][2 * pair]), slope = pair_of(&held_s[t][1][2 * pair]), dgate = pair_of(&held_s[t][2][2 * pair]);
          const F2 p = f2(pp_s[t][2 * pair].x, pp_s[t][2 * pair + 1].x), dyv = f2(dy_s[t][2 * pair].x, dy_s[t][2 * pair + 1].x);
          const F2 draw = mul(fma(sa, f2(1.0f / LOG2E), mul(sb, u)), slope);
          store_pair(at(g.du, t0 + k * AT_ONCE) + place(g.du), fma(sb, p, mul(skip, dyv)), count, w.paired);
          store_pair(at(g.ddelta, t0 + k * AT_ONCE) + place(g.ddelta), draw, count, w.paired);
          if (gated) store_pair(at(g.dz, t0 + k * AT_ONCE) + place(g.dz), mul(dgate, fma(skip, u, sy)), count, w.paired);
          dd = fma(dyv, u, dd);
          dbias = add(dbias, draw);
        }
        for (int x = tid; x < L * 2 * NP; x += THREADS) {
          const int t = x / (2 * NP), s = x % (2 * NP);
          if (t0 + t >= live) break;
          float v = 0.f;
#pragma unroll
          for (int k = 0; k < WARPS * PARTS; ++k)   // dc's parts in another order than db's, for the banks
            v += red[(t * WARPS + k / PARTS) * RED + (s < NP ? 0 : PARTS * NP) + ((k % PARTS) ^ (s < NP || PARTS == 1 ? 0 : 1)) * NP + s % NP];
          if (part_bc) part_bc[(t0 + t) * part_step + s] = v;
          else if (s < NP) { if (s < q.states) db_at(t0 + t)[s] = from_f<T>(v); }
          else if (s - NP < q.states) dc_at(t0 + t)[s - NP] = from_f<T>(v);
        }
        // the next chunk's sums are written behind its first barrier; what a thread prepared it reads itself
      }
    }
    float v[NS];
    put(v, carry);
    if constexpr (LOCAL) {
      if (owns) {
        store_states(w.carry + ((int64_t)split * q.rows * q.width + rc) * NP, v, NS * lane, NP, true);
        if (lane == 0) w.sum_p[(int64_t)split * q.rows * q.width + rc] = sum_p;
      }
      if (tid == 0 && tile == 0) w.cut[(int64_t)split * q.rows + r] = any_cut;
    } else if (owns && split == 0 && g.dstate_in) {
      store_states(g.dstate_in + rc * q.states, v, NS * lane, q.states, wide && NS * lane < q.states);
    }
  }
  if constexpr (!LOCAL) {
    const int64_t part = (int64_t)blockIdx.y * w.row_blocks + row_block;
    float v[NS];
    put(v, da);
    if (owns) store_states(w.part_a + (part * q.width + ch) * NP, v, NS * lane, NP, true);
    __syncthreads();
    float* both = &sum_s[0][0][0];   // (AT_ONCE, 2, CT) of the threads that prepared a pair
    static_assert(sizeof(sum_s) >= AT_ONCE * 2 * CT * 4, "room for the sums of a channel");
    if (step < AT_ONCE) {
      *reinterpret_cast<float2*>(&both[(step * 2 + 0) * CT + 2 * pair]) = halves(dd);
      *reinterpret_cast<float2*>(&both[(step * 2 + 1) * CT + 2 * pair]) = halves(dbias);
    }
    __syncthreads();
    for (int x = tid; x < 2 * CT; x += THREADS) {
      const int s = x / CT, c = x % CT;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) sum += both[(k * 2 + s) * CT + c];
      if (c0 + c < c_end) w.part_d[(part * 2 + s) * q.width + c0 + c] = sum;
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

// Gradients of b and c from the tiles of a group's channels, four states a thread (padded is a multiple of four and a power of two, so the
// only division that is left is the one by the groups; with an element a thread and 64-bit divisions it took 75 us, not 26).
// A step takes `blocks` blocks of the grid.  Those are for 134 MB, 32 steps x 8192 rows x 16 states from four tiles: 5.2 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) k_bc_sums(const float* part, int tiles, int steps, int rows, int groups, int states, int shift, unsigned blocks, BnbView db, BnbView dc) {
  const unsigned t = blockIdx.x / blocks;
  const int64_t j = (int64_t)(blockIdx.x - t * blocks) * 256 + threadIdx.x, of_step = (int64_t)rows * groups << (shift - 2);
  if (j >= of_step) return;
  const float4* at = reinterpret_cast<const float4*>(part) + t * of_step + j;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < tiles; ++k) {
    const float4 x = at[k * steps * of_step];
    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
  }
  const int s = (int)(j & ((1 << (shift - 2)) - 1)) * 4, padded = 1 << (shift - 1), n = s & (padded - 1);
  const int64_t cell = j >> (shift - 2), r = groups == 1 ? cell : cell / groups;
  const BnbView& o = s < padded ? db : dc;
  T* to = static_cast<T*>(o.data) + t * o.step + r * o.row + (cell - r * groups) * o.group + n;
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < states) to[i] = from_f<T>(f[i]);
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
  // CTAs that the chip holds: at 128 registers a thread 512 threads of an SM, with one lane a channel as many as shared memory has room for. (With two
  // of every size on an SM, 32 steps x 4096 rows x 256 channels of bfloat16 took 947 us backward at 4 states and 738 at 8, now 561 and 589.)
  const int fit = 148 * (p.kl == 1 ? 5 : p.kl == 2 ? 4 : 2);
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
  constexpr size_t RED = (size_t)L * WARPS * 2 * (NP < 32 ? 32 : NP) * 4;   // at most 32 KB, beside 40 KB of static shared memory
  Work w{};
  w.splits = p.splits;
  w.tiles_a_group = p.tiles_a_group;
  w.row_blocks = p.row_blocks;
  w.paired = a.width / a.groups % 2 == 0 && even_view(a.u, a.element) && even_view(a.delta, a.element) && even_view(g.dy, a.element) &&
             even_view(g.du, a.element) && even_view(g.ddelta, a.element) && (!a.z.data || (even_view(a.z, a.element) && even_view(g.dz, a.element)));
  w.paired_bc = even_view(a.b, a.element) && even_view(a.c, a.element) && a.b.group % 2 == 0 && a.c.group % 2 == 0;
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
    int shift = 3;
    while (1 << shift < 2 * NP) ++shift;
    const int64_t blocks = (((int64_t)a.rows * a.groups << (shift - 2)) + 255) / 256;
    if (blocks * a.steps > INT32_MAX) return BNB_ERR_UNSUPPORTED_DIMS;
    count_launch();
    k_bc_sums<T><<<(unsigned)(blocks * a.steps), 256, 0, st>>>(w.part_bc, p.tiles_a_group, a.steps, a.rows, a.groups, a.states, shift, (unsigned)blocks, g.db, g.dc);
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
