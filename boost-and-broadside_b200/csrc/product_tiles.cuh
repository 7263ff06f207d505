// Matrix products on tcgen05 tiles for operands of any size, with the epilogues of the gated feed-forward block fused
// into them (gated_mlp.cu).
//
// out (m, n) = sum over terms of A_t (m, k) B_t (n, k)^T.  One persistent CTA per SM walks over tiles of 128 x BN; a warp fetches (TMA
// boxes of 64 elements by 64 to 256, 128-byte swizzle, zeros outside the tensors, so that no size has to be a multiple of a
// tile), a warp issues the products, sixteen warps take finished accumulators out of tensor memory.  There are two accumulators: a tile's
// products run while the tile before is written out.
//
// An operand may lie in memory with its depth innermost (K-major) or with its rows innermost (MN-major): the same boxes, other descriptor
// bits.  So no operand of the backward is transposed in memory.
//
// 16-bit operands take one term.  Float32 ones are split into three bfloat16 pieces whose sum is exact to 24 bits, and the
// product into the six products of pieces that are not below 2^-24 of it, smallest first: six terms of the same loop.  The tensor cores
// truncate every addition to an accumulator, 2^-25 of it on average and always towards zero; so the last term, the only one of full size, is
// cut into runs of FLUSH stages (16 additions), and the runs are added, rounded, by the warps that take results out.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "launch_after.h"
#include "tile_rows.cuh"

namespace bnb {
namespace product {

using namespace tensor;

constexpr int BM = 128, BK = 64;              // tile rows; depth of a stage
constexpr int MAX_TERMS = 12;                 // two segments of six
constexpr int FLUSH = 4;                      // stages of a run
constexpr int OUT_WARPS = 16, CTA = 32 * (2 + OUT_WARPS);
constexpr uint32_t OUT_BYTES = OUT_WARPS * 2048;   // shared memory of the results on their way out
constexpr uint32_t A_BYTES = BM * BK * 2, SLAB = 64 * BK * 2;   // SLAB: 64 rows or columns by 64
enum : int { W_FULL = 101, W_EMPTY = 102, W_ACC = 103, W_DRAINED = 104 };

// What a tile's results become.
//   VALUES   out[job] (m, n), of type `out_kind`
//   PARTIAL  float32 sums of a part of the depth: part (splits, jobs, m, n)
//   GATE     columns come in pairs of tiles, g and u: h = act(g) u as operand pieces; g and u themselves where they are kept
//   BACK     columns are dh: dg = dh u act'(g), du = dh act(g), h = act(g) u as operand pieces, from the kept g and u
//   AGAIN    the same with g and u computed once more: a stage holds x and dy, and 64 columns of all three weights
enum class Out : int { VALUES, PARTIAL, GATE, BACK, AGAIN };

struct Epilogue {
  void* out[2];
  float* part;
  void* h;              // operand pieces (pieces, m, ld_h)
  void* dg;
  void* du;
  float* g;             // kept: blocks of 32 rows by 32 columns, see kept_at
  float* u;
  int64_t ld_out, ld_h, piece_stride;
  int out_kind;         // 0: float32, 1: the operands' type
  int activation;       // BNB_ACT_SILU or BNB_ACT_GELU
};

struct Product {
  CUtensorMap a[2], b[3];
  Epilogue e;
  int64_t m;
  int n, k_steps, terms;       // k_steps: stages of a term
  int jobs, splits, split_steps;   // jobs: outputs a[j] b[0]; split_steps: stages (over all terms) of a split
  int m_tiles, n_tiles;
  uint8_t a_map[MAX_TERMS], b_map[MAX_TERMS], a_piece[MAX_TERMS], b_piece[MAX_TERMS];
  int* host_status;
};

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

struct Tile { int job, split, m, n; };
// Neighbouring CTAs take tiles of up to 16 row tiles by as many column tiles as it takes: their operands come from L2.
__device__ __forceinline__ Tile tile_of(const Product& p, int i) {
  constexpr int GM = 16;
  const int per = p.m_tiles * p.n_tiles, js = i / per, rest = i - js * per;
  const int g = rest / (GM * p.n_tiles), in = rest - g * GM * p.n_tiles, first = g * GM, gm = min(GM, p.m_tiles - first);
  return {js % p.jobs, js / p.jobs, first + in % gm, in / gm};
}

constexpr int MAX_STAGES = 8;
struct Frame2 {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc[2], drained[2];
  alignas(8) int aborted[4];   // see mbar_wait: the last two hold an address
  int status;
  uint32_t tmem;
};

// act(g) and, where wanted, act'(g) of neighbouring columns, two in an instruction.  e^(-g^2/2) serves the distribution function and its
// density.  16-bit results: that function as 1/2 + sign(g) (1/2 - tail), the tail by the approximation 7.1.26 of Abramowitz and Stegun's
// Handbook (absolute error 1.5e-7); float32: by erff.  With one element at a time and divisions that scale, 38 instructions an element
// instead of 14.
template <bool SLOPE>
__device__ __forceinline__ void activate_pair(int kind, F2 g, F2& a, F2& da) {
  const float2 gs = halves(g);
  if (kind == BNB_ACT_SILU) {
    const float2 m = halves(mul(g, f2(-1.4426950408889634f))), den = halves(add(f2(ex2_fast(m.x), ex2_fast(m.y)), f2(1.0f)));
    const F2 s = f2(rcp_fast(den.x), rcp_fast(den.y));
    a = mul(g, s);
    if (SLOPE) da = mul(s, fma(g, fma(s, f2(-1.0f), f2(1.0f)), f2(1.0f)));
    return;
  }
  const float2 den = halves(fma(f2(fabsf(gs.x), fabsf(gs.y)), f2(0.3275911f * 0.70710678118654752440f), f2(1.0f)));
  const float2 m = halves(mul(mul(g, g), f2(-0.5f * 1.4426950408889634f)));
  const F2 t = f2(rcp_fast(den.x), rcp_fast(den.y)), q = f2(ex2_fast(m.x), ex2_fast(m.y));
  F2 poly = fma(t, f2(-0.5f * 1.061405429f), f2(0.5f * 1.453152027f));   // half of the series, negative
  poly = fma(t, poly, f2(-0.5f * 1.421413741f));
  poly = fma(t, poly, f2(0.5f * 0.284496736f));
  poly = fma(t, poly, f2(-0.5f * 0.254829592f));
  const float2 rest = halves(fma(mul(t, poly), q, f2(0.5f)));   // 1/2 - tail
  const F2 cdf = add(f2(copysignf(rest.x, gs.x), copysignf(rest.y, gs.y)), f2(0.5f));
  a = mul(g, cdf);
  if (SLOPE) da = fma(mul(g, q), f2(0.39894228040143267794f), cdf);
}
__device__ __forceinline__ void activate_exact(int kind, float g, float& a, float& da) {
  if (kind == BNB_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-g));
    a = g * s;
    da = s * fmaf(g, 1.0f - s, 1.0f);
  } else {
    const float cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752440f));
    a = g * cdf;
    da = fmaf(g * 0.39894228040143267794f, expf(-0.5f * g * g), cdf);
  }
}
template <bool EXACT, bool SLOPE>
__device__ __forceinline__ void activate(int kind, F2 g, F2& a, F2& da) {
  if constexpr (EXACT) {
    const float2 gs = halves(g);
    float2 v, d;
    activate_exact(kind, gs.x, v.x, d.x);
    activate_exact(kind, gs.y, v.y, d.y);
    a = f2(v.x, v.y);
    da = f2(d.x, d.y);
  } else {
    activate_pair<SLOPE>(kind, g, a, da);
  }
}

__device__ __forceinline__ uint32_t pair_of(float a, float b, __nv_bfloat16) { return pack_bf16(a, b); }
__device__ __forceinline__ uint32_t pair_of(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename E> __device__ __forceinline__ uint32_t pair_of(F2 v) {
  const float2 f = halves(v);
  return pair_of(f.x, f.y, E{});
}
__device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ void down(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void down(__half& o, float v) { o = __float2half_rn(v); }
__device__ __forceinline__ void down(float& o, float v) { o = v; }

// The operand pieces of eight values: one rounding, or three bfloat16 numbers that add up to the value.
template <typename E, int PIECES>
__device__ __forceinline__ void put_operand(void* base, int64_t piece_stride, int64_t at, float (&v)[8]) {
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    *reinterpret_cast<uint4*>(static_cast<E*>(base) + p * piece_stride + at) =
        make_uint4(pair_of(v[0], v[1], E{}), pair_of(v[2], v[3], E{}), pair_of(v[4], v[5], E{}), pair_of(v[6], v[7], E{}));
    if constexpr (PIECES > 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        E r;
        down(r, v[i]);
        v[i] -= up(r);
      }
    }
  }
}

template <typename E> struct Format { static constexpr uint32_t BITS = 0; };
template <> struct Format<__nv_bfloat16> { static constexpr uint32_t BITS = (1u << 7) | (1u << 10); };

template <int BN, Out OUT>
struct Shape {
  static constexpr uint32_t B_BYTES = BN * BK * 2, STAGE = (OUT == Out::AGAIN ? 2 : 1) * A_BYTES + B_BYTES;
  static constexpr int COLS = OUT == Out::GATE ? BN / 2 : OUT == Out::AGAIN ? BN / 3 : BN;   // of the output
  static constexpr int FIT = (int)((227 * 1024 - 1024 - sizeof(Frame2) - OUT_BYTES) / STAGE), STAGES = FIT < MAX_STAGES ? FIT : MAX_STAGES;
  static constexpr uint32_t OUT_AT = STAGES * STAGE, FRAME = OUT_AT + OUT_BYTES, BYTES = FRAME + sizeof(Frame2) + 1024;   // 1024: to the swizzle's boundary
};

// Results to memory: 32 rows of 64 columns at a time, a row a lane of PARTS warps.  A request that writes a little of many rows costs the load
// and store unit as much as one that writes whole lines of each (32 bytes of 16 rows: 16 of its cycles, 128 bytes of 4 rows: 4).  So
// the warps of the same rows put 16-bit results together in shared memory (rows of 128 bytes, the 16-byte pieces swizzled so that
// neither side meets a bank twice), then each writes whole rows: f(row, column, 16 bytes).
__device__ __forceinline__ uint32_t row_piece(int r, int q) { return r * 128 + ((q ^ (r & 7)) << 4); }
template <int PARTS>
__device__ __forceinline__ void put_columns(uint8_t* rows, int part, int lane, const uint32_t (&v)[32 / PARTS]) {
#pragma unroll
  for (int q = 0; q < 8 / PARTS; ++q)
    *reinterpret_cast<uint4*>(rows + row_piece(lane, part * (8 / PARTS) + q)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}
template <int PARTS, class F>
__device__ __forceinline__ void take_rows(const uint8_t* rows, int part, int lane, F f) {
#pragma unroll
  for (int i = 0; i < 8 / PARTS; ++i) {
    const int r = (32 / PARTS) * part + i * 4 + lane / 8, q = lane % 8;
    f(r, 8 * q, *reinterpret_cast<const uint4*>(rows + row_piece(r, q)));
  }
}
// Float32: a warp for itself, 16 columns at a time.
template <class F>
__device__ __forceinline__ void emit_floats(uint8_t* stage, int lane, const uint32_t (&v)[16], F f) {
  auto at = [](int r, int q) { return r * 64 + ((q ^ ((r >> 1) & 3)) << 4); };
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(stage + at(lane, q)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + lane / 4, q = lane % 4;
    f(r, 4 * q, *reinterpret_cast<const uint4*>(stage + at(r, q)));
  }
}
// The 16 bytes of a row from column `col` on: whole where they may be, else element by element up to `cols`.
template <typename E>
__device__ __forceinline__ void put16(E* row, int col, int cols, bool wide, uint4 raw) {
  constexpr int N = 16 / sizeof(E);
  if (wide && col + N <= cols) {
    *reinterpret_cast<uint4*>(row + col) = raw;
  } else {
    const E* e = reinterpret_cast<const E*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) if (col + i < cols) row[col + i] = e[i];
  }
}

// Sixteen warps take out in two groups, tiles in turn: while one group waits for accumulators, for its rows or for memory, the other
// computes.  (All sixteen on a tile at once wait together: 71 us for dh and its gradients at 65 536 x 128 x 512.)  Float32, whose runs need both
// sets of accumulators for one tile, has one group, and so has BACK: it waits for g and u from memory most, and 16 columns a warp leave
// the registers to have all of a segment's on their way at once (128 us against 113 at 8192 x 1024 x 4096).
template <typename E, int PIECES, bool A_MN, bool B_MN, int BN, Out OUT>
__global__ void __launch_bounds__(CTA, 1) k_product(const __grid_constant__ Product p) {
  using S = Shape<BN, OUT>;
  constexpr bool EXACT = PIECES > 1;
  constexpr int GROUPS = EXACT || OUT == Out::BACK ? 1 : 2, PARTS = OUT_WARPS / 4 / GROUPS;
  static_assert(!EXACT || 3 * BN <= 512, "two sets of accumulators and their sum");
  constexpr uint32_t SUM = 2 * BN;   // float32: where runs are added
  extern __shared__ uint8_t raw_smem[];
  uint8_t* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  Frame2& f = *reinterpret_cast<Frame2*>(smem + S::FRAME);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    f.aborted[0] = 0;
    f.aborted[1] = DEFAULT_POLL_LIMIT;
    *reinterpret_cast<int**>(&f.aborted[2]) = p.host_status;
    f.status = 0;
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(smem_u32(&f.full[i]), 1);
      mbar_init(smem_u32(&f.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&f.acc[i]), 1);
      mbar_init(smem_u32(&f.drained[i]), OUT_WARPS / GROUPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(smem_u32(&f.tmem), 512);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_next_start();
  wait_for_previous();
  const uint32_t tmem = f.tmem, base = smem_u32(smem);
  auto wait = [&](uint64_t& bar, uint32_t parity, int code) { mbar_wait(smem_u32(&bar), parity & 1u, &f.status, f.aborted, code); };
  const int tiles = p.m_tiles * p.n_tiles * p.jobs * p.splits, all_steps = p.k_steps * p.terms;
  // The end of the run of stages that begins at s: all of a tile's, or, in float32, all of the small terms, then FLUSH at a time.
  const int small = EXACT ? all_steps - all_steps / 6 : all_steps;
  auto run_end = [&](int s, int s1) { return !EXACT ? s1 : s < small ? min(s1, small) : min(s1, s + FLUSH); };

  if (warp == 0) {
    // fetching
    int step = 0;
    const uint32_t el = elect_one();
    for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
      const Tile t = tile_of(p, i);
      const int s0 = t.split * p.split_steps, s1 = min(all_steps, s0 + p.split_steps);
      int term = s0 / p.k_steps, k = s0 - term * p.k_steps;
      const int m0 = t.m * BM, n0 = t.n * S::COLS;
      for (int s = s0; s < s1; ++s, ++step) {
        const int slot = step % S::STAGES;
        if (step >= S::STAGES) wait(f.empty[slot], step / S::STAGES - 1, W_EMPTY);
        if (el) {
          const uint32_t bar = smem_u32(&f.full[slot]), at = base + slot * S::STAGE;
          const CUtensorMap* am = &p.a[p.jobs > 1 ? t.job : p.a_map[term]];
          const CUtensorMap* bm = &p.b[p.b_map[term]];
          const int ap = p.a_piece[term], bp = p.b_piece[term], kc = k * BK;
          mbar_expect_tx(bar, S::STAGE);
          if constexpr (OUT == Out::AGAIN) {
            tma_load(at, &p.a[0], kc, m0, 0, bar);
            tma_load(at + A_BYTES, &p.a[1], kc, m0, 0, bar);
#pragma unroll
            for (int j = 0; j < 2; ++j) tma_load(at + 2 * A_BYTES + j * SLAB, &p.b[j], kc, n0, 0, bar);
            tma_load(at + 2 * A_BYTES + 2 * SLAB, &p.b[2], n0, kc, 0, bar);
          } else {
            const uint32_t bt = at + A_BYTES;
            if constexpr (A_MN) {
#pragma unroll
              for (int j = 0; j < BM / 64; ++j) tma_load(at + j * SLAB, am, m0 + 64 * j, kc, ap, bar);
            } else {
              tma_load(at, am, kc, m0, ap, bar);
            }
            if constexpr (OUT == Out::GATE) {
              tma_load(bt, &p.b[0], kc, n0, bp, bar);
              tma_load(bt + S::B_BYTES / 2, &p.b[1], kc, n0, bp, bar);
            } else if constexpr (B_MN) {
#pragma unroll
              for (int j = 0; j < BN / 64; ++j) tma_load(bt + j * SLAB, bm, n0 + 64 * j, kc, bp, bar);
            } else {
              tma_load(bt, bm, kc, n0, bp, bar);
            }
          }
        }
        __syncwarp();
        if (++k == p.k_steps) k = 0, ++term;
      }
    }
    // every copy has landed before the CTA may leave
    for (int s = max(0, step - S::STAGES); s < step; ++s) wait(f.full[s % S::STAGES], s / S::STAGES, W_FULL);
  } else if (warp == 1) {
    // issuing
    constexpr uint32_t COMMON = (1u << 4) | Format<E>::BITS | ((uint32_t)(BM >> 4) << 24);
    constexpr uint32_t MN_A = 1u << 15, MN_B = 1u << 16;
    constexpr uint32_t A_K = A_MN ? 128 : 2, B_K = B_MN ? 128 : 2;   // 16 of depth in descriptor units (16 bytes)
    const uint32_t el = elect_one(), tm = uniform(tmem);
    auto low = [](uint32_t addr, bool mn) { return ((addr & 0x3FFFFu) >> 4) | (mn ? (SLAB >> 4) << 16 : 1u << 16); };
    int step = 0, done = 0;
    for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
      const Tile t = tile_of(p, i);
      const int s0 = t.split * p.split_steps, s1 = min(all_steps, s0 + p.split_steps);
      for (int s = s0; s < s1; ++done) {
        const int set = done & 1, end = run_end(s, s1);
        if (done >= 2) wait(f.drained[set], done / 2 - 1, W_DRAINED);
        tc_fence_after();
        for (uint32_t acc = 0; s < end; ++s, ++step, acc = 1) {
          const int slot = step % S::STAGES;
          wait(f.full[slot], step / S::STAGES, W_FULL);
          tc_fence_after();
          const uint32_t at = base + slot * S::STAGE;
          if constexpr (OUT == Out::AGAIN) {
            const uint32_t x = uniform(low(at, false)), dy = uniform(low(at + A_BYTES, false)), w = uniform(low(at + 2 * A_BYTES, false)),
                           d = uniform(low(at + 2 * A_BYTES + 2 * SLAB, true));
#pragma unroll
            for (uint32_t k = 0; k < BK / 16; ++k)
              mma_one<false>(el, tm + set * BN, x + 2 * k, w + 2 * k, COMMON | ((uint32_t)(128 >> 3) << 17), acc || k ? 1u : 0u);
#pragma unroll
            for (uint32_t k = 0; k < BK / 16; ++k)
              mma_one<false>(el, tm + set * BN + 128, dy + 2 * k, d + 128 * k, COMMON | ((uint32_t)(64 >> 3) << 17) | MN_B, acc || k ? 1u : 0u);
          } else {
            constexpr uint32_t IDESC = COMMON | ((uint32_t)(BN >> 3) << 17) | (A_MN ? MN_A : 0u) | (B_MN ? MN_B : 0u);
            const uint32_t a_lo = uniform(low(at, A_MN)), b_lo = uniform(low(at + A_BYTES, B_MN));
#pragma unroll
            for (uint32_t k = 0; k < BK / 16; ++k)
              mma_one<false>(el, tm + set * BN, a_lo + A_K * k, b_lo + B_K * k, IDESC, acc || k ? 1u : 0u);
          }
          tc_commit_if(el, smem_u32(&f.empty[slot]));
        }
        tc_commit_if(el, smem_u32(&f.acc[set]));
        __syncwarp();
      }
    }
  } else {
    // taking out: this warp's 32 rows (a quarter of tensor memory is a warp's by its number) and a part of every 64 columns
    constexpr int SEG = 64 / PARTS;   // columns of a warp among 64
    const int quarter = warp & 3, group = ((warp - 2) >> 2) % GROUPS, part = ((warp - 2) >> 2) / GROUPS;
    uint8_t* rows = smem + S::OUT_AT + quarter * 8192 + group * 4096;      // of the warps that share rows
    uint8_t* stage = smem + S::OUT_AT + (warp - 2) * 2048;                  // of this one
    auto meet = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + quarter * GROUPS + group), "n"(32 * PARTS) : "memory"); };
    const Epilogue& e = p.e;
    const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16);
    auto release = [&](int set) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&f.drained[set]));
    };
    auto pair = [](const uint32_t (&v)[8], int k) { return f2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])); };
    int done = group, turn = 0;
    for (int i = blockIdx.x + group * gridDim.x; i < tiles; i += GROUPS * gridDim.x) {
      const Tile t = tile_of(p, i);
      uint32_t acc = lanes + (done & 1) * BN;
      if constexpr (EXACT) {
        const int s0 = t.split * p.split_steps, s1 = min(all_steps, s0 + p.split_steps);
        for (int s = s0; s < s1; ++done) {
          const int set = done & 1;
          wait(f.acc[set], done / 2, W_ACC);
          tc_fence_after();
          // the columns that this warp takes out below
#pragma unroll 1
          for (int k0 = 0; k0 < BN / PARTS; k0 += 8) {
            uint32_t v[8], w[8];
            const int c = (k0 / SEG) * 64 + part * SEG + k0 % SEG;
            tmem_ld8_nowait(lanes + set * BN + c, v);
            if (s > s0) tmem_ld8_nowait(lanes + SUM + c, w);
            tmem_wait_ld();
            if (s > s0)
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) + __uint_as_float(w[k]));
            tmem_st8_nowait(lanes + SUM + c, v);
          }
          tmem_wait_st();
          release(set);
          s = run_end(s, s1);
        }
        acc = lanes + SUM;
      }
      const int set = done & 1;
      const int64_t row0 = (int64_t)t.m * BM + 32 * quarter;
      // kept g and u: a block of 32 x 32 is eight requests of a float4 a lane, its row's
      auto kept_at = [&](float* base_, int col, int q) {
        const int64_t block = (row0 >> 5) * ((e.ld_h + 31) >> 5) + (col >> 5);
        return reinterpret_cast<float4*>(base_) + (block * 8 + ((col & 31) >> 2) + q) * 32 + lane;
      };
      // A tile's accumulators are waited for once, and given back as soon as the last of them are in registers.
      bool waited = EXACT, released = EXACT;
      auto ready = [&] {
        if (!waited) wait(f.acc[set], done / 2, W_ACC), waited = true;
        tc_fence_after();
      };
#pragma unroll 1
      for (int c64 = 0; c64 < S::COLS; c64 += 64) {
        const int first = t.n * S::COLS + c64, c0 = c64 + part * SEG, col0 = first + part * SEG;
        if (first >= p.n) break;
        const bool in = row0 < p.m && col0 < p.n, last = c64 + 64 >= S::COLS || first + 64 >= p.n;
        auto taken = [&](int k) {   // eight columns from k on are in registers
          tmem_wait_ld();
          if (!EXACT && last && k + 8 == SEG) release(set), released = true;
        };
        uint4 kept[OUT == Out::BACK ? 2 : 1][SEG / 4];
        if constexpr (OUT == Out::BACK) {
#pragma unroll
          for (int q = 0; q < SEG / 4; ++q) {
            kept[0][q] = in ? *reinterpret_cast<const uint4*>(kept_at(e.g, col0, q)) : make_uint4(0u, 0u, 0u, 0u);
            kept[1][q] = in ? *reinterpret_cast<const uint4*>(kept_at(e.u, col0, q)) : make_uint4(0u, 0u, 0u, 0u);
          }
        }
        ready();
        if constexpr (OUT == Out::GATE || OUT == Out::BACK || OUT == Out::AGAIN) {
          constexpr int N = OUT == Out::GATE ? 1 : 3;   // h; dg, du
          using Held = std::conditional_t<EXACT, F2, uint32_t>;   // 16 bits: rounded at once
          Held held[N][SEG / 2];
          auto hold = [](Held& to, F2 v) {
            if constexpr (EXACT) to = v;
            else to = pair_of<E>(v);
          };
#pragma unroll
          for (int k0 = 0; k0 < SEG; k0 += 8) {
            uint32_t g[8], u[8], dh[8];
            if constexpr (OUT == Out::BACK) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const uint4 gq = kept[0][k0 / 4 + q], uq = kept[1][k0 / 4 + q];
                g[4 * q] = gq.x, g[4 * q + 1] = gq.y, g[4 * q + 2] = gq.z, g[4 * q + 3] = gq.w;
                u[4 * q] = uq.x, u[4 * q + 1] = uq.y, u[4 * q + 2] = uq.z, u[4 * q + 3] = uq.w;
              }
            } else {
              tmem_ld8_nowait(acc + c0 + k0, g);
              tmem_ld8_nowait(acc + S::COLS + c0 + k0, u);
            }
            if constexpr (OUT != Out::GATE) tmem_ld8_nowait(acc + (OUT == Out::AGAIN ? 128 : 0) + c0 + k0, dh);
            taken(k0);
            if constexpr (OUT == Out::GATE) {
              if (e.g && in)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  *reinterpret_cast<uint4*>(kept_at(e.g, col0 + k0, q)) = make_uint4(g[4 * q], g[4 * q + 1], g[4 * q + 2], g[4 * q + 3]);
                  *reinterpret_cast<uint4*>(kept_at(e.u, col0 + k0, q)) = make_uint4(u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              F2 a, da;
              activate<EXACT, OUT != Out::GATE>(e.activation, pair(g, k), a, da);
              hold(held[0][k0 / 2 + k], mul(a, pair(u, k)));
              if constexpr (OUT != Out::GATE) {
                hold(held[1][k0 / 2 + k], mul(mul(pair(dh, k), pair(u, k)), da));
                hold(held[2][k0 / 2 + k], mul(pair(dh, k), a));
              }
            }
          }
          void* const to[3] = {e.h, e.dg, e.du};
          // one group has room for two buffers in turn: then a buffer is free again when its warps have met over the other
#pragma unroll
          for (int o = 0; o < N; ++o) {
#pragma unroll
            for (int piece = 0; piece < PIECES; ++piece) {
              uint8_t* buf = GROUPS == 1 ? rows + (turn++ & 1) * 4096 : rows;
              if constexpr (GROUPS == 2) meet();   // what stood there is written
              if constexpr (EXACT) {
                uint32_t bits[SEG / 2];
#pragma unroll
                for (int k = 0; k < SEG / 2; ++k) {
                  const float2 v = halves(held[o][k]);
                  E x, y;
                  down(x, v.x);
                  down(y, v.y);
                  bits[k] = pair_of(v.x, v.y, E{});
                  held[o][k] = f2(v.x - up(x), v.y - up(y));
                }
                put_columns<PARTS>(buf, part, lane, bits);
              } else {
                put_columns<PARTS>(buf, part, lane, held[o]);
              }
              meet();
              E* at = static_cast<E*>(to[o]) + piece * e.piece_stride;
              take_rows<PARTS>(buf, part, lane, [&](int r, int c, uint4 raw) {
                if (row0 + r < p.m && first + c < e.ld_h) *reinterpret_cast<uint4*>(at + (row0 + r) * e.ld_h + first + c) = raw;
              });
            }
          }
        } else {
          const bool floats = OUT == Out::PARTIAL || e.out_kind == 0;
          uint32_t bits[SEG / 2];   // 16-bit results
#pragma unroll
          for (int k0 = 0; k0 < SEG; k0 += 16) {
            uint32_t v[16];
            tmem_ld16_nowait(acc + c0 + k0, v);
            tmem_wait_ld();
            if (!EXACT && last && k0 + 16 == SEG) release(set), released = true;
            if (floats) {
              float* to = OUT == Out::PARTIAL ? e.part + (int64_t)(t.split * p.jobs + t.job) * p.m * p.n : static_cast<float*>(e.out[t.job]);
              const int64_t ld = OUT == Out::PARTIAL ? p.n : e.ld_out;
              emit_floats(stage, lane, v, [&](int r, int c, uint4 raw) {
                if (row0 + r < p.m) put16(to + (row0 + r) * ld, col0 + k0 + c, p.n, ld % 4 == 0, raw);
              });
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k) bits[k0 / 2 + k] = pair_of(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1]), E{});
            }
          }
          if (!floats) {
            E* to = static_cast<E*>(e.out[t.job]);
            meet();
            put_columns<PARTS>(rows, part, lane, bits);
            meet();
            take_rows<PARTS>(rows, part, lane, [&](int r, int c, uint4 raw) {
              if (row0 + r < p.m) put16(to + (row0 + r) * e.ld_out, first + c, p.n, e.ld_out % 8 == 0, raw);
            });
          }
        }
      }
      if constexpr (!EXACT) {
        if (!released) {   // no columns here
          ready();
          release(set);
        }
        done += GROUPS;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (f.aborted[0] && warp == 0)   // copies may still be on their way here
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  __syncthreads();
  if (warp == 0) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace product
}  // namespace bnb
