// Matrix products on tcgen05 tiles for operands of any size, with the epilogues of the gated feed-forward block fused
// into them (gated_mlp.cu).
//
// out (m, n) = sum over terms of A_t (m, k) B_t (n, k)^T.  One persistent CTA per SM walks over tiles of 128 x BN; a warp fetches (TMA
// boxes of 64 elements by 64 to 256, 128-byte swizzle, zeros outside the tensors, so that no size has to be a multiple of a
// tile), a warp issues the products, eight warps take finished accumulators out of tensor memory.  There are two accumulators: a tile's
// products run while the tile before is written out.
//
// An operand may lie in memory with its depth innermost (K-major) or with its rows innermost (MN-major): the same boxes, other descriptor
// bits.  So no operand of the backward is transposed in memory.
//
// 16-bit operands take one term.  Float32 ones are split into three bfloat16 pieces whose sum is exact to 24 bits, and the
// product into the six products of pieces that are not below 2^-24 of it, smallest first: six terms of the same loop.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "tile_rows.cuh"

namespace bnb {
namespace product {

using namespace tensor;

constexpr int BM = 128, BK = 64;              // tile rows; depth of a stage
constexpr int MAX_TERMS = 12;                 // two segments of six
constexpr int OUT_WARPS = 8, CTA = 32 * (2 + OUT_WARPS);
constexpr uint32_t A_BYTES = BM * BK * 2, SLAB = 64 * BK * 2;   // SLAB: 64 rows or columns by 64
enum : int { W_FULL = 101, W_EMPTY = 102, W_ACC = 103, W_DRAINED = 104 };

enum class Out : int { VALUES, PARTIAL, GATE, BACK };

// What a tile's results become.
//   VALUES   out[job] (m, n), of type `out_kind`
//   PARTIAL  float32 sums of a part of the depth: part (splits, jobs, m, n)
//   GATE     columns come in pairs of tiles, g and u: h = act(g) u as operand pieces; g and u themselves where they are kept
//   BACK     columns are dh: dg = dh u act'(g), du = dh act(g), h = act(g) u as operand pieces
struct Epilogue {
  void* out[2];
  float* part;
  void* h;              // operand pieces (pieces, m, ld_h)
  void* dg;
  void* du;
  void* g;              // values (m, ld_h)
  void* u;
  int64_t ld_out, ld_h, piece_stride;
  int out_kind;         // 0: float32, 1: the operands' type
  int activation;       // BNB_ACT_SILU or BNB_ACT_GELU
};

struct Product {
  CUtensorMap a[2], b[2];
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

// act(g) and act'(g).  e^(-g^2/2) serves the distribution function and its density: for 16-bit results by the approximation 7.1.26
// of Abramowitz and Stegun's Handbook (absolute error 1.5e-7), for float32 by erff.
template <bool EXACT>
__device__ __forceinline__ void activate(int kind, float g, float& a, float& da) {
  if (kind == BNB_ACT_SILU) {
    const float s = EXACT ? 1.0f / (1.0f + expf(-g)) : __fdividef(1.0f, 1.0f + __expf(-g));
    a = g * s;
    da = s * fmaf(g, 1.0f - s, 1.0f);
    return;
  }
  float cdf, density;   // density: g e^(-g^2/2) / sqrt(2 pi)
  if constexpr (EXACT) {
    cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752440f));
    density = g * expf(-0.5f * g * g) * 0.39894228040143267794f;
  } else {
    const float x = fabsf(g) * 0.70710678118654752440f, t = __fdividef(1.0f, fmaf(0.3275911f, x, 1.0f)), q = __expf(-0.5f * g * g);
    const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float tail = 0.5f * poly * q;   // of |g|
    cdf = g < 0.f ? tail : 1.0f - tail;
    density = g * q * 0.39894228040143267794f;
  }
  a = g * cdf;
  da = cdf + density;
}

// Eight neighbouring results of a row.
__device__ __forceinline__ void put8(float* at, const float (&v)[8], int left, bool wide) {
  if (wide && left >= 8) {
    reinterpret_cast<float4*>(at)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(at)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < left) at[i] = v[i];
  }
}
__device__ __forceinline__ uint32_t pair_of(float a, float b, __nv_bfloat16) { return pack_bf16(a, b); }
__device__ __forceinline__ uint32_t pair_of(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ void down(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void down(__half& o, float v) { o = __float2half_rn(v); }
template <typename E>
__device__ __forceinline__ void put8(E* at, const float (&v)[8], int left, bool wide) {
  if (wide && left >= 8) {
    *reinterpret_cast<uint4*>(at) = make_uint4(pair_of(v[0], v[1], E{}), pair_of(v[2], v[3], E{}), pair_of(v[4], v[5], E{}), pair_of(v[6], v[7], E{}));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < left) down(at[i], v[i]);
  }
}
__device__ __forceinline__ void get8(const float* at, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(at)[0], b = reinterpret_cast<const float4*>(at)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename E>
__device__ __forceinline__ void get8(const E* at, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(at);
  const E* e = reinterpret_cast<const E*>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = up(e[i]);
}
// The operand pieces of eight values: one rounding, or three bfloat16 numbers that add up to the value.
template <typename E, int PIECES>
__device__ __forceinline__ void put_operand(void* base, int64_t piece_stride, int64_t at, float (&v)[8]) {
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    E* to = static_cast<E*>(base) + p * piece_stride + at;
    put8(to, v, 8, true);
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

template <typename E, int PIECES> struct Kind {
  using Value = E;
  static constexpr uint32_t FORMAT = 0;
};
template <> struct Kind<__nv_bfloat16, 1> {
  using Value = __nv_bfloat16;
  static constexpr uint32_t FORMAT = (1u << 7) | (1u << 10);
};
template <> struct Kind<__nv_bfloat16, 3> {
  using Value = float;
  static constexpr uint32_t FORMAT = (1u << 7) | (1u << 10);
};

template <bool A_MN, bool B_MN, int BN>
struct Shape {
  static constexpr uint32_t B_BYTES = BN * BK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int FIT = (int)((227 * 1024 - 1024 - sizeof(Frame2) - OUT_WARPS * 4096) / STAGE), STAGES = FIT < MAX_STAGES ? FIT : MAX_STAGES;
  static constexpr uint32_t OUT = STAGES * STAGE, FRAME = OUT + OUT_WARPS * 4096, BYTES = FRAME + sizeof(Frame2) + 1024;   // 1024: to the swizzle's boundary
};

template <typename E, int PIECES, bool A_MN, bool B_MN, int BN, Out OUT>
__global__ void __launch_bounds__(CTA, 1) k_product(const __grid_constant__ Product p) {
  using S = Shape<A_MN, B_MN, BN>;
  using V = typename Kind<E, PIECES>::Value;
  constexpr bool EXACT = PIECES > 1;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
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
      mbar_init(smem_u32(&f.drained[i]), OUT_WARPS);
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
  const uint32_t tmem = f.tmem, base = smem_u32(smem);
  auto wait = [&](uint64_t& bar, uint32_t parity, int code) { mbar_wait(smem_u32(&bar), parity & 1u, &f.status, f.aborted, code); };
  const int tiles = p.m_tiles * p.n_tiles * p.jobs * p.splits, all_steps = p.k_steps * p.terms;

  if (warp == 0) {
    // fetching
    int step = 0;
    const uint32_t el = elect_one();
    for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
      const Tile t = tile_of(p, i);
      const int s0 = t.split * p.split_steps, s1 = min(all_steps, s0 + p.split_steps);
      int term = s0 / p.k_steps, k = s0 - term * p.k_steps;
      const int m0 = t.m * BM, n0 = t.n * (OUT == Out::GATE ? BN / 2 : BN);
      for (int s = s0; s < s1; ++s, ++step) {
        const int slot = step % S::STAGES;
        if (step >= S::STAGES) wait(f.empty[slot], step / S::STAGES - 1, W_EMPTY);
        if (el) {
          const uint32_t bar = smem_u32(&f.full[slot]), at = base + slot * S::STAGE, bt = at + A_BYTES;
          const CUtensorMap* am = &p.a[p.jobs > 1 ? t.job : p.a_map[term]];
          const CUtensorMap* bm = &p.b[p.b_map[term]];
          const int ap = p.a_piece[term], bp = p.b_piece[term], kc = k * BK;
          mbar_expect_tx(bar, S::STAGE);
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
        __syncwarp();
        if (++k == p.k_steps) k = 0, ++term;
      }
    }
    // every copy has landed before the CTA may leave
    for (int s = max(0, step - S::STAGES); s < step; ++s) wait(f.full[s % S::STAGES], s / S::STAGES, W_FULL);
  } else if (warp == 1) {
    // issuing
    constexpr uint32_t IDESC = (1u << 4) | Kind<E, PIECES>::FORMAT | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24) |
                               (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);
    constexpr uint32_t A_K = A_MN ? 128 : 2, B_K = B_MN ? 128 : 2;   // 16 of depth in descriptor units (16 bytes)
    const uint32_t el = elect_one(), tm = uniform(tmem);
    auto low = [](uint32_t addr, bool mn) { return ((addr & 0x3FFFFu) >> 4) | (mn ? (SLAB >> 4) << 16 : 1u << 16); };
    int step = 0, done = 0;
    for (int i = blockIdx.x; i < tiles; i += gridDim.x, ++done) {
      const Tile t = tile_of(p, i);
      const int s0 = t.split * p.split_steps, s1 = min(all_steps, s0 + p.split_steps), set = done & 1;
      if (done >= 2) wait(f.drained[set], done / 2 - 1, W_DRAINED);
      tc_fence_after();
      for (int s = s0; s < s1; ++s, ++step) {
        const int slot = step % S::STAGES;
        wait(f.full[slot], step / S::STAGES, W_FULL);
        tc_fence_after();
        const uint32_t at = base + slot * S::STAGE, a_lo = uniform(low(at, A_MN)), b_lo = uniform(low(at + A_BYTES, B_MN));
#pragma unroll
        for (uint32_t k = 0; k < BK / 16; ++k)
          mma_one<false>(el, tm + set * BN, a_lo + A_K * k, b_lo + B_K * k, IDESC, s > s0 || k ? 1u : 0u);
        tc_commit_if(el, smem_u32(&f.empty[slot]));
      }
      tc_commit_if(el, smem_u32(&f.acc[set]));
      __syncwarp();
    }
  } else {
    // taking out: this warp's 32 rows (a quarter of tensor memory is a warp's by its number) and half of the columns
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint8_t* stage = smem + S::OUT + (warp - 2) * 4096;
    const Epilogue& e = p.e;
    int done = 0;
    for (int i = blockIdx.x; i < tiles; i += gridDim.x, ++done) {
      const Tile t = tile_of(p, i);
      const int set = done & 1;
      wait(f.acc[set], done / 2, W_ACC);
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(32 * quarter) << 16) + set * BN;
      const int64_t row0 = (int64_t)t.m * BM + 32 * quarter;
      // 32 columns from a row per lane to eight neighbours of a row per lane: request q, row 8 q + lane / 4, columns 8 (lane % 4) ..
      auto stage_in = [&](const float (&v)[32]) {
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<float4*>(stage + lane * 128 + ((q ^ (lane & 7)) << 4)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        __syncwarp();
      };
      auto staged = [&](int q, float (&v)[8]) {
        const int r = 8 * q + (lane >> 2), c = 2 * (lane & 3);
        const float4 a = *reinterpret_cast<const float4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
        const float4 b = *reinterpret_cast<const float4*>(stage + r * 128 + (((c + 1) ^ (r & 7)) << 4));
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      };
      const int my_cols = OUT == Out::GATE ? BN / 4 : BN / 2;   // of the output
      static_assert(OUT == Out::GATE ? BN >= 128 : BN >= 64, "a warp takes 32 columns at a time");
#pragma unroll 1
      for (int c0 = half * my_cols; c0 < (half + 1) * my_cols; c0 += 32) {
        const int col0 = t.n * (OUT == Out::GATE ? BN / 2 : BN) + c0, col = col0 + 8 * (lane & 3);
        if (col0 >= p.n) break;
        uint32_t bits[32];
        float v[32];
        tmem_ld32(acc + c0, bits);
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(bits[k]);
        if constexpr (OUT == Out::GATE) {
          tmem_ld32(acc + BN / 2 + c0, bits);
          if (e.g) {
            stage_in(v);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int64_t r = row0 + 8 * q + (lane >> 2);
              float o[8];
              staged(q, o);
              if (r < p.m && col < e.ld_h) put8(static_cast<V*>(e.g) + r * e.ld_h + col, o, 8, true);
            }
            float w[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) w[k] = __uint_as_float(bits[k]);
            stage_in(w);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int64_t r = row0 + 8 * q + (lane >> 2);
              float o[8];
              staged(q, o);
              if (r < p.m && col < e.ld_h) put8(static_cast<V*>(e.u) + r * e.ld_h + col, o, 8, true);
            }
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            float a, da;
            activate<EXACT>(e.activation, v[k], a, da);
            v[k] = a * __uint_as_float(bits[k]);
          }
          stage_in(v);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int64_t r = row0 + 8 * q + (lane >> 2);
            float o[8];
            staged(q, o);
            if (r < p.m && col < e.ld_h) put_operand<E, PIECES>(e.h, e.piece_stride, r * e.ld_h + col, o);
          }
        } else {
          stage_in(v);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int64_t r = row0 + 8 * q + (lane >> 2);
            float o[8];
            staged(q, o);
            if constexpr (OUT == Out::BACK) {
              if (r < p.m && col < e.ld_h) {
                const int64_t at = r * e.ld_h + col;
                float g[8], u[8], dg[8], du[8], h[8];
                get8(static_cast<const V*>(e.g) + at, g);
                get8(static_cast<const V*>(e.u) + at, u);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  float a, da;
                  activate<EXACT>(e.activation, g[k], a, da);
                  dg[k] = o[k] * u[k] * da;
                  du[k] = o[k] * a;
                  h[k] = a * u[k];
                }
                put_operand<E, PIECES>(e.dg, e.piece_stride, at, dg);
                put_operand<E, PIECES>(e.du, e.piece_stride, at, du);
                put_operand<E, PIECES>(e.h, e.piece_stride, at, h);
              }
            } else if (r < p.m && col < p.n) {
              const int left = p.n - col;
              if constexpr (OUT == Out::PARTIAL) {
                put8(e.part + (((int64_t)t.split * p.jobs + t.job) * p.m + r) * p.n + col, o, left, p.n % 4 == 0);
              } else if (e.out_kind == 0) {
                put8(static_cast<float*>(e.out[t.job]) + r * e.ld_out + col, o, left, e.ld_out % 4 == 0);
              } else {
                put8(static_cast<E*>(e.out[t.job]) + r * e.ld_out + col, o, left, e.ld_out % 8 == 0);
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&f.drained[set]));
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
