// The host side of product_tiles.cuh for the operators made of it (gated_mlp.cu, linear.cu): operands and their copies, tensor maps, the
// choice of a tile's width, sums over a depth that is cut.
#pragma once

#include <algorithm>
#include <type_traits>

#include "launch_count.h"
#include "product_tiles.cuh"
#include "tensor_kernels.h"

namespace bnb {
namespace product {
namespace {

inline size_t round256(size_t v) { return (v + 255) / 256 * 256; }
inline int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }
inline int64_t round32(int64_t v) { return (v + 31) / 32 * 32; }

constexpr int SMS = 148;

// ------------------------------------------------------------------ operands

// (pieces, rows, cols) 16-bit elements.
struct Operand { const void* data; int64_t rows, cols, ld, piece_stride; };

// Whether a tensor map can describe rows as they lie: no rows that share memory (a gradient expanded from one row) among them.
inline bool lies_well(const void* p, int64_t cols, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && ld >= cols; }
// What the products cannot read as it lies (float32, strides or addresses off 16 bytes, overlapping rows): copied as operand pieces.
struct PackJob { const void* src; void* dst; int64_t rows, src_ld, piece_stride; int cols, dst_ld, kind; };   // kind: 0 float32, else the operands' type
constexpr int MAX_JOBS = 5;
struct PackJobs { PackJob job[MAX_JOBS]; };
template <typename E, int PIECES>
__global__ void __launch_bounds__(256) k_pack(const __grid_constant__ PackJobs jobs) {
  const PackJob& j = jobs.job[blockIdx.y];
  const int groups = j.dst_ld / 8;
  const int64_t total = j.rows * groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / groups;
    const int c = (int)(i - r * groups) * 8;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t at = r * j.src_ld + c + k;
      v[k] = c + k >= j.cols ? 0.f : j.kind == 0 ? static_cast<const float*>(j.src)[at] : up(static_cast<const E*>(j.src)[at]);
    }
    put_operand<E, PIECES>(j.dst, j.piece_stride, r * j.dst_ld + c, v);
  }
}

template <typename E, int PIECES>
int pack(const PackJobs& jobs, int n_jobs, cudaStream_t st) {
  if (!n_jobs) return BNB_OK;
  int64_t most = 1;
  for (int i = 0; i < n_jobs; ++i) most = std::max(most, jobs.job[i].rows * (jobs.job[i].dst_ld / 8));
  count_launch();
  k_pack<E, PIECES><<<dim3((unsigned)std::min<int64_t>((most + 255) / 256, SMS * 16), n_jobs), 256, 0, st>>>(jobs);
  return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
}

// Sums of the parts of a depth: four threads share a cell's parts, each in their order, and are added in theirs.
template <typename E>
__global__ void __launch_bounds__(256) k_add_parts(const float* part, int splits, int64_t cells, int jobs, void* out0, void* out1, int out_kind) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + lane;
  float v = 0.f;
  if (i < cells * jobs) {
#pragma unroll 8
    for (int s = q; s < splits; s += 4) v += part[s * cells * jobs + i];
  }
  sums[q][lane] = v;
  __syncthreads();
  if (q || i >= cells * jobs) return;
  v = (v + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
  void* out = i < cells ? out0 : out1;
  const int64_t at = i < cells ? i : i - cells;
  if (out_kind == 0) static_cast<float*>(out)[at] = v;
  else down(static_cast<E*>(out)[at], v);
}

// A linear layer's result from its sum: bias, activation and residual.  E: the call's type, float among them.
template <typename E>
__device__ __forceinline__ void put_linear(const Epilogue& e, int64_t r, int c, float v) {
  auto value = [](const void* from, int64_t at) {
    if constexpr (sizeof(E) == 4) return static_cast<const float*>(from)[at];
    else return up(static_cast<const E*>(from)[at]);
  };
  if (e.bias) v += e.bias_kind == 0 ? static_cast<const float*>(e.bias)[c] : value(e.bias, c);
  if (e.g) e.g[kept_index(r, c, e.ld_h)] = v;
  float da = 1.f;
  if (e.activation != BNB_ACT_NONE) activate_exact(e.activation, v, v, da);
  if (e.slopes) e.slopes[kept_slope_index(r, c, e.ld_h)] = __float2half_rn(da * KEPT_SCALE);
  if (e.other) v += value(e.other, r * e.ld_other + c);
  down(static_cast<E*>(e.out[0])[r * e.ld_out + c], v);
}

// The same for a linear layer.
template <typename E>
__global__ void __launch_bounds__(256) k_add_linear(const __grid_constant__ Epilogue e, const float* part, int splits, int64_t m, int n) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int64_t cells = m * n, i = (int64_t)blockIdx.x * 64 + lane;
  let_next_start();
  wait_for_previous();
  float v = 0.f;
  if (i < cells) {
#pragma unroll 8
    for (int s = q; s < splits; s += 4) v += part[s * cells + i];
  }
  sums[q][lane] = v;
  __syncthreads();
  if (q || i >= cells) return;
  v = (v + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
  const int64_t r = i / n;
  const int c = (int)(i - r * n);
  if (e.out_kind == 0) put_linear<float>(e, r, c, v);
  else put_linear<E>(e, r, c, v);
}

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                            const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline Encode encoder() {
  static const Encode f = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<Encode>(p);
  }();
  return f;
}
// The encoder is a driver call and needs the device's context on this thread; a thread that has made no runtime call yet
// (autograd's) has none, and cudaSetDevice gives it one.
inline bool has_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}
// Boxes of 64 columns by box_rows rows of one piece.
inline bool map_of(CUtensorMap& m, const Operand& o, int pieces, int box_rows, bool half) {
  const Encode enc = encoder();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)pieces};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(pieces > 1 ? o.piece_stride : o.rows * o.ld) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
  return enc(&m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.data), dims, strides, box, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ------------------------------------------------------------------ products

// Clocks of a stage of two CTAs on 256 x 256, see shape_of.
constexpr double PAIR_STAGE = 640.0;
struct Shaped { int bn, tiles, splits, split_steps; bool pair; };
// The width of a tile: the one with the least time.  A stage moves (128 + BN) rows of 128 bytes into shared memory and the products read
// them once from there, at 128 bytes a clock: 2 (128 + BN) clocks, more than the products themselves take at any BN up to 256 (measured:
// 790 clocks a stage at 256).  A tile's fixed cost (fill, the last results) is about 1200.  Then, where tiles leave SMs idle and results can be
// added, the depth is cut so that all have work, no part below 8 stages; the sums' launch costs some 6000 clocks.  Two CTAs on 256 x 256 (16-bit operands) each hold their rows
// and half of the columns' operand: 2 (128 + 128) clocks of shared memory, as much as the products take.  8192 x 4096 outputs, us of one and of two CTAs to a tile: width
// 4096 231 and 187, 2048 121 and 101, 1024 70 and 68 (its results bound it); a stage is 0.79 of a single one's there, and counts for a little more, since 74 pairs divide work less
// evenly than 148 CTAs (4736 rows, five rounds for four: 136 and 153).
inline Shaped shape_of(int64_t m, int64_t n, int jobs, int steps, int most, int least, int out_of_bn, bool may_split) {
  const int64_t mt = (m + BM - 1) / BM;
  Shaped best{};
  double cost = 0;
  for (int bn = most; bn >= least; bn /= 2) {
    const int64_t tiles = mt * ((n + bn / out_of_bn - 1) / (bn / out_of_bn)) * jobs;
    for (int cut = 0; cut <= (may_split && tiles < SMS ? 1 : 0); ++cut) {
      int splits = cut ? (int)std::max<int64_t>(1, std::min<int64_t>(SMS / tiles, steps / 8)) : 1;
      const int split_steps = (steps + splits - 1) / splits;
      splits = (steps + split_steps - 1) / split_steps;
      const double rounds = (double)((tiles * splits + SMS - 1) / SMS), c = rounds * (split_steps * 2.0 * (BM + bn) + 1200.0) + (splits > 1 ? 6000.0 : 0.0);
      if (best.bn == 0 || c < cost) {
        best = {bn, (int)tiles, splits, split_steps, false};
        cost = c;
      }
    }
  }
  if (may_split && most == 256) {
    const int64_t tiles = (mt + 1) / 2 * ((n + 255) / 256) * jobs;
    const double rounds = (double)((tiles + SMS / 2 - 1) / (SMS / 2)), c = rounds * (steps * PAIR_STAGE + 1200.0);
    if (c < cost) best = {256, (int)tiles, 1, steps, true};
  }
  return best;
}

template <typename E, int PIECES, bool A_MN, bool B_MN, int BN, Out OUT, bool PAIR = false>
int launch(const Product& p, int tiles, cudaStream_t st) {
  constexpr uint32_t bytes = Shape<BN, OUT, PIECES, PAIR>::BYTES;
  auto kernel = k_product<E, PIECES, A_MN, B_MN, BN, OUT, PAIR>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return BNB_ERR_LAUNCH;
  if constexpr (PAIR) return launch_clusters_after(2, kernel, dim3(2 * std::min(tiles, SMS / 2)), Crew<PIECES, BN, OUT>::THREADS, bytes, st, p);
  return launch_after(kernel, dim3(std::min(tiles, SMS)), Crew<PIECES, BN, OUT>::THREADS, bytes, st, p);
}

// Pieces of a float32 product that are not below 2^-24 of it, smallest first.
constexpr int PAIRS[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};

struct Sides { Operand a[2], b[3]; int segments; };   // segments: a[s] b[s]^T are added

// Widths of tiles that are built: two sets of accumulators are 512 columns, and float32 adds runs in a third.
template <int PIECES> constexpr int MOST = PIECES > 1 ? 128 : 256;

// A linear layer's widest tile: narrow ones are bound by their epilogues, which have more warps at 128 columns.  65536 rows x 512 outputs with GELU, us with tiles
// of 256 and 128 columns: width 128 42.1 and 39.0, 512 50.6 and 49.4; 8192 x 1024 x 4096 75.0 and 79.6.
inline int most_of_linear(int pieces, int k_steps) { return pieces > 1 || k_steps <= 8 ? 128 : 256; }

template <typename E, int PIECES, bool A_MN, bool B_MN, Out OUT>
int at_width(const Product& p, int bn, int tiles, bool pair, cudaStream_t st) {
  if constexpr (PIECES == 1 && (OUT == Out::VALUES || OUT == Out::LINEAR))
    if (pair) return launch<E, PIECES, A_MN, B_MN, 256, OUT, true>(p, tiles, st);
  if constexpr (PIECES == 1)
    if (bn == 256) return launch<E, PIECES, A_MN, B_MN, 256, OUT>(p, tiles, st);
  if (bn == 128) return launch<E, PIECES, A_MN, B_MN, 128, OUT>(p, tiles, st);
  if constexpr (OUT != Out::GATE) return launch<E, PIECES, A_MN, B_MN, 64, OUT>(p, tiles, st);
  return BNB_ERR_BAD_ARGUMENT;
}

template <typename E, int PIECES, bool A_MN, bool B_MN, Out OUT>
int multiply(const Sides& s, int64_t m, int64_t n, int64_t depth, int jobs, const Epilogue& e, float* part, cudaStream_t st) {
  Product p{};
  p.e = e;
  p.m = m;
  p.n = (int)n;
  p.jobs = jobs;
  p.k_steps = (int)((depth + BK - 1) / BK);
  p.terms = s.segments * (PIECES > 1 ? 6 : 1);
  for (int t = 0; t < p.terms; ++t) {
    const int seg = t % s.segments, pair = t / s.segments;
    p.a_map[t] = p.b_map[t] = (uint8_t)seg;
    p.a_piece[t] = PIECES > 1 ? (uint8_t)PAIRS[pair][0] : 0;
    p.b_piece[t] = PIECES > 1 ? (uint8_t)PAIRS[pair][1] : 0;
  }
  constexpr bool again = OUT == Out::AGAIN;
  constexpr int LEAST = OUT == Out::GATE ? 128 : 64, OF = OUT == Out::GATE ? 2 : 1;
  const int most = OUT == Out::LINEAR ? most_of_linear(PIECES, p.k_steps) : MOST<PIECES>;
  Shaped z = again ? Shaped{64, (int)((m + BM - 1) / BM * ((n + 63) / 64)), 1, p.k_steps, false}
                   : shape_of(m, n, jobs, p.k_steps * p.terms, most, LEAST, OF, OUT == Out::VALUES || OUT == Out::LINEAR);
  p.splits = z.splits;
  p.split_steps = z.split_steps;
  p.m_tiles = (int)((m + (z.pair ? 2 * BM : BM) - 1) / (z.pair ? 2 * BM : BM));
  p.n_tiles = (int)((n + z.bn / OF - 1) / (z.bn / OF));
  p.host_status = host_status_word(st);
  constexpr bool half = std::is_same<E, __half>::value;
  const int a_maps = again ? 2 : jobs > 1 ? jobs : s.segments, b_maps = again ? 3 : OUT == Out::GATE ? 2 : s.segments;
  bool ok = has_context();
  for (int i = 0; i < a_maps; ++i) ok = ok && map_of(p.a[i], s.a[i], PIECES, A_MN ? BK : BM, half);
  for (int i = 0; i < b_maps; ++i) ok = ok && map_of(p.b[i], s.b[i], PIECES, again || B_MN ? BK : z.pair ? z.bn / 2 : z.bn / OF, half);
  if (!ok) return BNB_ERR_LAUNCH;
  const int total = z.tiles * z.splits;
  if constexpr (again) {
    return launch<E, PIECES, false, false, 192, OUT>(p, total, st);
  } else if constexpr (OUT == Out::LINEAR) {
    if (z.splits > 1) {
      p.e.part = part;
      if (const int r = at_width<E, PIECES, A_MN, B_MN, Out::PARTIAL>(p, z.bn, total, z.pair, st)) return r;
      return launch_after(k_add_linear<E>, dim3((unsigned)((m * n + 63) / 64)), 256, 0, st, p.e, (const float*)part, z.splits, m, (int)n);
    }
    return at_width<E, PIECES, A_MN, B_MN, OUT>(p, z.bn, total, z.pair, st);
  } else if constexpr (OUT == Out::VALUES) {
    if (z.splits > 1) {
      p.e.part = part;
      if (const int r = at_width<E, PIECES, A_MN, B_MN, Out::PARTIAL>(p, z.bn, total, z.pair, st)) return r;
      const int64_t cells = m * n;
      count_launch();
      k_add_parts<E><<<(unsigned)((cells * jobs + 63) / 64), 256, 0, st>>>(part, z.splits, cells, jobs, e.out[0], e.out[1], e.out_kind);
      return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
    }
    return at_width<E, PIECES, A_MN, B_MN, OUT>(p, z.bn, total, z.pair, st);
  } else {
    return at_width<E, PIECES, A_MN, B_MN, OUT>(p, z.bn, total, z.pair, st);
  }
}
inline size_t part_bytes(int64_t m, int64_t n, int64_t depth, int jobs, int terms, int most) {
  const Shaped z = shape_of(m, n, jobs, (int)((depth + BK - 1) / BK) * terms, most, 64, 1, true);
  return z.splits > 1 ? round256((size_t)z.splits * jobs * m * n * 4) : 0;
}

}  // namespace
}  // namespace product
}  // namespace bnb
