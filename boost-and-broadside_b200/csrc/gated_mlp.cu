// The gated feed-forward block of any size, y = (act(x Wg^T) * (x Wu^T)) Wd^T, forward and backward (GatedMLP, attention.py:21-37, as an
// operator of its own with gradients; act is erf GELU or SiLU):
//
//   dh = dy Wd,  dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
//
// Six width x hidden products a row forward and twelve backward: the tensor cores bound it, from widths on whose rows cost more
// than their memory.  Forward is two launches: both projections, the activation and their product in one, where g and u of a tile
// meet in tensor memory, and the down projection.  Backward is four: dh with the gate's derivatives (and h once more), dx over both
// halves, dWg and dWu, dWd.  product_tiles.cuh has the products.
//
// h, dg and du are rounded to the operands' type between the products: they are operands of the next one.  g and u are not: they
// enter the backward as float32, either kept by the forward or, where that is cheaper, computed once more (see recomputes).  Sums over the
// depth are float32; where the depth is cut into parts (few tiles), the parts are added in a fixed order.
#include <algorithm>
#include <mutex>

#include "launch_count.h"
#include "product_tiles.cuh"
#include "tensor_kernels.h"

namespace bnb {
namespace product {
namespace {

size_t round256(size_t v) { return (v + 255) / 256 * 256; }
int64_t round8(int64_t v) { return (v + 7) / 8 * 8; }

// ------------------------------------------------------------------ operands

// (pieces, rows, cols) 16-bit elements.
struct Operand { const void* data; int64_t rows, cols, ld, piece_stride; };

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

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                            const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encoder() {
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
bool has_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}
// Boxes of 64 columns by box_rows rows of one piece.
bool map_of(CUtensorMap& m, const Operand& o, int pieces, int box_rows, bool half) {
  const Encode enc = encoder();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)pieces};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(pieces > 1 ? o.piece_stride : o.rows * o.ld) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
  return enc(&m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.data), dims, strides, box, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ------------------------------------------------------------------ products

constexpr int SMS = 148;

struct Shaped { int bn, tiles, splits, split_steps; };
// The width of a tile: the one with the least time.  A stage moves (128 + BN) rows of 128 bytes into shared memory and the products read
// them once from there, at 128 bytes a clock: 2 (128 + BN) clocks, more than the products themselves take at any BN up to 256 (measured:
// 790 clocks a stage at 256).  A tile's fixed cost (fill, the last results) is about 1200.  Then, where tiles leave SMs idle and results can be
// added, the depth is cut so that all have work, no part below 8 stages; the sums' launch costs some 6000 clocks.
Shaped shape_of(int64_t m, int64_t n, int jobs, int steps, int most, int least, int out_of_bn, bool may_split) {
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
        best = {bn, (int)tiles, splits, split_steps};
        cost = c;
      }
    }
  }
  return best;
}

template <typename E, int PIECES, bool A_MN, bool B_MN, int BN, Out OUT>
int launch(const Product& p, int tiles, cudaStream_t st) {
  constexpr uint32_t bytes = Shape<BN, OUT>::BYTES;
  auto kernel = k_product<E, PIECES, A_MN, B_MN, BN, OUT>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return BNB_ERR_LAUNCH;
  return launch_after(kernel, dim3(std::min(tiles, SMS)), CTA, bytes, st, p);
}

// Pieces of a float32 product that are not below 2^-24 of it, smallest first.
constexpr int PAIRS[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};

struct Sides { Operand a[2], b[3]; int segments; };   // segments: a[s] b[s]^T are added

// Widths of tiles that are built: two sets of accumulators are 512 columns, and float32 adds runs in a third.
template <int PIECES> constexpr int MOST = PIECES > 1 ? 128 : 256;

template <typename E, int PIECES, bool A_MN, bool B_MN, Out OUT>
int at_width(const Product& p, int bn, int tiles, cudaStream_t st) {
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
  Shaped z = again ? Shaped{64, (int)((m + BM - 1) / BM * ((n + 63) / 64)), 1, p.k_steps}
                   : shape_of(m, n, jobs, p.k_steps * p.terms, MOST<PIECES>, LEAST, OF, OUT == Out::VALUES);
  p.splits = z.splits;
  p.split_steps = z.split_steps;
  p.m_tiles = (int)((m + BM - 1) / BM);
  p.n_tiles = (int)((n + z.bn / OF - 1) / (z.bn / OF));
  p.host_status = host_status_word(st);
  constexpr bool half = std::is_same<E, __half>::value;
  const int a_maps = again ? 2 : jobs > 1 ? jobs : s.segments, b_maps = again ? 3 : OUT == Out::GATE ? 2 : s.segments;
  bool ok = has_context();
  for (int i = 0; i < a_maps; ++i) ok = ok && map_of(p.a[i], s.a[i], PIECES, A_MN ? BK : BM, half);
  for (int i = 0; i < b_maps; ++i) ok = ok && map_of(p.b[i], s.b[i], PIECES, again || B_MN ? BK : z.bn / OF, half);
  if (!ok) return BNB_ERR_LAUNCH;
  const int total = z.tiles * z.splits;
  if constexpr (again) {
    return launch<E, PIECES, false, false, 192, OUT>(p, total, st);
  } else if constexpr (OUT == Out::VALUES) {
    if (z.splits > 1) {
      p.e.part = part;
      if (const int r = at_width<E, PIECES, A_MN, B_MN, Out::PARTIAL>(p, z.bn, total, st)) return r;
      const int64_t cells = m * n;
      count_launch();
      k_add_parts<E><<<(unsigned)((cells * jobs + 63) / 64), 256, 0, st>>>(part, z.splits, cells, jobs, e.out[0], e.out[1], e.out_kind);
      return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
    }
    return at_width<E, PIECES, A_MN, B_MN, OUT>(p, z.bn, total, st);
  } else {
    return at_width<E, PIECES, A_MN, B_MN, OUT>(p, z.bn, total, st);
  }
}
size_t part_bytes(int64_t m, int64_t n, int64_t depth, int jobs, int terms, int most) {
  const Shaped z = shape_of(m, n, jobs, (int)((depth + BK - 1) / BK) * terms, most, 64, 1, true);
  return z.splits > 1 ? round256((size_t)z.splits * jobs * m * n * 4) : 0;
}

// ------------------------------------------------------------------ the block

int check(const BnbGatedBlock* c) {
  if (!c) return BNB_ERR_NULL_POINTER;
  if (c->rows < 0 || c->element < 0 || c->element > 2 || c->weight_element < 0 || c->weight_element > 2 ||
      (c->activation != BNB_ACT_SILU && c->activation != BNB_ACT_GELU)) return BNB_ERR_BAD_ARGUMENT;
  if (c->width < 1 || c->hidden < 1 || c->width > 1 << 20 || c->hidden > 1 << 20 || c->rows > (int64_t)1 << 31) return BNB_ERR_UNSUPPORTED_DIMS;
  if (c->weight_element != c->element && c->weight_element != BNB_ELEM_F32) return BNB_ERR_UNSUPPORTED_DIMS;
  if (!c->gate_w || !c->up_w || !c->down_w || (c->rows && !c->x)) return BNB_ERR_NULL_POINTER;
  return BNB_OK;
}

// Whether the backward computes g and u once more.  Kept in float32 they cost the same at any width, computing them costs with the width: for
// 33.5 million rows x hidden columns, keeping takes 44 us more forward and 113 for the backward's launch, computing 64 at a width of 128
// and 230 at 1024.  So up to 512, in 16 bits; float32 takes six times the products, and keeps.
bool recomputes(const BnbGatedBlock& c) { return c.element != BNB_ELEM_F32 && c.width <= 512; }

int64_t round32(int64_t v) { return (v + 31) / 32 * 32; }
// Whether a tensor map can describe rows as they lie: no rows that share memory (a gradient expanded from one row) among them.
bool lies_well(const void* p, int64_t cols, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && ld >= cols; }

// Where everything of a call stands in its scratch; sizes alone with base = null.
struct Layout {
  int pieces;
  int64_t M, D, F, ld_h;
  Operand x, gate, up, down, dy, h, dg, du;
  float* part;
  PackJobs jobs;
  int n_jobs;
  size_t total;

  Layout(const BnbGatedBlock& c, const void* dy_in, int64_t dy_ld, bool backward, uint8_t* base)
      : pieces(c.element == BNB_ELEM_F32 ? 3 : 1), M(c.rows), D(c.width), F(c.hidden), ld_h(round8(c.hidden)), dy{}, dg{}, du{}, part(nullptr), jobs{}, n_jobs(0), total(0) {
    auto take = [&](size_t bytes) {
      uint8_t* at = base ? base + total : nullptr;
      total += round256(bytes);
      return at;
    };
    auto operand = [&](const void* p, int64_t rows, int64_t cols, int64_t ld, int element) {
      if (pieces == 1 && element == c.element && lies_well(p, cols, ld)) return Operand{p, rows, cols, ld, 0};
      const int64_t to = round8(cols), stride = rows * to;
      void* at = take((size_t)pieces * stride * 2);
      jobs.job[n_jobs++] = {p, at, rows, ld, stride, (int)cols, (int)to, element == BNB_ELEM_F32 ? 0 : 1};
      return Operand{at, rows, cols, to, stride};
    };
    auto between = [&] { return Operand{take((size_t)pieces * M * ld_h * 2), M, F, ld_h, M * ld_h}; };
    x = operand(c.x, M, D, c.x_row, c.element);
    gate = operand(c.gate_w, F, D, D, c.weight_element);
    up = operand(c.up_w, F, D, D, c.weight_element);
    down = operand(c.down_w, D, F, F, c.weight_element);
    h = between();
    const int t = pieces > 1 ? 6 : 1, most = pieces > 1 ? MOST<3> : MOST<1>;
    size_t parts = 0;
    if (!backward) {
      parts = part_bytes(M, D, F, 1, t, most);
    } else {
      dy = operand(dy_in, M, D, dy_ld, c.element);
      dg = between();
      du = between();
      parts = std::max({part_bytes(M, D, F, 1, 2 * t, most), part_bytes(F, D, M, 2, t, most), part_bytes(D, F, M, 1, t, most)});
    }
    part = reinterpret_cast<float*>(take(parts));
  }
};

template <typename E, int PIECES>
int pack(const Layout& l, cudaStream_t st) {
  if (!l.n_jobs) return BNB_OK;
  int64_t most = 1;
  for (int i = 0; i < l.n_jobs; ++i) most = std::max(most, l.jobs.job[i].rows * (l.jobs.job[i].dst_ld / 8));
  count_launch();
  k_pack<E, PIECES><<<dim3((unsigned)std::min<int64_t>((most + 255) / 256, SMS * 16), l.n_jobs), 256, 0, st>>>(l.jobs);
  return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
}

Epilogue between(const BnbGatedBlock& c, const Layout& l) {
  Epilogue e{};
  e.activation = c.activation;
  e.ld_h = l.ld_h;
  e.piece_stride = l.M * l.ld_h;
  e.h = const_cast<void*>(l.h.data);
  e.dg = const_cast<void*>(l.dg.data);
  e.du = const_cast<void*>(l.du.data);
  if (c.kept && !recomputes(c)) {
    e.g = static_cast<float*>(c.kept);
    e.u = e.g + round32(l.M) * round32(l.F);
  }
  return e;
}

template <typename E, int PIECES>
int forward(const BnbGatedBlock& c, const Layout& l, cudaStream_t st) {
  if (const int r = pack<E, PIECES>(l, st)) return r;
  const Sides up{{l.x, {}}, {l.gate, l.up}, 1};
  if (const int r = multiply<E, PIECES, false, false, Out::GATE>(up, l.M, l.F, l.D, 1, between(c, l), nullptr, st)) return r;
  Epilogue e{};
  e.out[0] = c.y;
  e.ld_out = l.D;
  e.out_kind = PIECES > 1 ? 0 : 1;
  return multiply<E, PIECES, false, false, Out::VALUES>({{l.h, {}}, {l.down, {}}, 1}, l.M, l.D, l.F, 1, e, l.part, st);
}

template <typename E, int PIECES>
int backward(const BnbGatedBlock& c, const BnbGatedBlockGrads& g, const Layout& l, cudaStream_t st) {
  if (const int r = pack<E, PIECES>(l, st)) return r;
  int r;
  if constexpr (PIECES == 1) {
    r = recomputes(c) ? multiply<E, PIECES, false, false, Out::AGAIN>({{l.x, l.dy}, {l.gate, l.up, l.down}, 1}, l.M, l.F, l.D, 1, between(c, l), nullptr, st)
                      : multiply<E, PIECES, false, true, Out::BACK>({{l.dy, {}}, {l.down, {}}, 1}, l.M, l.F, l.D, 1, between(c, l), nullptr, st);
  } else {
    r = multiply<E, PIECES, false, true, Out::BACK>({{l.dy, {}}, {l.down, {}}, 1}, l.M, l.F, l.D, 1, between(c, l), nullptr, st);
  }
  if (r) return r;
  Epilogue e{};
  const int own = PIECES > 1 ? 0 : 1, weights = c.weight_element == BNB_ELEM_F32 ? 0 : 1;
  if (g.dx) {
    e.out[0] = g.dx;
    e.ld_out = l.D;
    e.out_kind = own;
    if (r = multiply<E, PIECES, false, true, Out::VALUES>({{l.dg, l.du}, {l.gate, l.up}, 2}, l.M, l.D, l.F, 1, e, l.part, st); r) return r;
  }
  e.out_kind = weights;
  if (g.dgate_w && g.dup_w) {
    e.out[0] = g.dgate_w;
    e.out[1] = g.dup_w;
    e.ld_out = l.D;
    if (r = multiply<E, PIECES, true, true, Out::VALUES>({{l.dg, l.du}, {l.x, {}}, 1}, l.F, l.D, l.M, 2, e, l.part, st); r) return r;
  }
  if (g.ddown_w) {
    e.out[0] = g.ddown_w;
    e.out[1] = nullptr;
    e.ld_out = l.F;
    return multiply<E, PIECES, true, true, Out::VALUES>({{l.dy, {}}, {l.h, {}}, 1}, l.D, l.F, l.M, 1, e, l.part, st);
  }
  return BNB_OK;
}

}  // namespace
}  // namespace product
}  // namespace bnb

using namespace bnb;
using namespace bnb::product;

extern "C" size_t bnb_gated_block_kept_bytes(const BnbGatedBlock* c) {
  if (check(c)) return 0;
  return recomputes(*c) ? 0 : (size_t)2 * round32(c->rows) * round32(c->hidden) * 4;
}

extern "C" size_t bnb_gated_block_scratch_bytes(const BnbGatedBlock* c, int backward) {
  if (check(c) || c->rows == 0) return 0;
  // operands that may have to be copied count as copied: dy's address is not known yet
  return Layout(*c, reinterpret_cast<const void*>(1), c->width, backward != 0, nullptr).total;
}

extern "C" int bnb_gated_block_fwd(const BnbGatedBlock* c, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int st = check(c)) return st;
  if (c->rows == 0) return BNB_OK;
  if (!c->y) return BNB_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(c->y) | reinterpret_cast<uintptr_t>(c->kept) | reinterpret_cast<uintptr_t>(scratch)) & 15) return BNB_ERR_MISALIGNED;
  const Layout l(*c, nullptr, 0, false, static_cast<uint8_t*>(scratch));
  if (!scratch || scratch_bytes < l.total) return BNB_ERR_SCRATCH_TOO_SMALL;
  const auto s = static_cast<cudaStream_t>(stream);
  return c->element == BNB_ELEM_F32 ? forward<__nv_bfloat16, 3>(*c, l, s)
       : c->element == BNB_ELEM_BF16 ? forward<__nv_bfloat16, 1>(*c, l, s) : forward<__half, 1>(*c, l, s);
}

extern "C" int bnb_gated_block_bwd(const BnbGatedBlock* c, const BnbGatedBlockGrads* g, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int st = check(c)) return st;
  if (!g) return BNB_ERR_NULL_POINTER;
  const auto s = static_cast<cudaStream_t>(stream);
  const size_t cells = (size_t)c->width * c->hidden * (c->weight_element == BNB_ELEM_F32 ? 4 : 2);
  if (c->rows == 0) {
    for (void* p : {g->dgate_w, g->dup_w, g->ddown_w})
      if (p && cudaMemsetAsync(p, 0, cells, s) != cudaSuccess) return BNB_ERR_LAUNCH;
    return BNB_OK;
  }
  if (!g->dy || (!c->kept && !recomputes(*c)) || (g->dgate_w == nullptr) != (g->dup_w == nullptr)) return BNB_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(c->kept) | reinterpret_cast<uintptr_t>(scratch) | reinterpret_cast<uintptr_t>(g->dx) | reinterpret_cast<uintptr_t>(g->dgate_w) |
       reinterpret_cast<uintptr_t>(g->dup_w) | reinterpret_cast<uintptr_t>(g->ddown_w)) & 15) return BNB_ERR_MISALIGNED;
  const Layout l(*c, g->dy, g->dy_row, true, static_cast<uint8_t*>(scratch));
  if (!scratch || scratch_bytes < l.total) return BNB_ERR_SCRATCH_TOO_SMALL;
  return c->element == BNB_ELEM_F32 ? backward<__nv_bfloat16, 3>(*c, *g, l, s)
       : c->element == BNB_ELEM_BF16 ? backward<__nv_bfloat16, 1>(*c, *g, l, s) : backward<__half, 1>(*c, *g, l, s);
}
