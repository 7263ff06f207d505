// The linear layer of any size with what surrounds it, y = act(z) + r, z = x W^T + b, forward and backward:
//
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz,  dr = dy
//
// Forward is one launch: bias, activation and residual enter where the sums leave tensor memory (Out::LINEAR of product_tiles.cuh).  A product of two
// operations for each of rows x width x out forward and twice that backward: the tensor cores bound it, or, for few rows or a small width, memory.
//
// The backward of an activation needs z as it was before any rounding.  Either it is computed once more, with dy taken to dz behind it
// (Out::SLOPE), or the forward keeps it in float32 (see recomputes).  dz is rounded to the operands' type: it is an operand of the two
// products behind it, and the bias's gradient is the sum of the same numbers.  Without an activation dz is dy as it lies.
#include "product_calls.cuh"

namespace bnb {
namespace product {
namespace {

int check(const BnbLinear* c) {
  if (!c) return BNB_ERR_NULL_POINTER;
  if (c->rows < 0 || c->element < 0 || c->element > 2 || c->weight_element < 0 || c->weight_element > 2 || c->bias_element < 0 || c->bias_element > 2 ||
      (c->activation != BNB_ACT_NONE && c->activation != BNB_ACT_SILU && c->activation != BNB_ACT_GELU)) return BNB_ERR_BAD_ARGUMENT;
  if (c->width < 1 || c->out < 1 || c->width > 1 << 20 || c->out > 1 << 20 || c->rows > (int64_t)1 << 31) return BNB_ERR_UNSUPPORTED_DIMS;
  if (c->weight_element != c->element && c->weight_element != BNB_ELEM_F32) return BNB_ERR_UNSUPPORTED_DIMS;
  if (c->bias && c->bias_element != c->element && c->bias_element != BNB_ELEM_F32) return BNB_ERR_UNSUPPORTED_DIMS;
  if (!c->weight || (c->rows && !c->x)) return BNB_ERR_NULL_POINTER;
  return BNB_OK;
}

// Whether the backward computes z once more: keeping it costs 8 bytes a result, written and read, computing it 2 width operations.
// At the measured rates (6.5 TB/s, 1.4 PFLOP/s) they are even at a width of 860, and keeping holds the memory; float32 takes six times
// the products, and keeps.
bool recomputes(const BnbLinear& c) { return c.activation == BNB_ACT_NONE || (c.element != BNB_ELEM_F32 && c.width <= 512); }
bool keeps(const BnbLinear& c) { return !recomputes(c); }

// dz from the kept z, eight neighbouring columns a thread, a row a lane.
template <typename E, int PIECES>
__global__ void __launch_bounds__(256) k_slope(const float* z, const void* dy, int64_t ld_dy, int wide, int activation, int64_t m, int n, void* dz, int64_t ld, int64_t piece_stride) {
  using T = std::conditional_t<(PIECES > 1), float, E>;
  let_next_start();
  wait_for_previous();
  const int64_t groups = ld / 8, blocks = (m + 31) / 32, total = blocks * groups * 32;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t block = i / (groups * 32), rest = i - block * groups * 32, r = block * 32 + rest % 32;
    const int c = (int)(rest / 32) * 8;
    if (r >= m) continue;
    float v[8];
    const float4 z0 = *reinterpret_cast<const float4*>(z + kept_index(r, c, ld)), z1 = *reinterpret_cast<const float4*>(z + kept_index(r, c + 4, ld));
    const float zs[8] = {z0.x, z0.y, z0.z, z0.w, z1.x, z1.y, z1.z, z1.w};
    const T* row = static_cast<const T*>(dy) + r * ld_dy;
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < 8; k += N) {
      const uint4 raw = get16(row, c + k, n, wide);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if constexpr (PIECES > 1) v[k + j] = e[j];
        else v[k + j] = up(e[j]);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float a, da;
      activate_exact(activation, c + k < n ? zs[k] : 0.f, a, da);
      v[k] *= da;
    }
    put_operand<E, PIECES>(dz, piece_stride, r * ld + c, v);
  }
}

// Sums over rows of operand pieces: 64 columns and a share of the rows a CTA, 32 threads' rows added in a fixed order.
template <typename E, int PIECES>
__global__ void __launch_bounds__(256) k_column_sums(const Operand o, float* part, int n) {
  __shared__ float sums[32][65];
  let_next_start();
  wait_for_previous();
  const int q = threadIdx.x % 8, t = threadIdx.x / 8, col = blockIdx.x * 64 + q * 8;
  const int64_t r0 = o.rows * blockIdx.y / gridDim.y, r1 = o.rows * (blockIdx.y + 1) / gridDim.y;
  float v[8] = {};
  if (col < o.ld) {
    for (int64_t r = r0 + t; r < r1; r += 32) {
#pragma unroll
      for (int p = PIECES - 1; p >= 0; --p) {
        const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const E*>(o.data) + p * o.piece_stride + r * o.ld + col);
        const E* e = reinterpret_cast<const E*>(&raw);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += up(e[k]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) sums[t][q * 8 + k] = v[k];
  __syncthreads();
  if (threadIdx.x >= 64) return;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += sums[i][threadIdx.x];
  const int c = blockIdx.x * 64 + threadIdx.x;
  if (c < n) part[(int64_t)blockIdx.y * n + c] = s;
}
// How many CTAs share the rows: enough for every SM, no fewer than 128 rows each.
int row_shares(int64_t rows, int n) { return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 127) / 128, SMS * 4 / ((n + 63) / 64))); }

// Where everything of a call stands in its scratch; sizes alone with base = null.
struct Layout {
  int pieces;
  int64_t M, K, N, ld;
  Operand x, w, dz;
  float* part;
  float* sums;
  PackJobs jobs;
  int n_jobs;
  size_t total;

  Layout(const BnbLinear& c, const void* dy, int64_t dy_row, bool backward, uint8_t* base)
      : pieces(c.element == BNB_ELEM_F32 ? 3 : 1), M(c.rows), K(c.width), N(c.out), ld(round8(c.out)), dz{}, part(nullptr), sums(nullptr), jobs{}, n_jobs(0), total(0) {
    auto take = [&](size_t bytes) {
      uint8_t* at = base ? base + total : nullptr;
      total += round256(bytes);
      return at;
    };
    auto operand = [&](const void* p, int64_t rows, int64_t cols, int64_t row, int element) {
      if (pieces == 1 && element == c.element && lies_well(p, cols, row)) return Operand{p, rows, cols, row, 0};
      const int64_t to = round8(cols), stride = rows * to;
      void* at = take((size_t)pieces * stride * 2);
      jobs.job[n_jobs++] = {p, at, rows, row, stride, (int)cols, (int)to, element == BNB_ELEM_F32 ? 0 : 1};
      return Operand{at, rows, cols, to, stride};
    };
    x = operand(c.x, M, K, c.x_row, c.element);
    w = operand(c.weight, N, K, K, c.weight_element);
    const int t = pieces > 1 ? 6 : 1, most = pieces > 1 ? MOST<3> : MOST<1>;
    size_t parts = 0;
    if (!backward) {
      parts = part_bytes(M, N, K, 1, t, most);
    } else {
      dz = c.activation == BNB_ACT_NONE ? operand(dy, M, N, dy_row, c.element) : Operand{take((size_t)pieces * M * ld * 2), M, N, ld, M * ld};
      parts = std::max(part_bytes(M, K, N, 1, t, most), part_bytes(N, K, M, 1, t, most));
      sums = reinterpret_cast<float*>(take((size_t)row_shares(M, (int)N) * N * 4));
    }
    part = reinterpret_cast<float*>(take(parts));
  }
};

template <typename E, int PIECES>
int forward(const BnbLinear& c, const Layout& l, cudaStream_t st) {
  if (const int r = pack<E, PIECES>(l.jobs, l.n_jobs, st)) return r;
  Epilogue e{};
  e.out[0] = c.y;
  e.ld_out = l.N;
  e.out_kind = PIECES > 1 ? 0 : 1;
  e.ld_h = l.ld;
  e.g = keeps(c) ? static_cast<float*>(c.kept) : nullptr;
  e.activation = c.activation;
  e.bias = c.bias;
  e.bias_kind = c.bias_element == BNB_ELEM_F32 ? 0 : 1;
  e.other = c.residual;
  e.ld_other = c.residual_row;
  e.other_wide = reinterpret_cast<uintptr_t>(c.residual) % 16 == 0 && c.residual_row % (PIECES > 1 ? 4 : 8) == 0;
  return multiply<E, PIECES, false, false, Out::LINEAR>({{l.x, {}}, {l.w, {}}, 1}, l.M, l.N, l.K, 1, e, l.part, st);
}

template <typename E, int PIECES>
int backward(const BnbLinear& c, const BnbLinearGrads& g, const Layout& l, cudaStream_t st) {
  if (const int r = pack<E, PIECES>(l.jobs, l.n_jobs, st)) return r;
  int r = BNB_OK;
  if (c.activation != BNB_ACT_NONE) {
    const int wide = reinterpret_cast<uintptr_t>(g.dy) % 16 == 0 && g.dy_row % (PIECES > 1 ? 4 : 8) == 0;
    if (keeps(c)) {
      const int64_t work = (l.M + 31) / 32 * 32 * (l.ld / 8);
      r = launch_after(k_slope<E, PIECES>, dim3((unsigned)std::min<int64_t>((work + 255) / 256, SMS * 32)), 256, 0, st, static_cast<const float*>(c.kept), g.dy, g.dy_row, wide,
                       (int)c.activation, l.M, (int)l.N, const_cast<void*>(l.dz.data), l.ld, l.dz.piece_stride);
    } else if constexpr (PIECES == 1) {
      Epilogue e{};
      e.h = const_cast<void*>(l.dz.data);
      e.ld_h = l.ld;
      e.activation = c.activation;
      e.bias = c.bias;
      e.bias_kind = c.bias_element == BNB_ELEM_F32 ? 0 : 1;
      e.other = g.dy;
      e.ld_other = g.dy_row;
      e.other_wide = wide;
      r = multiply<E, PIECES, false, false, Out::SLOPE>({{l.x, {}}, {l.w, {}}, 1}, l.M, l.N, l.K, 1, e, nullptr, st);
    }
  }
  if (r) return r;
  Epilogue e{};
  if (g.dx) {
    e.out[0] = g.dx;
    e.ld_out = l.K;
    e.out_kind = PIECES > 1 ? 0 : 1;
    if (r = multiply<E, PIECES, false, true, Out::VALUES>({{l.dz, {}}, {l.w, {}}, 1}, l.M, l.K, l.N, 1, e, l.part, st); r) return r;
  }
  if (g.dweight) {
    e.out[0] = g.dweight;
    e.ld_out = l.K;
    e.out_kind = c.weight_element == BNB_ELEM_F32 ? 0 : 1;
    if (r = multiply<E, PIECES, true, true, Out::VALUES>({{l.dz, {}}, {l.x, {}}, 1}, l.N, l.K, l.M, 1, e, l.part, st); r) return r;
  }
  if (g.dbias) {
    const int shares = row_shares(l.M, (int)l.N);
    if (r = launch_after(k_column_sums<E, PIECES>, dim3((unsigned)((l.N + 63) / 64), shares), 256, 0, st, l.dz, l.sums, (int)l.N); r) return r;
    count_launch();
    k_add_parts<E><<<(unsigned)((l.N + 63) / 64), 256, 0, st>>>(l.sums, shares, l.N, 1, g.dbias, nullptr, c.bias_element == BNB_ELEM_F32 ? 0 : 1);
    return cudaGetLastError() == cudaSuccess ? BNB_OK : BNB_ERR_LAUNCH;
  }
  return BNB_OK;
}

}  // namespace
}  // namespace product
}  // namespace bnb

using namespace bnb;
using namespace bnb::product;

extern "C" size_t bnb_linear_kept_bytes(const BnbLinear* c) {
  if (check(c)) return 0;
  return keeps(*c) ? (size_t)round32(c->rows) * round32(c->out) * 4 : 0;
}

extern "C" size_t bnb_linear_scratch_bytes(const BnbLinear* c, int backward) {
  if (check(c) || c->rows == 0) return 0;
  // a dy that may have to be copied counts as copied: its address is not known yet
  return Layout(*c, reinterpret_cast<const void*>(1), c->out, backward != 0, nullptr).total;
}

extern "C" int bnb_linear_fwd(const BnbLinear* c, void* scratch, size_t scratch_bytes, void* stream) {
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

extern "C" int bnb_linear_bwd(const BnbLinear* c, const BnbLinearGrads* g, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int st = check(c)) return st;
  if (!g) return BNB_ERR_NULL_POINTER;
  const auto s = static_cast<cudaStream_t>(stream);
  if (c->rows == 0) {
    const size_t weight = (size_t)c->width * c->out * (c->weight_element == BNB_ELEM_F32 ? 4 : 2), bias = (size_t)c->out * (c->bias_element == BNB_ELEM_F32 ? 4 : 2);
    if (g->dweight && cudaMemsetAsync(g->dweight, 0, weight, s) != cudaSuccess) return BNB_ERR_LAUNCH;
    if (g->dbias && cudaMemsetAsync(g->dbias, 0, bias, s) != cudaSuccess) return BNB_ERR_LAUNCH;
    return BNB_OK;
  }
  if (!g->dy || (!c->kept && keeps(*c))) return BNB_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(c->kept) | reinterpret_cast<uintptr_t>(scratch) | reinterpret_cast<uintptr_t>(g->dx) | reinterpret_cast<uintptr_t>(g->dweight)) & 15)
    return BNB_ERR_MISALIGNED;
  const Layout l(*c, g->dy, g->dy_row, true, static_cast<uint8_t*>(scratch));
  if (!scratch || scratch_bytes < l.total) return BNB_ERR_SCRATCH_TOO_SMALL;
  return c->element == BNB_ELEM_F32 ? backward<__nv_bfloat16, 3>(*c, *g, l, s)
       : c->element == BNB_ELEM_BF16 ? backward<__nv_bfloat16, 1>(*c, *g, l, s) : backward<__half, 1>(*c, *g, l, s);
}
