// The linear layer of any size with what surrounds it, y = act(z) + r, z = x W^T + b, forward and backward:
//
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz,  dr = dy
//
// Forward is one launch: bias, activation and residual enter where the sums leave tensor memory (Out::LINEAR of product_tiles.cuh).  A product of two
// operations for each of rows x width x out forward and twice that backward: the tensor cores bound it, or, for few rows or a small width, memory.
//
// The backward of an activation reads what the forward kept of it: act'(z) in 16 bits, or z in float32 (see keeps_slopes).  Up to a width of some 400 computing z once more
// moves fewer bytes, but its second epilogue takes longer than they do: 65536 x 128 x 512 bfloat16 forward and backward 152 us, 145 with slopes kept
// (float16, with z kept: 151 and 158); 16384 x 512 x 2048 214 and 188; 8192 x 1024 x 4096 with z kept 250, with slopes 231.  dz is rounded to the operands' type, as an
// operand of the two products behind it; the bias's gradient sums it before that.  Without an activation dz is dy as it lies.
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

bool keeps(const BnbLinear& c) { return c.activation != BNB_ACT_NONE; }
// Whether the forward keeps act'(z) in 16 bits (see KEPT_SCALE) or z in float32.  Where dz becomes an operand of bfloat16 and its sums a bias's gradient of bfloat16, both are
// rounded to a relative 2^-9, which a slope's 2^-12 leaves as it is.  Beside float16's rounding, and in a bias's gradient in float32, it would show.
bool keeps_slopes(const BnbLinear& c) { return keeps(c) && c.element == BNB_ELEM_BF16 && (!c.bias || c.bias_element == BNB_ELEM_BF16); }

// ------------------------------------------------------------------ few rows

// A single token's layer reads its weight once and computes next to nothing: memory bounds it, and tiles of 128 rows of which one is
// there keep too few loads on their way (1 x 4096 x 4096 bfloat16: 13.0 us with tiles and a cut depth).  Here a CTA takes NB outputs, its threads the depth in pieces of
// 16 bytes; sums are float32, of a thread's pieces, then of a warp's lanes, then of the warps, in this order.  Float32 weights of a 16-bit
// call are rounded to its type on the way, as the tiles' copies are.
constexpr int FEW_THREADS = 256;
struct FewRows {
  const void* x;
  const void* weight;
  int64_t x_row;
  int rows, width, out, x_wide;
  Epilogue e;
};
template <typename T, typename E>   // eight values, of E or of float
__device__ __forceinline__ void eight(const T* at, F2 (&f)[4]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 raw = *reinterpret_cast<const uint4*>(at);
    f[0] = pair_up(raw.x, T{}), f[1] = pair_up(raw.y, T{}), f[2] = pair_up(raw.z, T{}), f[3] = pair_up(raw.w, T{});
  } else {
    const float4 a = reinterpret_cast<const float4*>(at)[0], b = reinterpret_cast<const float4*>(at)[1];
    f[0] = f2(a.x, a.y), f[1] = f2(a.z, a.w), f[2] = f2(b.x, b.y), f[3] = f2(b.z, b.w);
    if constexpr (!std::is_same<E, float>::value)
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = pair_up(pair_of<E>(f[i]), E{});
  }
}
template <typename E, typename W, int M, int NB>
__global__ void __launch_bounds__(FEW_THREADS) k_few_rows(const __grid_constant__ FewRows p) {
  __shared__ float sums[FEW_THREADS / 32][M * NB];
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n0 = blockIdx.x * NB, pieces = p.width / 8;
  const E* x = static_cast<const E*>(p.x);
  const W* w = static_cast<const W*>(p.weight);
  F2 acc[M][NB];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[m][n] = f2(0.f);
#pragma unroll 2
  for (int i = threadIdx.x; i < pieces; i += FEW_THREADS) {
    F2 ws[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n) eight<W, E>(w + (int64_t)min(n0 + n, p.out - 1) * p.width + i * 8, ws[n]);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const E* row = x + (int64_t)min(m, p.rows - 1) * p.x_row + i * 8;
      F2 xs[4];
      if (p.x_wide) {
        eight<E, E>(row, xs);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (sizeof(E) == 4) xs[k] = f2(row[2 * k], row[2 * k + 1]);
          else xs[k] = f2(up(row[2 * k]), up(row[2 * k + 1]));
        }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[m][n] = fma(xs[k], ws[n][k], acc[m][n]);
    }
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float2 s = halves(acc[m][n]);
      float v = s.x + s.y;
#pragma unroll
      for (int by = 16; by; by >>= 1) v += __shfl_xor_sync(0xffffffffu, v, by);
      if (lane == 0) sums[warp][m * NB + n] = v;
    }
  __syncthreads();
  const int m = threadIdx.x / NB, c = n0 + threadIdx.x % NB;
  if (threadIdx.x >= M * NB || m >= p.rows || c >= p.out) return;
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < FEW_THREADS / 32; ++i) v += sums[i][threadIdx.x];
  put_linear<E>(p.e, m, c, v);
}

// Whether a call goes there: pieces of 16 bytes everywhere in the weight, depth enough for the threads, and no more rows than pay.  4096 x 4096, us:
// bfloat16 1 row 9.1, 4 rows 11.8, 8 rows 27.9 (tiles: 13); float32 1 row 14.5, 8 rows 40 (tiles: 62).
bool few_rows(const BnbLinear& c) {
  return c.rows <= (c.element == BNB_ELEM_F32 ? 8 : 4) && c.width >= 1024 && c.width % 8 == 0 && reinterpret_cast<uintptr_t>(c.weight) % 16 == 0;
}
template <typename E, typename W>
int few(const FewRows& p, cudaStream_t st) {
  auto with = [&](auto kernel, int nb) { return launch_after(kernel, dim3((unsigned)((p.out + nb - 1) / nb)), FEW_THREADS, 0, st, p); };
  if (p.rows == 1) return with(k_few_rows<E, W, 1, 4>, 4);
  if (p.rows == 2) return with(k_few_rows<E, W, 2, 4>, 4);
  if constexpr (sizeof(E) == 4)
    if (p.rows > 4) return with(k_few_rows<E, W, 8, 2>, 2);
  return with(k_few_rows<E, W, 4, 4>, 4);
}

// ------------------------------------------------------------------ slopes and sums

// Sums over a warp of eight columns, of which every lane has a row: lane 4 c has column c's.  Lanes give away half of their columns a step while there are
// several: nine shuffles where one column after the other takes forty.
__device__ __forceinline__ float column_sum(const F2 (&v)[4], int lane) {
  auto swap = [](F2 x, int by) {
    const float2 f = halves(x);
    return f2(__shfl_xor_sync(0xffffffffu, f.x, by), __shfl_xor_sync(0xffffffffu, f.y, by));
  };
  const bool b16 = lane & 16, b8 = lane & 8, b4 = lane & 4;
  const F2 p = add(b16 ? v[2] : v[0], swap(b16 ? v[0] : v[2], 16)), q = add(b16 ? v[3] : v[1], swap(b16 ? v[1] : v[3], 16));   // columns 4-7 or 0-3
  const float2 r = halves(add(b8 ? q : p, swap(b8 ? p : q, 8)));
  float s = (b4 ? r.y : r.x) + __shfl_xor_sync(0xffffffffu, b4 ? r.x : r.y, 4);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  return s + __shfl_xor_sync(0xffffffffu, s, 1);
}

// dz from the kept slopes, or from the kept z.  A warp takes blocks of 32 x 32 of the same columns, eight warps side by side: what was kept, a row a lane, dy and dz as
// whole pieces of rows through shared memory (a lane's own row straight from memory is 32 lines a request).  sums: null, or (gridDim.y, n) sums over the
// rows before dz is rounded, a lane's rows one behind the other, then the lanes.
template <int PIECES> constexpr int SLOPE_CTAS = PIECES > 1 ? 1 : 2;   // of an SM
template <typename E, int PIECES, bool SLOPES>
__global__ void __launch_bounds__(256, SLOPE_CTAS<PIECES>) k_slope(const uint4* kept, const void* dy, int64_t ld_dy, int wide, int activation, int64_t m, int n, void* dz, int64_t ld,
                                                                       int64_t piece_stride, float* sums) {
  constexpr bool EXACT = PIECES > 1;
  using T = std::conditional_t<EXACT, float, E>;
  constexpr int N = 16 / sizeof(T), ROW = 32 / N, KEPT = SLOPES ? 4 : 8;   // pieces of a block's row: 4, float32 8
  __shared__ uint4 staged[8][32 * ROW];
  let_next_start();
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4* const mine = staged[warp];
  auto spot = [](int r, int q) { return r * ROW + (q ^ ((r / (8 / ROW)) % ROW)); };
  auto out = [](int r, int q) { return r * 4 + (q ^ ((r / 2) % 4)); };   // dz: four pieces of a row, whatever dy was
  const int64_t columns = (ld + 31) / 32, blocks = (m + 31) / 32;
  const int64_t column = (int64_t)blockIdx.x * 8 + warp;
  if (column >= columns) return;
  const int c0 = (int)column * 32;
  F2 total[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) total[k] = f2(0.f);
  uint4 held[KEPT], in[ROW];
  auto fetch = [&](int64_t b) {
    const uint4* from = kept + (b * columns + column) * KEPT * 32 + lane;
#pragma unroll
    for (int q = 0; q < KEPT; ++q) held[q] = from[q * 32];
#pragma unroll
    for (int q = 0; q < ROW; ++q) {
      const int64_t r = b * 32 + q * (32 / ROW) + lane / ROW;
      const int c = c0 + lane % ROW * N;
      in[q] = r < m && c < n ? get16(static_cast<const T*>(dy) + r * ld_dy, c, n, wide) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  for (int64_t b = blockIdx.y; b < blocks; b += gridDim.y) {
    const int64_t r0 = b * 32;
    fetch(b);
    __syncwarp();
#pragma unroll
    for (int q = 0; q < ROW; ++q) mine[spot(q * (32 / ROW) + lane / ROW, lane % ROW)] = in[q];
    __syncwarp();
    const int there = r0 + lane < m ? n - c0 : 0;   // columns of this row; nothing was kept behind the last row and column
    F2 v[16];
#pragma unroll
    for (int q = 0; q < 4; ++q) {   // eight columns
      F2 d[4], a;
      if constexpr (SLOPES) {
        const uint32_t raw[4] = {held[q].x, held[q].y, held[q].z, held[q].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 s = halves(pair_up(raw[k], __half{}));
          d[k] = mul(f2(8 * q + 2 * k < there ? s.x : 0.f, 8 * q + 2 * k + 1 < there ? s.y : 0.f), f2(1.f / KEPT_SCALE));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4 z = held[2 * q + k / 2];
          const float x = __uint_as_float(k % 2 ? z.z : z.x), y = __uint_as_float(k % 2 ? z.w : z.y);
          activate<EXACT, true>(activation, f2(8 * q + 2 * k < there ? x : 0.f, 8 * q + 2 * k + 1 < there ? y : 0.f), a, d[k]);
        }
      }
      if constexpr (EXACT) {
        const uint4 raw[2] = {mine[spot(lane, 2 * q)], mine[spot(lane, 2 * q + 1)]};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          v[4 * q + k] = mul(d[k], k % 2 ? f2(__uint_as_float(raw[k / 2].z), __uint_as_float(raw[k / 2].w)) : f2(__uint_as_float(raw[k / 2].x), __uint_as_float(raw[k / 2].y)));
      } else {
        uint4* const at = &mine[spot(lane, q)];   // dz's place too
        const uint4 raw = *at;
        const uint32_t g[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * q + k] = mul(d[k], pair_up(g[k], E{}));
        *at = make_uint4(pair_of<E>(v[4 * q]), pair_of<E>(v[4 * q + 1]), pair_of<E>(v[4 * q + 2]), pair_of<E>(v[4 * q + 3]));
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) total[4 * q + k] = add(total[4 * q + k], v[4 * q + k]);
    }
#pragma unroll
    for (int piece = 0; piece < PIECES; ++piece) {
      __syncwarp();
      if constexpr (EXACT) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t bits[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            bits[k] = pair_of<E>(v[4 * q + k]);
            v[4 * q + k] = add(v[4 * q + k], mul(pair_up(bits[k], E{}), f2(-1.f)));
          }
          mine[out(lane, q)] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
        }
        __syncwarp();
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = q * 8 + lane / 4, c = c0 + lane % 4 * 8;
        if (r0 + r < m && c < ld) *reinterpret_cast<uint4*>(static_cast<E*>(dz) + piece * piece_stride + (r0 + r) * ld + c) = mine[out(r, lane % 4)];
      }
    }
  }
  if (!sums) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const F2 eight[4] = {total[4 * q], total[4 * q + 1], total[4 * q + 2], total[4 * q + 3]};
    const float s = column_sum(eight, lane);
    const int c = c0 + 8 * q + lane / 4;
    if (lane % 4 == 0 && c < n) sums[(int64_t)blockIdx.y * n + c] = s;
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
    constexpr int UNROLL = 4;   // rows whose loads are on their way together
    const E* from = static_cast<const E*>(o.data) + col;
    auto add_row = [&](const uint4 (&raw)[PIECES]) {
#pragma unroll
      for (int p = PIECES - 1; p >= 0; --p) {
        const E* e = reinterpret_cast<const E*>(&raw[p]);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += up(e[k]);
      }
    };
    int64_t r = r0 + t;
    for (; r + (UNROLL - 1) * 32 < r1; r += UNROLL * 32) {
      uint4 raw[UNROLL][PIECES];
#pragma unroll
      for (int i = 0; i < UNROLL; ++i)
#pragma unroll
        for (int p = 0; p < PIECES; ++p) raw[i][p] = *reinterpret_cast<const uint4*>(from + p * o.piece_stride + (r + 32 * i) * o.ld);
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) add_row(raw[i]);
    }
    for (; r < r1; r += 32) {
      uint4 raw[PIECES];
#pragma unroll
      for (int p = 0; p < PIECES; ++p) raw[p] = *reinterpret_cast<const uint4*>(from + p * o.piece_stride + r * o.ld);
      add_row(raw);
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
// How many CTAs share the rows: six an SM, no fewer than 128 rows each.
int row_shares(int64_t rows, int n) { return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 127) / 128, SMS * 6 / ((n + 63) / 64))); }

// How many CTAs share the row blocks of k_slope: four an SM.
int slope_shares(int64_t rows, int64_t ld) { return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 31) / 32, SMS * 4 / ((ld + 255) / 256))); }

// Where everything of a call stands in its scratch; sizes alone with base = null.
struct Layout {
  int pieces;
  int64_t M, K, N, ld;
  Operand x, w, dz;
  float* part;
  float* sums;     // of a bias's gradient: shares of rows
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
      parts = part_bytes(M, N, K, 1, t, most_of_linear(pieces, (int)((K + BK - 1) / BK)));
    } else {
      dz = c.activation == BNB_ACT_NONE ? operand(dy, M, N, dy_row, c.element) : Operand{take((size_t)pieces * M * ld * 2), M, N, ld, M * ld};
      parts = std::max(part_bytes(M, K, N, 1, t, most), part_bytes(N, K, M, 1, t, most));
      sums = reinterpret_cast<float*>(take((size_t)std::max(row_shares(M, (int)N), slope_shares(M, ld)) * N * 4));
    }
    part = reinterpret_cast<float*>(take(parts));
  }
};

Epilogue ends_of(const BnbLinear& c) {
  const bool floats = c.element == BNB_ELEM_F32;
  Epilogue e{};
  e.out[0] = c.y;
  e.ld_out = c.out;
  e.out_kind = floats ? 0 : 1;
  e.ld_h = round8(c.out);
  if (keeps_slopes(c)) e.slopes = static_cast<__half*>(c.kept);
  else if (keeps(c)) e.g = static_cast<float*>(c.kept);
  e.activation = c.activation;
  e.bias = c.bias;
  e.bias_kind = c.bias_element == BNB_ELEM_F32 ? 0 : 1;
  e.other = c.residual;
  e.ld_other = c.residual_row;
  e.other_wide = reinterpret_cast<uintptr_t>(c.residual) % 16 == 0 && c.residual_row % (floats ? 4 : 8) == 0;
  return e;
}
template <typename E, int PIECES>
int forward(const BnbLinear& c, const Layout& l, cudaStream_t st) {
  if (const int r = pack<E, PIECES>(l.jobs, l.n_jobs, st)) return r;
  return multiply<E, PIECES, false, false, Out::LINEAR>({{l.x, {}}, {l.w, {}}, 1}, l.M, l.N, l.K, 1, ends_of(c), l.part, st);
}
template <typename E>
int forward_few(const BnbLinear& c, cudaStream_t st) {
  const int per = sizeof(E) == 4 ? 4 : 8;
  const FewRows p{c.x, c.weight, c.x_row, (int)c.rows, c.width, c.out, reinterpret_cast<uintptr_t>(c.x) % 16 == 0 && c.x_row % per == 0, ends_of(c)};
  return c.weight_element == BNB_ELEM_F32 ? few<E, float>(p, st) : few<E, E>(p, st);
}

template <typename E, int PIECES>
int backward(const BnbLinear& c, const BnbLinearGrads& g, const Layout& l, cudaStream_t st) {
  if (const int r = pack<E, PIECES>(l.jobs, l.n_jobs, st)) return r;
  int r = BNB_OK, shares = 0;   // of sums that are there already
  if (keeps(c)) {
    const int wide = reinterpret_cast<uintptr_t>(g.dy) % 16 == 0 && g.dy_row % (PIECES > 1 ? 4 : 8) == 0;
    shares = slope_shares(l.M, l.ld);
    auto slope = [&](auto kernel) {
      return launch_after(kernel, dim3((unsigned)((l.ld + 255) / 256), (unsigned)shares), 256, 0, st, static_cast<const uint4*>(c.kept), g.dy, g.dy_row, wide,
                          (int)c.activation, l.M, (int)l.N, const_cast<void*>(l.dz.data), l.ld, l.dz.piece_stride, g.dbias ? l.sums : nullptr);
    };
    if constexpr (std::is_same<E, __nv_bfloat16>::value && PIECES == 1) r = keeps_slopes(c) ? slope(k_slope<E, 1, true>) : slope(k_slope<E, 1, false>);
    else r = slope(k_slope<E, PIECES, false>);
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
    if (!shares) {
      shares = row_shares(l.M, (int)l.N);
      if (r = launch_after(k_column_sums<E, PIECES>, dim3((unsigned)((l.N + 63) / 64), (unsigned)shares), 256, 0, st, l.dz, l.sums, (int)l.N); r) return r;
    }
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
  return keeps(*c) ? (size_t)round32(c->rows) * round32(c->out) * (keeps_slopes(*c) ? 2 : 4) : 0;
}

extern "C" size_t bnb_linear_scratch_bytes(const BnbLinear* c, int backward) {
  if (check(c) || c->rows == 0 || (!backward && few_rows(*c))) return 0;
  // a dy that may have to be copied counts as copied: its address is not known yet
  return Layout(*c, reinterpret_cast<const void*>(1), c->out, backward != 0, nullptr).total;
}

extern "C" int bnb_linear_fwd(const BnbLinear* c, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int st = check(c)) return st;
  if (c->rows == 0) return BNB_OK;
  if (!c->y) return BNB_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(c->y) | reinterpret_cast<uintptr_t>(c->kept) | reinterpret_cast<uintptr_t>(scratch)) & 15) return BNB_ERR_MISALIGNED;
  const auto s = static_cast<cudaStream_t>(stream);
  if (few_rows(*c)) return c->element == BNB_ELEM_F32 ? forward_few<float>(*c, s) : c->element == BNB_ELEM_BF16 ? forward_few<__nv_bfloat16>(*c, s) : forward_few<__half>(*c, s);
  const Layout l(*c, nullptr, 0, false, static_cast<uint8_t*>(scratch));
  if (!scratch || scratch_bytes < l.total) return BNB_ERR_SCRATCH_TOO_SMALL;
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
