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
#include "product_calls.cuh"

namespace bnb {
namespace product {
namespace {

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
  if (const int r = pack<E, PIECES>(l.jobs, l.n_jobs, st)) return r;
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
  if (const int r = pack<E, PIECES>(l.jobs, l.n_jobs, st)) return r;
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
