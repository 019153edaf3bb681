// Gated MLP in bf16 weights, y = (silu(min(x Wg^T, L)) clip(x Wu^T, -L, L))
// Wd^T, and its gradients, as products of gemm16.h: gate and up projections
// with the activation and the product as one kernel's epilogue, the down
// projection, and backward
//   dh = dy Wd, in whose epilogue dG, dU and h are made,
//   dx = dG Wg + dU Wu (one contraction over both),
//   dWg = dG^T x, dWu = dU^T x, dWd = dy^T h (one launch).
// Operands of a product are bf16 and its sums FP32: h, dG and dU are rounded
// to bf16 once, as MFMA operands, everything before them is FP32.
#include "gated.h"
#include "gemm16.h"

namespace glm53 {
namespace {

size_t round_up(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <class G>
hipError_t launch_tiles(Gemm16Args g, hipStream_t st) {
  g.tiles = 0;
  for (int q = 0; q < g.problems; ++q) g.tiles += cdiv(g.pair[q].m, G::BM) * cdiv(g.pair[q].n, G::kColumns);
  g.group_m = 8;
  gemm16_kernel<G><<<static_cast<uint32_t>(g.tiles * g.splits), G::kThreads, G::kLds, st>>>(g);
  return hipGetLastError();
}

template <bool A_COLUMN, OperandForm B, Gemm16Epilogue EPI>
hipError_t launch_product(Gemm16Args g, hipStream_t st) {
  g.splits = 1;
  return launch_tiles<Gemm16<2, 2, 4, 4, A_COLUMN, B, EPI>>(g, st);
}

Gemm16Pair pair(const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb, uint16_t* out, int64_t m, int64_t n) {
  return {a, b, out, lda, ldb, n, m, n};
}

Gemm16Args product(int64_t k) {
  Gemm16Args g{};
  g.k = k;
  g.problems = g.segments = 1;
  return g;
}

}  // namespace

size_t gated_space(int64_t rows, int64_t hidden, int64_t inter, bool backward) {
  const size_t plane = round_up(2 * static_cast<size_t>(rows) * static_cast<size_t>(inter));
  return backward ? 3 * plane : plane;
}

hipError_t launch_gated(const GatedArgs& a, hipStream_t st) {
  uint16_t* h = static_cast<uint16_t*>(a.space);
  Gemm16Args g = product(a.hidden);
  g.pair[0] = pair(a.x, a.hidden, a.wg, a.hidden, h, a.rows, a.inter);
  g.pair[1] = g.pair[0];
  g.pair[1].b = a.wu;
  g.limit = a.limit;
  g.gate = a.gate;
  g.up = a.up;
  if (hipError_t e = launch_product<false, kRow, kSwiglu>(g, st); e != hipSuccess) return e;
  Gemm16Args d = product(a.inter);
  d.pair[0] = pair(h, a.inter, a.wd, a.inter, a.y, a.rows, a.hidden);
  return launch_product<false, kRow, kStore>(d, st);
}

hipError_t launch_gated_backward(const GatedArgs& a, hipStream_t st) {
  uint8_t* space = static_cast<uint8_t*>(a.space);
  const size_t plane = gated_space(a.rows, a.hidden, a.inter, false);
  uint16_t* dg = reinterpret_cast<uint16_t*>(space);
  uint16_t* du = reinterpret_cast<uint16_t*>(space + plane);
  uint16_t* h = reinterpret_cast<uint16_t*>(space + 2 * plane);
  Gemm16Args g = product(a.hidden);
  g.pair[0] = pair(a.dy, a.hidden, a.wd, a.inter, nullptr, a.rows, a.inter);
  g.limit = a.limit;
  g.gate = a.gate;
  g.up = a.up;
  g.d_gate = dg;
  g.d_up = du;
  g.h = a.d_wd != nullptr ? h : nullptr;
  if (hipError_t e = launch_product<false, kColumn, kSwigluGrad>(g, st); e != hipSuccess) return e;
  if (a.dx != nullptr) {
    Gemm16Args x = product(a.inter);
    x.segments = 2;
    x.pair[0] = pair(dg, a.inter, a.wg, a.hidden, a.dx, a.rows, a.hidden);
    x.pair[1] = pair(du, a.inter, a.wu, a.hidden, a.dx, a.rows, a.hidden);
    if (hipError_t e = launch_product<false, kColumn, kStore>(x, st); e != hipSuccess) return e;
  }
  Gemm16Args w = product(a.rows);
  w.problems = 0;
  if (a.d_wg) w.pair[w.problems++] = pair(dg, a.inter, a.x, a.hidden, a.d_wg, a.inter, a.hidden);
  if (a.d_wu) w.pair[w.problems++] = pair(du, a.inter, a.x, a.hidden, a.d_wu, a.inter, a.hidden);
  if (a.d_wd) w.pair[w.problems++] = pair(a.dy, a.hidden, h, a.inter, a.d_wd, a.hidden, a.inter);
  if (w.problems == 0) return hipSuccess;
  return launch_product<true, kColumn, kStore>(w, st);
}

}  // namespace glm53
