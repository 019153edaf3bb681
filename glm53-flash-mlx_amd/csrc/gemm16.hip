// The shape of a tiled product: output tile and parts of the contraction.
#include <initializer_list>

#include "gemm16.h"

namespace glm53 {
namespace {

struct Shape {
  Gemm16Tile tile;
  int rows, cols, step;
  int64_t slots;
  float step_us, step_full_us, fixed_us;
};
constexpr Shape kShapes[] = {{kTile64, 64, 128, 128, 256, 1.1f, 1.1f, 4.0f},
                             {kTile128, 128, 128, 64, 512, 0.95f, 1.05f, 6.0f},
                             {kTile256, 256, 256, 64, 256, 1.6f, 1.6f, 12.0f}};
// 4-bit products, whose vector instructions and MFMAs take turns: smaller tiles,
// three a CU, where the large ones are few (300 x 4096 x 4096: 39.6 us; 46.6 in 64 x
// 128 tiles of two blocks a step, 43.4 in 128 x 128 tiles).  256 x 256 results and a
// group's sums do not fit the registers.
constexpr Shape kScaledShapes[] = {{kTile64, 64, 128, 64, 768, 0.62f, 1.2f, 5.0f},
                                   {kTile128, 128, 128, 64, 512, 0.95f, 1.4f, 5.0f}};

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t tiles_of(const Gemm16Args& g, const Shape& s, int planes) {
  int64_t tiles = 0;
  for (int q = 0; q < g.problems; ++q) tiles += cdiv(g.pair[q].m, s.rows) * cdiv(g.pair[q].n, s.cols / planes);
  return tiles;
}

// By the time that each shape is expected to take, from what the shapes
// measured over 16 to 8,192 rows, 1,000 to 8,192 columns and contractions of
// 1,000 to 8,192 (bf16, row form):
//   tile        a step    workgroups at once   and, once a round
//   64 x 128    1.1 us of 128 k   256 (1 a CU)   4 us
//   128 x 128   0.95 to 1.05 of 64   512 (2 a CU)   6 us
//   256 x 256   1.6 us of 64      256 (1 a CU)   12 us
// The large tile has the best rate (1.35 PFLOP/s between its start and end)
// and needs about 256 tiles; a small batch has few tiles, and splitting the
// contraction fills the chip at the price of the FP32 partial results written
// and read again, 8 bytes an output and part at 6.5 TB/s, and a second launch, 3 us.
// Every epilogue is priced alike: that of SwiGLU's gradient, which reads G and U
// (134 MB at 8,192 x 2048) with all tiles there at once, takes a quarter of its
// product's time.
// 300 x 4096 x 4096 in 128 x 128 tiles: 66 us whole, 44 in 2 parts, 35 in 4;
// 2,048 rows: 71 whole, 91 in 2; 4,096 rows: 135, and 113 in 256 x 256 tiles.
template <int COUNT>
Gemm16Plan plan_of(const Gemm16Args& g, bool pair_b, const Shape (&shapes)[COUNT]) {
  const int planes = pair_b ? 2 : 1;
  int64_t outputs = 0;
  for (int q = 0; q < g.problems; ++q) outputs += g.pair[q].m * partial_ld(g.pair[q].n) * planes;
  Gemm16Plan best{};
  for (const Shape& s : shapes) {
    const int64_t tiles = tiles_of(g, s, planes), steps = cdiv(g.k, s.step) * g.segments;
    for (int most : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (most > 1 && steps < 2 * most) break;
      const int splits = used_splits(steps, most);
      const int64_t units = tiles * splits, rounds = cdiv(units, s.slots);
      float us = static_cast<float>(rounds * cdiv(steps, splits)) * (units > 256 ? s.step_full_us : s.step_us);
      us += s.tile == kTile256 ? static_cast<float>(rounds) * s.fixed_us : s.fixed_us;
      if (splits > 1) us += 3.0f + 8.0f * static_cast<float>(outputs) * static_cast<float>(splits) / 6.5e6f;
      if (best.splits == 0 || us < best.us) best = {s.tile, splits, splits > 1 ? outputs * splits : 0, us};
    }
  }
  return best;
}

}  // namespace

Gemm16Plan gemm16_plan(const Gemm16Args& g, bool pair_b) { return plan_of(g, pair_b, kShapes); }
Gemm16Plan gemm16_plan_scaled(const Gemm16Args& g) { return plan_of(g, false, kScaledShapes); }

}  // namespace glm53
