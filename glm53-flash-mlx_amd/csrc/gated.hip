// Gated MLP in bf16 weights, y = (silu(min(x Wg^T, L)) clip(x Wu^T, -L, L))
// Wd^T, and its gradients, as products of gemm16.h: gate and up projections
// with the activation and the product as one kernel's epilogue, the down
// projection, and backward
//   dh = dy Wd, in whose epilogue dG and dU are made,
//   dx = dG Wg + dU Wu (one contraction over both),
//   dWg = dG^T x, dWu = dU^T x, dWd = dy^T h.
// Operands of a product are bf16 and its sums FP32: h, dG and dU are rounded
// to bf16 once, as MFMA operands, everything before them is FP32.  Over many
// rows those roundings average out to about the results' own; up to kFewRows
// rows, where a gradient holds few of them, they are carried as a high and a
// low bf16 part, both multiplied.
#include <algorithm>
#include <initializer_list>

#include "gated.h"
#include "gemm16.h"

namespace glm53 {
namespace {

size_t round_up(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ------------------------------------------------------------- few rows ---
//
// Few rows: the call costs the weights' bytes.  A workgroup makes 16
// weight rows' results, its wavefronts taking parts of the contraction, joined
// in LDS in their order; weights go from memory to the MFMA through registers
// alone, a wavefront's loads all under way at once.  Rows of x are the MFMA's
// rows, so a lane's four results belong to one weight row.  1 x 4096 x 2048:
// 7.9 us for gate and up, 5.9 for down, 50 MB at 3.6 TB/s; 1 x 7168 x 18432: 145
// us, 5.5 TB/s.
constexpr int kFewRows = 16;
constexpr int kFewWaves = 16;
// K steps of 32 that a wavefront has in flight (1 x 4096 x 2048 by 16 wavefronts: 2
// steps 14.0 us, 4 15.1, 8 15.3; by 8 wavefronts 4 steps 16.1, 8 15.6)
constexpr int kFewSteps = 2;

template <int V>
struct Int {
  static constexpr int value = V;
};

// y[m, n] = sum_k x[m, k] w(n)[k] of the 16 rows that row(n) gives, per wavefront
// into part.  X: float rows are split into two bf16 operands, which keep 16 of
// their 24 bits, and whose products are added at the end: an infinite weight
// times a low part, of either sign or zero, is left out.
template <int MT, class X>
__device__ __forceinline__ void few_rows(const X* x, int rows, const uint16_t* w_row, int K, float (*part)[16 * MT][16]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int steps = (K + 31) / 32, each = (steps + kFewWaves - 1) / kFewWaves;
  const int first = wave * each, last = first + each < steps ? first + each : steps;
  const X* x_row[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) x_row[i] = x + static_cast<int64_t>(16 * i + r < rows ? 16 * i + r : rows - 1) * K + 8 * q;
  w_row += 8 * q;
  f32x4 acc[MT], low[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = low[i] = (f32x4){0, 0, 0, 0};
  constexpr bool kFloat = sizeof(X) == 4;
  constexpr int kHalves = kFloat ? 2 : 1;
  const auto multiply = [&](f32x4& acc, f32x4& low, const u32x4 (&v)[kHalves], const u32x4& w, bool in) {
    const u32x4 zero = {0, 0, 0, 0};
    const bf16x8 b = __builtin_bit_cast(bf16x8, in ? w : zero);
    if constexpr (kFloat) {
      u32x4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f0 = __uint_as_float(v[i >> 1][2 * (i & 1)]), f1 = __uint_as_float(v[i >> 1][2 * (i & 1) + 1]);
        const uint16_t h0 = f32_to_bf16(f0), h1 = f32_to_bf16(f1);
        hi[i] = h0 | static_cast<uint32_t>(h1) << 16;
        lo[i] = f32_to_bf16(low_part(f0, h0)) | static_cast<uint32_t>(f32_to_bf16(low_part(f1, h1))) << 16;
      }
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, in ? hi : zero), b, acc, 0, 0, 0);
      low = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, in ? lo : zero), b, low, 0, 0, 0);
    } else {
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, in ? v[0] : zero), b, acc, 0, 0, 0);
    }
  };
  // U whole steps, every load on its way before the first is used
  const auto batch = [&](int s, auto count) {
    constexpr int U = decltype(count)::value;
    u32x4 w[U], v[U][MT][kHalves];
    const uint16_t* wb = w_row + 32 * s;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = *reinterpret_cast<const u32x4*>(wb + 32 * u);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < kHalves; ++h) v[u][i][h] = *reinterpret_cast<const u32x4*>(x_row[i] + 32 * s + 32 * u + 4 * h);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i) multiply(acc[i], low[i], v[u][i], w[u], true);
  };
  int s = first;
  const int whole_last = last < K / 32 ? last : K / 32;
  for (; s + kFewSteps <= whole_last; s += kFewSteps) batch(s, Int<kFewSteps>{});
  for (; s < whole_last; ++s) batch(s, Int<1>{});
  if (s < last) {  // the end of K: what lies past it reads the step's first columns and is left out
    const bool in = 32 * s + 8 * q < K;
    const int at = in ? 32 * s : 32 * s - 8 * q;
    const u32x4 w = *reinterpret_cast<const u32x4*>(w_row + at);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      u32x4 v[kHalves];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) v[h] = *reinterpret_cast<const u32x4*>(x_row[i] + at + 4 * h);
      multiply(acc[i], low[i], v, w, in);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      part[wave][16 * i + 4 * q + e][r] = kFloat && fabsf(low[i][e]) < INFINITY ? acc[i][e] + low[i][e] : acc[i][e];
  __syncthreads();
}

template <int MT>
__device__ __forceinline__ float few_sum(const float (*part)[16 * MT][16], int m, int n) {
  float v = part[0][m][n];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) v += part[w][m][n];
  return v;
}

// 8 gate and the 8 up rows of the same outputs a workgroup; h goes on in FP32,
// for few_rows to split.
template <int MT>
__global__ __launch_bounds__(64 * kFewWaves) void few_gate_up_kernel(GatedArgs a, float* h) {
  __shared__ float part[kFewWaves][16 * MT][16];
  const int r = threadIdx.x & 15;
  const int64_t n0 = 8 * static_cast<int64_t>(blockIdx.x);
  const uint16_t* w = (r < 8 ? a.wg : a.wu) + (n0 + (r & 7)) * a.hidden;
  few_rows<MT>(a.x, static_cast<int>(a.rows), w, static_cast<int>(a.hidden), part);
  if (threadIdx.x >= 128 * MT) return;
  const int n = threadIdx.x & 7, m = threadIdx.x >> 3;
  if (m >= a.rows) return;
  const float gate = few_sum<MT>(part, m, n), up = few_sum<MT>(part, m, 8 + n);
  const int64_t at = m * a.inter + n0 + n;
  if (a.gate != nullptr) {
    a.gate[at] = gate;
    a.up[at] = up;
  }
  const float c = clamp_gate(gate, a.limit), v = c * sigmoid_f32(c) * clamp_up(up, a.limit);
  h[at] = v;
  if (a.h != nullptr) {
    const uint16_t high = f32_to_bf16(v);
    a.h[at] = high;
    if (MT == 1) a.h[a.rows * a.inter + at] = f32_to_bf16(low_part(v, high));
  }
}

template <int MT>
__global__ __launch_bounds__(64 * kFewWaves) void few_down_kernel(GatedArgs a, const float* h) {
  __shared__ float part[kFewWaves][16 * MT][16];
  const int64_t n0 = 16 * static_cast<int64_t>(blockIdx.x);
  const int r = threadIdx.x & 15, cols = a.hidden - n0 < 16 ? 8 : 16;  // hidden is a multiple of 8
  few_rows<MT>(h, static_cast<int>(a.rows), a.wd + (n0 + (r < cols ? r : cols - 1)) * a.inter, static_cast<int>(a.inter), part);
  if (threadIdx.x >= 256 * MT) return;
  const int n = threadIdx.x & 15, m = threadIdx.x >> 4;
  if (m < a.rows && n < cols) a.y[m * a.hidden + n0 + n] = f32_to_bf16(few_sum<MT>(part, m, n));
}

template <int MT>
hipError_t launch_few(const GatedArgs& a, hipStream_t st) {
  float* h = static_cast<float*>(a.space);
  few_gate_up_kernel<MT><<<static_cast<uint32_t>(a.inter / 8), 64 * kFewWaves, 0, st>>>(a, h);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  few_down_kernel<MT><<<static_cast<uint32_t>(cdiv(a.hidden, 16)), 64 * kFewWaves, 0, st>>>(a, h);
  return hipGetLastError();
}

// From 17 to 32 rows two MFMA rows share the weights, while no kernel has more
// than a workgroup a CU; x and h, which come to every workgroup from L2, then
// cost more than the tiled product's partial results (17 and 32 rows, 4096 x
// 2048: 21 and 27 us here, 28 and 30 tiled; 4096 x 4096: 37 and 48, 36 and 37;
// 24 rows, 7168 x 2048: 42, 36).
bool few(int64_t rows, int64_t hidden, int64_t inter) {
  return rows <= kFewRows || (rows <= 32 && hidden <= 4096 && inter <= 2048);
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

// Parts that h, dG and dU are carried in, one after the other.
int parts(int64_t rows) { return rows <= kFewRows ? 2 : 1; }

// Bytes of h, dG or dU.
size_t plane_bytes(int64_t rows, int64_t inter) {
  return round_up(2 * static_cast<size_t>(parts(rows)) * static_cast<size_t>(rows) * static_cast<size_t>(inter));
}

// The workspace: forward h where it is not kept, backward dG and dU; then the
// partial results of one product at a time.
struct Space {
  uint16_t *h, *dg, *du;
  float* partial;
  int64_t room;  // floats at partial
};
Space carve(const GatedArgs& a, bool backward) {
  uint8_t* p = static_cast<uint8_t*>(a.space);
  const size_t plane = plane_bytes(a.rows, a.inter);
  Space s{};
  s.h = a.h;
  if (backward) {
    s.dg = reinterpret_cast<uint16_t*>(p);
    s.du = reinterpret_cast<uint16_t*>(p + plane);
  } else if (s.h == nullptr) {
    s.h = reinterpret_cast<uint16_t*>(p);
  }
  const size_t before = (backward ? 2 : s.h == a.h ? 0 : 1) * plane;
  s.partial = reinterpret_cast<float*>(p + before);
  s.room = static_cast<int64_t>((a.space_bytes - before) / sizeof(float));
  return s;
}

Gemm16Args gate_up(const GatedArgs& a, const Space& s) {
  Gemm16Args g = product(a.hidden);
  g.pair[0] = pair(a.x, a.hidden, a.wg, a.hidden, s.h, a.rows, a.inter);
  g.pair[1] = g.pair[0];
  g.pair[1].b = a.wu;
  g.limit = a.limit;
  g.gate = a.gate;
  g.up = a.up;
  g.partial = s.partial;
  g.room = s.room;
  return g;
}
Gemm16Args down(const GatedArgs& a, const Space& s) {
  Gemm16Args g = product(a.inter);
  g.pair[0] = pair(s.h, a.inter, a.wd, a.inter, a.y, a.rows, a.hidden);
  g.partial = s.partial;
  g.room = s.room;
  return g;
}
Gemm16Args hidden_grad(const GatedArgs& a, const Space& s) {
  Gemm16Args g = product(a.hidden);
  g.pair[0] = pair(a.dy, a.hidden, a.wd, a.inter, nullptr, a.rows, a.inter);
  g.limit = a.limit;
  g.gate = a.gate;
  g.up = a.up;
  g.d_gate = s.dg;
  g.d_up = s.du;
  g.low = parts(a.rows) == 2 ? a.rows * a.inter : 0;
  g.partial = s.partial;
  g.room = s.room;
  return g;
}
Gemm16Args input_grad(const GatedArgs& a, const Space& s) {
  Gemm16Args g = product(a.inter);
  g.segments = 0;
  for (int part = 0; part < parts(a.rows); ++part) {
    const int64_t at = part * a.rows * a.inter;
    g.pair[g.segments++] = pair(s.dg + at, a.inter, a.wg, a.hidden, a.dx, a.rows, a.hidden);
    g.pair[g.segments++] = pair(s.du + at, a.inter, a.wu, a.hidden, a.dx, a.rows, a.hidden);
  }
  g.partial = s.partial;
  g.room = s.room;
  return g;
}
Gemm16Pair weight_grad(const GatedArgs& a, const Space& s, int which, int part) {
  const int64_t at = part * a.rows * a.inter;
  if (which == 1) return pair(s.dg + at, a.inter, a.x, a.hidden, a.d_wg, a.inter, a.hidden);
  if (which == 2) return pair(s.du + at, a.inter, a.x, a.hidden, a.d_wu, a.inter, a.hidden);
  return pair(a.dy, a.hidden, s.h + at, a.inter, a.d_wd, a.hidden, a.inter);
}
// Those of the weights' gradients, dWg, dWu and dWd, that `which` (bits 1, 2
// and 4) names; a single one where they are carried in two parts.
Gemm16Args weight_grads(const GatedArgs& a, const Space& s, int which) {
  Gemm16Args g = product(a.rows);
  g.partial = s.partial;
  g.room = s.room;
  if (parts(a.rows) == 2) {
    g.segments = 2;
    for (int part = 0; part < 2; ++part) g.pair[part] = weight_grad(a, s, which, part);
    return g;
  }
  g.problems = 0;
  for (int one : {1, 2, 4})
    if (which & one) g.pair[g.problems++] = weight_grad(a, s, one, 0);
  return g;
}

int64_t most(std::initializer_list<int64_t> v) { return std::max(v); }

}  // namespace

size_t gated_space(int64_t rows, int64_t hidden, int64_t inter, bool backward) {
  const size_t plane = plane_bytes(rows, inter);
  GatedArgs a{};
  a.rows = rows;
  a.hidden = hidden;
  a.inter = inter;
  const Space s{};
  if (backward) {
    int64_t partial = most({gemm16_plan(hidden_grad(a, s), false).partial, gemm16_plan(input_grad(a, s), false).partial});
    for (int which = 1; which < 8; ++which) {  // dWd is [hidden, inter], the others [inter, hidden]: their tiles differ
      if (parts(rows) == 2 && (which & (which - 1)) != 0) continue;
      partial = most({partial, gemm16_plan(weight_grads(a, s, which), false).partial});
    }
    return 2 * plane + sizeof(float) * static_cast<size_t>(partial);
  }
  if (few(rows, hidden, inter)) return round_up(4 * static_cast<size_t>(rows) * static_cast<size_t>(inter));  // h in FP32
  const int64_t partial = most({gemm16_plan(gate_up(a, s), true).partial, gemm16_plan(down(a, s), false).partial});
  return plane + sizeof(float) * static_cast<size_t>(partial);
}

hipError_t launch_gated(const GatedArgs& a, hipStream_t st) {
  if (few(a.rows, a.hidden, a.inter)) return a.rows <= kFewRows ? launch_few<1>(a, st) : launch_few<2>(a, st);
  const Space s = carve(a, false);
  const Gemm16Args g = gate_up(a, s), d = down(a, s);
  if (hipError_t e = gemm16<false, kRow, kSwiglu>(g, gemm16_plan(g, true), st); e != hipSuccess) return e;
  return gemm16<false, kRow, kStore>(d, gemm16_plan(d, false), st);
}

hipError_t launch_gated_backward(const GatedArgs& a, hipStream_t st) {
  const Space s = carve(a, true);
  const auto weights = [&](int which) {
    if (which == 0) return hipSuccess;
    const Gemm16Args g = weight_grads(a, s, which);
    return gemm16<true, kColumn, kStore>(g, gemm16_plan(g, false), st);
  };
  const int pair = (a.d_wg ? 1 : 0) | (a.d_wu ? 2 : 0), down = a.d_wd ? 4 : 0;
  if (a.dx != nullptr || pair != 0) {
    const Gemm16Args g = hidden_grad(a, s);
    if (hipError_t e = gemm16<false, kColumn, kSwigluGrad>(g, gemm16_plan(g, false), st); e != hipSuccess) return e;
  }
  if (a.dx != nullptr) {
    const Gemm16Args x = input_grad(a, s);
    if (hipError_t e = gemm16<false, kColumn, kStore>(x, gemm16_plan(x, false), st); e != hipSuccess) return e;
  }
  if (parts(a.rows) == 2) {
    for (int one : {1, 2, 4})
      if (hipError_t e = weights((pair | down) & one); e != hipSuccess) return e;
    return hipSuccess;
  }
  // The weights' gradients in one launch, or the down projection's apart, where
  // the numbers of tiles fill the chip's rounds better: 8,192 rows, 4096 x 2048
  // (256 and 128 large tiles): 420 us in one launch, 384 in two.
  if (pair != 0 && down != 0 &&
      gemm16_plan(weight_grads(a, s, pair | down), false).us >
          gemm16_plan(weight_grads(a, s, pair), false).us + gemm16_plan(weight_grads(a, s, down), false).us) {
    if (hipError_t e = weights(pair); e != hipSuccess) return e;
    return weights(down);
  }
  return weights(pair | down);
}

}  // namespace glm53
