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

// ------------------------------------------------------------- few rows ---
//
// Up to 16 rows: the call costs the weights' bytes.  A workgroup makes 16
// weight rows' results, its wavefronts taking parts of the contraction, joined
// in LDS in their order; weights go from memory to the MFMA through registers
// alone, a wavefront's loads all under way at once.  Rows of x are the MFMA's
// rows, so a lane's four results belong to one weight row.
constexpr int kFewRows = 16;
constexpr int kFewWaves = 16;
constexpr int kFewSteps = 4;  // K steps of 32 that a wavefront has in flight

// y[m, n] = sum_k x[m, k] w(n)[k] of the 16 rows that row(n) gives, per wavefront
// into part.  X: float rows are split into two bf16 operands, whose products
// are added: no rounding of x.
__device__ __forceinline__ float low_part(float f, uint16_t high) {
  const float h = bf16_to_f32(high);  // an infinity or NaN is in the high part alone
  return fabsf(h) < INFINITY ? f - h : 0.0f;
}

template <class X>
__device__ __forceinline__ void few_rows(const X* x, int rows, const uint16_t* w_row, int K, float (*part)[16][16]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int steps = (K + 31) / 32, each = (steps + kFewWaves - 1) / kFewWaves;
  const int first = wave * each, last = first + each < steps ? first + each : steps;
  const X* x_row = x + static_cast<int64_t>(r < rows ? r : rows - 1) * K;
  f32x4 acc = {0, 0, 0, 0};
  constexpr bool kFloat = sizeof(X) == 4;
  for (int s0 = first; s0 < last; s0 += kFewSteps) {
    u32x4 w[kFewSteps], v[kFewSteps][kFloat ? 2 : 1];
#pragma unroll
    for (int u = 0; u < kFewSteps; ++u) {  // past the wavefront's part or past K: read what is there, left out below
      const int k = 32 * (s0 + u < last ? s0 + u : last - 1) + 8 * q, kk = k < K ? k : 0;
      w[u] = *reinterpret_cast<const u32x4*>(w_row + kk);
#pragma unroll
      for (int h = 0; h < (kFloat ? 2 : 1); ++h) v[u][h] = *reinterpret_cast<const u32x4*>(x_row + kk + 4 * h);
    }
#pragma unroll
    for (int u = 0; u < kFewSteps; ++u) {
      const bool in = s0 + u < last && 32 * (s0 + u) + 8 * q < K;
      const u32x4 zero = {0, 0, 0, 0};
      const bf16x8 b = __builtin_bit_cast(bf16x8, in ? w[u] : zero);
      if constexpr (kFloat) {
        u32x4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f0 = __uint_as_float(v[u][i >> 1][2 * (i & 1)]), f1 = __uint_as_float(v[u][i >> 1][2 * (i & 1) + 1]);
          const uint16_t h0 = f32_to_bf16(f0), h1 = f32_to_bf16(f1);
          hi[i] = h0 | static_cast<uint32_t>(h1) << 16;
          lo[i] = f32_to_bf16(low_part(f0, h0)) | static_cast<uint32_t>(f32_to_bf16(low_part(f1, h1))) << 16;
        }
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, in ? hi : zero), b, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, in ? lo : zero), b, acc, 0, 0, 0);
      } else {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, in ? v[u][0] : zero), b, acc, 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[wave][4 * q + i][r] = acc[i];
  __syncthreads();
}

__device__ __forceinline__ float few_sum(const float (*part)[16][16], int m, int n) {
  float v = part[0][m][n];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) v += part[w][m][n];
  return v;
}

// 8 gate and the 8 up rows of the same outputs a workgroup; h stays FP32.
__global__ __launch_bounds__(64 * kFewWaves) void few_gate_up_kernel(GatedArgs a, float* h) {
  __shared__ float part[kFewWaves][16][16];
  const int r = threadIdx.x & 15;
  const int64_t n0 = 8 * static_cast<int64_t>(blockIdx.x);
  const uint16_t* w = (r < 8 ? a.wg : a.wu) + (n0 + (r & 7)) * a.hidden;
  few_rows(a.x, static_cast<int>(a.rows), w, static_cast<int>(a.hidden), part);
  if (threadIdx.x >= 128) return;
  const int n = threadIdx.x & 7, m = threadIdx.x >> 3;
  if (m >= a.rows) return;
  const float gate = few_sum(part, m, n), up = few_sum(part, m, 8 + n);
  const int64_t at = m * a.inter + n0 + n;
  if (a.gate != nullptr) {
    a.gate[at] = gate;
    a.up[at] = up;
  }
  const float c = clamp_gate(gate, a.limit);
  h[at] = c * sigmoid_f32(c) * clamp_up(up, a.limit);
}

__global__ __launch_bounds__(64 * kFewWaves) void few_down_kernel(GatedArgs a, const float* h) {
  __shared__ float part[kFewWaves][16][16];
  const int64_t n0 = 16 * static_cast<int64_t>(blockIdx.x);
  const int r = threadIdx.x & 15, cols = a.hidden - n0 < 16 ? 8 : 16;  // hidden is a multiple of 8
  few_rows(h, static_cast<int>(a.rows), a.wd + (n0 + (r < cols ? r : cols - 1)) * a.inter, static_cast<int>(a.inter), part);
  if (threadIdx.x >= 256) return;
  const int n = threadIdx.x & 15, m = threadIdx.x >> 4;
  if (m < a.rows && n < cols) a.y[m * a.hidden + n0 + n] = f32_to_bf16(few_sum(part, m, n));
}

hipError_t launch_few(const GatedArgs& a, hipStream_t st) {
  float* h = static_cast<float*>(a.space);
  few_gate_up_kernel<<<static_cast<uint32_t>(a.inter / 8), 64 * kFewWaves, 0, st>>>(a, h);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  few_down_kernel<<<static_cast<uint32_t>(cdiv(a.hidden, 16)), 64 * kFewWaves, 0, st>>>(a, h);
  return hipGetLastError();
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
  const size_t values = static_cast<size_t>(rows) * static_cast<size_t>(inter);
  if (backward) return 3 * round_up(2 * values);
  return round_up((rows <= kFewRows ? 4 : 2) * values);
}

hipError_t launch_gated(const GatedArgs& a, hipStream_t st) {
  if (a.rows <= kFewRows) return launch_few(a, st);
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
  const size_t plane = round_up(2 * static_cast<size_t>(a.rows) * static_cast<size_t>(a.inter));
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
