// Linear with 4-bit weights: y = x W^T + bias, W[n, k] = scale q + offset per
// row and group of 32, 64 or 128 columns.
#include "gemm16.h"
#include "int4.h"

namespace glm53 {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <class G>
hipError_t launch_tiles(Gemm16Args g, hipStream_t st) {
  g.tiles = cdiv(g.pair[0].m, G::BM) * cdiv(g.pair[0].n, G::kColumns);
  g.group_m = 8;
  gemm16_kernel<G><<<static_cast<uint32_t>(g.tiles * g.splits), G::kThreads, G::kLds, st>>>(g);
  return hipGetLastError();
}

// ------------------------------------------------------------- few rows ---
//
// Up to 16 rows: the call costs the codes' bytes.  A workgroup makes 16
// output columns, its wavefronts taking parts of the contraction, joined in
// LDS in their order; no code passes through LDS.  A lane loads 32 codes of
// one row (16 bytes; a wavefront 64 bytes of each of 16 rows), the four
// quarters of the wavefront exchange dwords so that each MFMA contracts 32
// consecutive columns, which lie in one group.  Codes become bf16 by or-ing
// them into the mantissa of 128 (128 + q is exact), and a group's FP32 result
//   sum x w = scale (sum x (128 + q)) + (offset - 128 scale) sum x
// is scaled once, sum x coming from an MFMA with ones: no weight is rounded.
// Operands: rows of x as the MFMA's rows, so that a lane's four results have
// one output column, one scale and one offset.
constexpr int kFewRows = 16;
constexpr int kFewWaves = 8;
constexpr int kFewBlocks = 4;  // blocks of 128 columns that a wavefront has in flight

// Quarter q's dword s of four becomes quarter s's dword q.
__device__ __forceinline__ void exchange_quarters(u32x4& v) {
  auto swap32 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  };
  auto swap16 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  };
  uint32_t a = v[0], b = v[1], c = v[2], d = v[3];
  swap32(a, c);
  swap32(b, d);
  swap16(a, b);
  swap16(c, d);
  v = (u32x4){a, b, c, d};
}

// 8 codes as bf16 128 + q, in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ bf16x8 codes_operand(uint32_t v) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = ((v >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  return __builtin_bit_cast(bf16x8, r);
}
// 8 values of x in that order.
__device__ __forceinline__ bf16x8 codes_order(u32x4 x) {
  const u32x4 r = {__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                   __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
  return __builtin_bit_cast(bf16x8, r);
}

// One output in the formula's own order: for results that the kernel below
// cannot tell from inf - inf of its two sums.
__device__ __attribute__((noinline)) float one_output(const Int4Args& a, int64_t m, int64_t n) {
  float y = 0.0f;
  for (int64_t k = 0; k < a.K; ++k) {
    const int64_t t = n * (a.K >> a.group_log2) + (k >> a.group_log2);
    const float scale = table_value(a.scales, a.tables_f32, t);
    const float offset = a.offsets != nullptr ? table_value(a.offsets, a.tables_f32, t) : -8.0f * scale;
    const int q = (a.codes[(n * a.K + k) >> 1] >> (4 * (k & 1))) & 15;
    y += bf16_to_f32(a.x[m * a.K + k]) * fmaf(static_cast<float>(q), scale, offset);
  }
  return y;
}

template <int GROUP_LOG2>
__global__ __launch_bounds__(64 * kFewWaves) void int4_few_kernel(Int4Args a) {
  constexpr int kGroups = 128 >> GROUP_LOG2;           // groups of a block
  constexpr int kSteps = 1 << (GROUP_LOG2 - 5);        // MFMAs of a group
  __shared__ float part[kFewWaves][kFewRows][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int64_t n0 = 16 * static_cast<int64_t>(blockIdx.x);
  const int64_t n = n0 + r < a.N ? n0 + r : a.N - 1;
  const int64_t m = r < a.rows ? r : a.rows - 1;
  const uint8_t* row = a.codes + n * (a.K >> 1) + 16 * q;
  const uint16_t* x = a.x + m * a.K + 8 * q;
  const int64_t table = n * (a.K >> GROUP_LOG2);
  const int64_t blocks = (a.K + 127) / 128;
  const int64_t each = (blocks + kFewWaves - 1) / kFewWaves;
  const int64_t first = wave * each, last = first + each < blocks ? first + each : blocks;
  f32x4 total = {0, 0, 0, 0};
  const u32x4 one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  const bf16x8 ones = __builtin_bit_cast(bf16x8, one);
  for (int64_t b0 = first; b0 < last; b0 += kFewBlocks) {
    u32x4 code[kFewBlocks], xs[kFewBlocks][4];
    float scale[kFewBlocks][kGroups], offset[kFewBlocks][kGroups];
#pragma unroll
    for (int u = 0; u < kFewBlocks; ++u) {
      const int64_t k = 128 * (b0 + u);
      if (b0 + u >= last) break;
      code[u] = (u32x4){0, 0, 0, 0};
      if (k + 32 * q < a.K) code[u] = *reinterpret_cast<const u32x4*>(row + (k >> 1));
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (k + 32 * s < a.K) xs[u][s] = *reinterpret_cast<const u32x4*>(x + k + 32 * s);
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (k + (g << GROUP_LOG2) >= a.K) break;
        const int64_t t = table + (k >> GROUP_LOG2) + g;
        scale[u][g] = table_value(a.scales, a.tables_f32, t);
        offset[u][g] = a.offsets != nullptr ? table_value(a.offsets, a.tables_f32, t) : -8.0f * scale[u][g];
      }
    }
#pragma unroll
    for (int u = 0; u < kFewBlocks; ++u) {
      const int64_t k = 128 * (b0 + u);
      if (b0 + u >= last) break;
      exchange_quarters(code[u]);
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (k + (g << GROUP_LOG2) >= a.K) break;
        f32x4 d = {0, 0, 0, 0}, sum = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const bf16x8 v = codes_order(xs[u][g * kSteps + s]);
          d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, codes_operand(code[u][g * kSteps + s]), d, 0, 0, 0);
          sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ones, sum, 0, 0, 0);
        }
        const float c = offset[u][g] - 128.0f * scale[u][g];
#pragma unroll
        for (int i = 0; i < 4; ++i) total[i] += scale[u][g] * d[i] + c * sum[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[wave][4 * q + i][r] = total[i];
  __syncthreads();
  if (threadIdx.x >= 16 * kFewRows) return;
  const int col = threadIdx.x & 15, mm = threadIdx.x >> 4;
  if (mm >= a.rows || n0 + col >= a.N) return;
  float y = part[0][mm][col];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) y += part[w][mm][col];
  if (!(fabsf(y) < INFINITY)) y = one_output(a, mm, n0 + col);
  if (a.bias != nullptr) y += table_value(a.bias, a.tables_f32, n0 + col);
  a.y[mm * a.N + n0 + col] = f32_to_bf16(y);
}

hipError_t launch_few(const Int4Args& a, hipStream_t st) {
  const dim3 grid(static_cast<uint32_t>(cdiv(a.N, 16)));
  if (a.group_log2 == 5)
    int4_few_kernel<5><<<grid, 64 * kFewWaves, 0, st>>>(a);
  else if (a.group_log2 == 6)
    int4_few_kernel<6><<<grid, 64 * kFewWaves, 0, st>>>(a);
  else
    int4_few_kernel<7><<<grid, 64 * kFewWaves, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

size_t int4_space(int64_t rows, int64_t N, int64_t K) { return 0; }

hipError_t launch_int4(const Int4Args& a, hipStream_t st) {
  if (a.rows <= kFewRows) return launch_few(a, st);
  Gemm16Args g{};
  g.k = a.K;
  g.problems = g.segments = g.splits = 1;
  g.pair[0] = {a.x, nullptr, a.y, a.K, a.K, a.N, a.rows, a.N};
  g.codes = a.codes;
  g.scales = a.scales;
  g.offsets = a.offsets;
  g.bias = a.bias;
  g.scales_f32 = a.tables_f32;
  g.group_log2 = a.group_log2;
  return launch_tiles<Gemm16<2, 2, 4, 4, false, kCodes, kBias>>(g, st);
}

}  // namespace glm53
