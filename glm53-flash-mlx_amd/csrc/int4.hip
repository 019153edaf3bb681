// Linear with 4-bit weights: y = x W^T + bias, W[n, k] = scale q + offset per
// row and group of 32, 64 or 128 columns.
#include <algorithm>

#include "gemm16.h"
#include "int4.h"

namespace glm53 {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ------------------------------------------------------------- few rows ---
//
// Few rows: the call costs the codes' bytes.  A workgroup makes 16
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
//
// 1 x 4096 x 4096, groups of 64: 5.9 us, 9 MB at 1.5 TB/s: a call this small is
// bound by the launch and the first loads' way (8 wavefronts a workgroup 6.5
// us, 4 8.9).  16 x 4096 x 7168: 12 us, x coming to every CU from L2.
//
// From 17 to 32 rows two MFMA rows share the codes (32 x 4096 x 4096 12.3 us here,
// 18.6 by the staged product below; 32 x 8192 x 2048 14.6, 17.7; 17 and 32 x 14336
// x 4096 33 and 43.5, 44).
bool few(int64_t rows) { return rows <= 32; }

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

template <class T>
__device__ __forceinline__ T load_at(const void* base, uint32_t off) {
  return *reinterpret_cast<const T*>(static_cast<const uint8_t*>(base) + off);
}
template <bool F32>
__device__ __forceinline__ float table_load(const void* base, uint32_t off) {
  if (F32) return load_at<float>(base, off);
  return bf16_to_f32(load_at<uint16_t>(base, off));
}

// x of a phase that is put in LDS: more where several workgroups of a CU are
// under way, one loading while another computes (8 x 4096 x 4096, one a CU, 64
// KB: 7.6 us, and 7.0 from L2; 12 x 8192 x 2048, two, 48 KB: 7.3 and 8.1; 8 x
// 8192 x 4096, 64 KB: 11.1 and 10.7).
constexpr int64_t kFewXBytes = 32768, kFewXBytesMany = 49152;
constexpr int kPhase = 8192;  // columns whose tables (and x) a workgroup has in LDS at a time

// Table entries (scale, offset - 128 scale) of an output column and phase in
// LDS: its groups, zeros in the last block's place past them.
__host__ __device__ constexpr int few_table_groups(int columns, int group_log2) { return (columns + 127) / 128 << (7 - group_log2); }

// Entries from one column to the next: odd, so that the 16 columns' entries of a
// group, which 16 lanes read at once, lie on different banks.
__host__ __device__ constexpr int few_table_ld(int columns, int group_log2) {
  return few_table_groups(columns, group_log2) | 1;
}

// XLDS: x lies in LDS, [columns / 8][rows] pieces of 8 in the codes' order (few
// rows, whose x fits); otherwise each wavefront reads its part from L2.
template <int W, int MT, int GROUP_LOG2, bool F32, bool OFFSETS, bool XLDS>
__global__ __launch_bounds__(64 * W) void int4_few_kernel(Int4Args a) {
  constexpr int kGroups = 128 >> GROUP_LOG2;     // groups of a block
  constexpr int kSteps = 1 << (GROUP_LOG2 - 5);  // MFMAs of a group
  constexpr int kTable = F32 ? 4 : 2;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4, K = static_cast<int>(a.K), rows = static_cast<int>(a.rows);
  const int64_t n0 = 16 * static_cast<int64_t>(blockIdx.x);
  const int cols = a.N - n0 < 16 ? static_cast<int>(a.N - n0) : 16;
  const int nr = r < cols ? r : cols - 1;
  const int groups = K >> GROUP_LOG2;
  // bases of the workgroup and a lane's byte offsets from them
  const uint8_t* codes = a.codes + n0 * (a.K >> 1);
  const uint8_t* scales = static_cast<const uint8_t*>(a.scales) + n0 * groups * kTable;
  const uint8_t* offsets = OFFSETS ? static_cast<const uint8_t*>(a.offsets) + n0 * groups * kTable : nullptr;
  const uint32_t code_off = static_cast<uint32_t>(nr) * (K >> 1);
  int mr[MT];
  uint32_t x_off[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    mr[i] = 16 * i + r < rows ? 16 * i + r : rows - 1;
    x_off[i] = static_cast<uint32_t>(mr[i]) * (2 * K) + 16 * q;
  }
  const int phase_columns = K < kPhase ? K : kPhase;
  f32x2* tables = reinterpret_cast<f32x2*>(lds);
  const int table_ld = few_table_ld(phase_columns, GROUP_LOG2);
  uint8_t* x_lds = lds + 128 * table_ld;

  f32x4 total[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) total[i] = (f32x4){0, 0, 0, 0};
  const u32x4 one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  const bf16x8 ones = __builtin_bit_cast(bf16x8, one);
  for (int k0 = 0; k0 < K; k0 += kPhase) {
    const int columns = K - k0 < kPhase ? K - k0 : kPhase;
    const int blocks = (columns + 127) / 128, each = (blocks + W - 1) / W;
    const int first = wave * each, last = first + each < blocks ? first + each : blocks;
    // Codes and x of a block, without a branch: what lies past K reads an
    // address that is there and meets scale 0.  Branches around the steps would
    // have the compiler move each step's loads behind them.
    u32x4 code[2], xs[2][XLDS ? 1 : MT][4];
    const auto load = [&](int b, int to) {
      const int k = k0 + 128 * b;
      const uint32_t piece = k + 128 <= K || k + 32 * q < K ? 16 * q : 0;
      code[to] = load_at<u32x4>(codes, code_off + (k >> 1) + piece);
      if constexpr (!XLDS) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int s = 0; s < 4; ++s) xs[to][i][s] = load_at<u32x4>(a.x, x_off[i] + 2 * (k + 32 * s < K ? k + 32 * s : k));
      }
    };
    if (first < last) load(first, 0);
    if (k0 > 0) __syncthreads();  // the phase before is read
    const int entries = few_table_groups(columns, GROUP_LOG2), phase_groups = columns >> GROUP_LOG2;
    for (int c = wave; c < 16; c += W)  // a column's groups are consecutive in memory and in LDS
      for (int g = lane; g < entries; g += 64) {
        f32x2 v = {0.0f, 0.0f};
        if (g < phase_groups && c < cols) {
          const uint32_t at = (static_cast<uint32_t>(c) * groups + (k0 >> GROUP_LOG2) + g) * kTable;
          const float scale = table_load<F32>(scales, at);
          v = (f32x2){scale, OFFSETS ? table_load<F32>(offsets, at) - 128.0f * scale : -136.0f * scale};
        }
        tables[c * table_ld + g] = v;
      }
    if constexpr (XLDS) {
      for (int m = 0; m < rows; ++m)
        for (int c = threadIdx.x; c < columns / 8; c += 64 * W)
          *reinterpret_cast<bf16x8*>(x_lds + 16 * (c * rows + m)) = codes_order(load_at<u32x4>(a.x, 2 * (m * K + k0) + 16 * c));
    }
    __syncthreads();
    const auto compute = [&](int b, int from) {
      u32x4 cd = code[from];
      exchange_quarters(cd);
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const f32x2 t = tables[r * table_ld + b * kGroups + g];
        f32x4 d[MT], sum[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) d[i] = sum[i] = (f32x4){0, 0, 0, 0};
#pragma unroll
        for (int s = g * kSteps; s < (g + 1) * kSteps; ++s) {
          const bf16x8 w = codes_operand(cd[s]);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            bf16x8 v;
            if constexpr (XLDS) {
              const int at = 128 * b + 32 * s < columns ? 16 * b + 4 * s : 0;
              v = *reinterpret_cast<const bf16x8*>(x_lds + 16 * ((at + q) * rows + mr[i]));
            } else {
              v = codes_order(xs[from][i][s]);
            }
            d[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, w, d[i], 0, 0, 0);
            sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ones, sum[i], 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) total[i][e] += t[0] * d[i][e] + t[1] * sum[i][e];
      }
    };
    for (int b = first; b < last; b += 2) {
      if (b + 1 < last) load(b + 1, 1);
      compute(b, 0);
      if (b + 2 < last) load(b + 2, 0);
      if (b + 1 < last) compute(b + 1, 1);
    }
  }
  __syncthreads();  // the last phase is read; its place holds the partial sums
  float(*part)[16 * MT][16] = reinterpret_cast<float(*)[16 * MT][16]>(lds);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][16 * i + 4 * q + e][r] = total[i][e];
  __syncthreads();
  for (int at = threadIdx.x; at < 256 * MT; at += 64 * W) {
    const int col = at & 15, m = at >> 4;
    if (m >= rows || col >= cols) continue;
    float y = part[0][m][col];
#pragma unroll
    for (int w = 1; w < W; ++w) y += part[w][m][col];
    if (!(fabsf(y) < INFINITY))
      y = one_output(a.x + m * a.K, codes + static_cast<int64_t>(col) * (K >> 1), scales + int64_t{col} * groups * kTable,
                     OFFSETS ? offsets + int64_t{col} * groups * kTable : nullptr, F32, GROUP_LOG2, K);
    if (a.bias != nullptr) y += table_value(a.bias, a.tables_f32, n0 + col);
    a.y[m * a.N + n0 + col] = f32_to_bf16(y);
  }
}

template <int W, int MT, int GROUP_LOG2, bool XLDS>
hipError_t launch_few(const Int4Args& a, hipStream_t st) {
  const dim3 grid(static_cast<uint32_t>(cdiv(a.N, 16))), block(64 * W);
  const int columns = static_cast<int>(a.K < kPhase ? a.K : kPhase);
  const size_t staged = 128 * few_table_ld(columns, GROUP_LOG2) + (XLDS ? 2 * static_cast<size_t>(a.rows * columns) : 0);
  const size_t lds = staged > 1024 * W * MT ? staged : 1024 * W * MT;
  if (a.tables_f32) {
    if (a.offsets != nullptr)
      int4_few_kernel<W, MT, GROUP_LOG2, true, true, XLDS><<<grid, block, lds, st>>>(a);
    else
      int4_few_kernel<W, MT, GROUP_LOG2, true, false, XLDS><<<grid, block, lds, st>>>(a);
  } else {
    if (a.offsets != nullptr)
      int4_few_kernel<W, MT, GROUP_LOG2, false, true, XLDS><<<grid, block, lds, st>>>(a);
    else
      int4_few_kernel<W, MT, GROUP_LOG2, false, false, XLDS><<<grid, block, lds, st>>>(a);
  }
  return hipGetLastError();
}

template <int W, int MT, bool XLDS>
hipError_t launch_few_group(const Int4Args& a, hipStream_t st) {
  if (a.group_log2 == 5) return launch_few<W, MT, 5, XLDS>(a, st);
  if (a.group_log2 == 6) return launch_few<W, MT, 6, XLDS>(a, st);
  return launch_few<W, MT, 7, XLDS>(a, st);
}

// Wavefronts a workgroup: 16 while the chip's 256 CUs have a workgroup or two
// each, which 16 wavefronts keep in loads; with more workgroups fewer, whose
// parts of the contraction are longer (x in LDS: 448 workgroups 8.3 us by 16,
// 8.6 by 8; 896: 14.6, 13.2, by 4 14.0; 2,048: 18.6, 16.7, 14.1.  x from L2:
// 256: 8.1, 8.7; 448: 11.2, 9.4, 10.8; 896: 27.0, 23.0, 23.3; 2,048: 39, 29, 26).
hipError_t launch_few_rows(const Int4Args& a, hipStream_t st) {
  const int64_t blocks = cdiv(a.N, 16);
  if (a.rows > 16) return launch_few_group<8, 2, false>(a, st);
  if (2 * a.rows * (a.K < kPhase ? a.K : kPhase) <= (blocks <= 256 ? kFewXBytes : kFewXBytesMany)) {
    if (blocks <= 512) return launch_few_group<16, 1, true>(a, st);
    if (blocks <= 1024) return launch_few_group<8, 1, true>(a, st);
    return launch_few_group<4, 1, true>(a, st);
  }
  if (blocks <= 256) return launch_few_group<16, 1, false>(a, st);
  if (blocks <= 1024) return launch_few_group<8, 1, false>(a, st);
  return launch_few_group<4, 1, false>(a, st);
}

}  // namespace

namespace {

// ------------------------------------------------------------ many rows ---
//
// Tiled products of x by the codes' values 128 + q, whose group sums are scaled
// in FP32 as above.

// The values as bf16 [N, K], and scale and base of every group in the order
// that the product's tiles load them, [K / group][tiles of 128 columns][scale,
// base][128].  Tables: the first workgroups, 128 columns and kTurn groups each,
// turned in LDS.  Values: a thread takes kExpand pieces of 8 codes (4 bytes), 256
// apart, so that a wavefront reads 256 bytes and writes 1 KB in a row; bound by
// the writes, 2 bytes a weight.  4096 x 4096: 9.4 us.
constexpr int kExpand = 4, kTurn = 16;

int64_t value_blocks(const Int4Args& a) { return cdiv(a.N * (a.K >> 3), 256 * kExpand); }
int64_t table_blocks(const Int4Args& a) { return cdiv(a.N, 128) * cdiv(a.K >> a.group_log2, kTurn); }

template <bool F32>
__global__ __launch_bounds__(256) void int4_expand_kernel(Int4Args a, int64_t table_blocks, uint16_t* w, float* tables) {
  __shared__ float turn[2][kTurn][128 + 1];
  if (blockIdx.x >= table_blocks) {
    const int64_t first = (blockIdx.x - table_blocks) * int64_t{256 * kExpand}, all = a.N * (a.K >> 3);
    uint32_t codes[kExpand];
#pragma unroll
    for (int u = 0; u < kExpand; ++u) {
      const int64_t at = first + u * 256 + threadIdx.x;
      codes[u] = reinterpret_cast<const uint32_t*>(a.codes)[at < all ? at : all - 1];
    }
#pragma unroll
    for (int u = 0; u < kExpand; ++u) {
      const int64_t at = first + u * 256 + threadIdx.x;
      if (at < all) *reinterpret_cast<u32x4*>(w + 8 * at) = code_values(codes[u]);
    }
    return;
  }
  const int64_t groups = a.K >> a.group_log2, bands = (groups + kTurn - 1) / kTurn, tiles = (a.N + 127) / 128;
  const int64_t tile = blockIdx.x / bands, g0 = (blockIdx.x - tile * bands) * kTurn;
  constexpr int kEach = 128 * kTurn / 256;  // entries of a thread, all on their way before the first is used
  const int g = threadIdx.x % kTurn, n0 = threadIdx.x / kTurn;
  float scale[kEach], offset[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int64_t n = 128 * tile + n0 + 256 / kTurn * i;
    const int64_t t = n < a.N && g0 + g < groups ? n * groups + g0 + g : 0;  // past the edges: never used
    scale[i] = table_value(a.scales, F32, t);
    offset[i] = table_value(a.offsets != nullptr ? a.offsets : a.scales, F32, t);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    turn[0][g][n0 + 256 / kTurn * i] = scale[i];
    turn[1][g][n0 + 256 / kTurn * i] = code_base(scale[i], a.offsets != nullptr, offset[i]);
  }
  __syncthreads();
  for (int i = 0; i < kTurn && g0 + i < groups; ++i)
    tables[((g0 + i) * tiles + tile) * 256 + threadIdx.x] = turn[threadIdx.x >> 7][i][threadIdx.x & 127];
}

// Up to this many rows the codes become values in the tiled product's own
// stage, tile row by tile row; beyond, in memory once, for products whose
// larger tiles the conversion would hold up (64 rows, 4096 x 4096: 21 us staged;
// 128: 29; 200: 45, 35 from memory; 300: 75, 39; 1536 x 4096 in groups of 32, 200
// and 300 rows: 27 and 30, 31 and 32).
constexpr int64_t kStagedRows = 128;

Gemm16Args product(const Int4Args& a) {
  Gemm16Args g{};
  g.k = a.K;
  g.problems = g.segments = 1;
  g.pair[0] = {a.x, nullptr, a.y, a.K, a.K, a.N, a.rows, a.N};
  g.codes = a.codes;
  g.scales = a.scales;
  g.offsets = a.offsets;
  g.bias = a.bias;
  g.scales_f32 = a.tables_f32;
  g.group_log2 = a.group_log2;
  return g;
}

// 64 x 128 tiles; as many parts of the contraction as fill the chip once.
Gemm16Plan staged_plan(const Int4Args& a) {
  const int64_t tiles = cdiv(a.rows, 64) * cdiv(a.N, 128), steps = cdiv(a.K, 128);
  const int splits = used_splits(steps, std::max<int64_t>(1, std::min<int64_t>({16, 256 / tiles, steps / 2})));
  return {kTile64, splits, splits > 1 ? splits * a.rows * partial_ld(a.N) : 0, 0.0f};
}

template <int GROUP>
hipError_t launch_staged(const Gemm16Args& g, hipStream_t st) {
  if (g.scales_f32) return gemm16_launch<Gemm16<1, 4, 4, 2, 2, false, kCodesF32, kBias, GROUP>, kBias>(g, st);
  return gemm16_launch<Gemm16<1, 4, 4, 2, 2, false, kCodes, kBias, GROUP>, kBias>(g, st);
}

template <int GROUP>
hipError_t launch_values(Gemm16Args g, const Gemm16Plan& plan, hipStream_t st) {
  g.splits = plan.splits;
  if (plan.tile == kTile64) return gemm16_launch<Gemm16<2, 2, 2, 4, 1, false, kCodeValues, kBias, GROUP>, kBias>(g, st);
  return gemm16_launch<Gemm16<2, 2, 4, 4, 1, false, kCodeValues, kBias, GROUP>, kBias>(g, st);
}

size_t value_bytes(int64_t N, int64_t K) { return (2 * static_cast<size_t>(N) * static_cast<size_t>(K) + 255) & ~size_t{255}; }
size_t table_bytes(int64_t N, int64_t K, int group_log2) {
  return 1024 * static_cast<size_t>(cdiv(N, 128)) * static_cast<size_t>(K >> group_log2);
}

}  // namespace

size_t int4_space(int64_t rows, int64_t N, int64_t K) {
  if (few(rows)) return 0;
  Int4Args a{};
  a.rows = rows;
  a.N = N;
  a.K = K;
  if (rows <= kStagedRows) return sizeof(float) * static_cast<size_t>(staged_plan(a).partial);
  return value_bytes(N, K) + table_bytes(N, K, 5) + sizeof(float) * static_cast<size_t>(gemm16_plan_scaled(product(a)).partial);
}

hipError_t launch_int4(const Int4Args& a, hipStream_t st) {
  if (few(a.rows)) return launch_few_rows(a, st);
  Gemm16Args g = product(a);
  if (a.rows <= kStagedRows) {
    const Gemm16Plan plan = staged_plan(a);
    g.splits = plan.splits;
    g.partial = static_cast<float*>(a.space);
    g.room = static_cast<int64_t>(a.space_bytes / sizeof(float));
    return a.group_log2 == 5 ? launch_staged<32>(g, st) : launch_staged<64>(g, st);
  }
  uint16_t* w = static_cast<uint16_t*>(a.space);
  float* tables = reinterpret_cast<float*>(static_cast<uint8_t*>(a.space) + value_bytes(a.N, a.K));
  const size_t before = value_bytes(a.N, a.K) + table_bytes(a.N, a.K, a.group_log2);
  g.pair[0].b = w;
  g.tables = tables;
  g.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(a.space) + before);
  g.room = static_cast<int64_t>((a.space_bytes - before) / sizeof(float));
  const int64_t turns = table_blocks(a), blocks = turns + value_blocks(a);
  if (blocks * 256 >= (int64_t{1} << 32)) return hipErrorInvalidValue;  // a grid has fewer than 2^32 threads
  if (a.tables_f32)
    int4_expand_kernel<true><<<static_cast<uint32_t>(blocks), 256, 0, st>>>(a, turns, w, tables);
  else
    int4_expand_kernel<false><<<static_cast<uint32_t>(blocks), 256, 0, st>>>(a, turns, w, tables);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const Gemm16Plan plan = gemm16_plan_scaled(g);
  return a.group_log2 == 5 ? launch_values<32>(g, plan, st) : launch_values<64>(g, plan, st);
}

}  // namespace glm53
