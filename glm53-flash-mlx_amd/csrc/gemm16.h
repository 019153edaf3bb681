// Tiled matrix products of 16-bit operands on the bf16 MFMA, the core of the
// gated MLP and of the 4-bit linear over many rows:
//
//   out[m, n] = sum_k a(m, k) b(n, k),  FP32 accumulation
//
// A workgroup computes a BM x BN tile, its wavefronts a grid of them.  Each K
// step of 64 stages both operands in LDS while the step before is
// multiplied (two or three stages, one barrier a step).  An operand is stored either
// with k contiguous (rows of 64 k: "row" form) or with m or n contiguous
// ("column" form, the contraction over rows: gradients), which is read from
// LDS by the transposing ds_read_b64_tr_b16, so no operand is ever
// transposed in memory.
//
// Bound by the matrix pipes where the tiles fill the chip: a step of a 256 x 256
// tile takes 1.45 to 1.6 us on every CU, 1.35 to 1.48 PFLOP/s (the library's
// product of 8192^3: 1.35), and ~12 us a tile go to its first loads and its
// epilogue.  8,192 rows, 4096 x 2048: gate and up with SwiGLU 250 us, 1.10
// PFLOP/s, down 126, SwiGLU's gradient 161, x's gradient over both segments
// 234, 1.17 PFLOP/s, dWg and dWu together 231, 1.19.
#pragma once

#include <initializer_list>

#include "common.h"

namespace glm53 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kStepK = 64;          // contraction columns of one LDS stage
constexpr int kOperandTile = 2048;  // 16 rows x 64 k, or its share of a column stage

// One product's operands, or one segment of a contraction over several.
struct Gemm16Pair {
  const uint16_t* a;  // row form [m, lda], column form [k, lda]
  const uint16_t* b;
  uint16_t* out;      // [m, ldo]
  int64_t lda, ldb, ldo, m, n;
};

struct Gemm16Args {
  Gemm16Pair pair[4];
  int64_t k;       // of each pair
  int problems;    // pairs that are products of their own
  int segments;    // pairs whose contractions are added into pair[0].out
  int splits;      // parts of the contraction, each to `partial` and none without a K step (used_splits)
  float* partial;  // of each problem [splits][planes][m][partial_ld(n)], at partial_at floats
  int64_t room;    // floats at partial
  int64_t partial_at[4];
  int64_t tiles;   // output tiles of all problems; tiles * splits below 2^31
  int group_m;     // tile rows that one XCD's neighbouring workgroups share
  // SwiGLU: pair[0].b gate and pair[1].b up rows, out = h; gate/up (f32
  // [m, n]) null or what the gradient needs.  Its gradient (out unused): reads
  // gate and up, writes d_gate and d_up.
  float limit;
  float* gate;
  float* up;
  uint16_t* d_gate;
  uint16_t* d_up;
  int64_t low;  // 0, or values from d_gate and d_up to the low parts that are written there too
  // 4-bit b: codes [n, k / 2], scales and offsets [n, k / group], bias [n]
  const uint8_t* codes;
  const void* scales;
  const void* offsets;  // null: -8 scale
  const void* bias;     // or null
  bool scales_f32;
  int group_log2;
  const float* tables;  // with kCodeValues: [k / group][tiles of 128 columns][scale, base][128]
};

enum Gemm16Epilogue { kStore, kSwiglu, kSwigluGrad, kBias };
// b as 4-bit codes with bf16 or FP32 tables, or (kCodeValues) as the bf16 values
// 128 + q of the codes, [n, k], with `tables`: the products of kBias.
enum OperandForm { kRow, kColumn, kCodes, kCodesF32, kCodeValues };

// Row length of the partial results: whole groups of four.
__host__ __device__ __forceinline__ int64_t partial_ld(int64_t n) { return (n + 3) & ~int64_t{3}; }

__device__ __forceinline__ float sigmoid_f32(float g) { return __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

// g' = min(g, L), u' = clip(u, -L, L); a NaN stays one.
__device__ __forceinline__ float clamp_gate(float g, float limit) { return g > limit ? limit : g; }
__device__ __forceinline__ float clamp_up(float u, float limit) { return u > limit ? limit : u < -limit ? -limit : u; }

__device__ __forceinline__ u32x2 pack_bf16x4(f32x4 v) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4));
}

// What `high` (bf16) leaves of f; an infinity or NaN is in the high part alone.
__device__ __forceinline__ float low_part(float f, uint16_t high) {
  const float h = bf16_to_f32(high);
  return fabsf(h) < INFINITY ? f - h : 0.0f;
}
__device__ __forceinline__ u32x2 low_bf16x4(f32x4 v, u32x2 high) {
  return pack_bf16x4((f32x4){low_part(v[0], high[0] & 0xFFFF), low_part(v[1], high[0] >> 16),
                             low_part(v[2], high[1] & 0xFFFF), low_part(v[3], high[1] >> 16)});
}

__device__ __forceinline__ float table_value(const void* t, bool f32, int64_t i) {
  return f32 ? static_cast<const float*>(t)[i] : bf16_to_f32(static_cast<const uint16_t*>(t)[i]);
}

// Outputs n .. n + 3 of row m (m and n in range; n % 4 == 0).
__device__ __forceinline__ void store_plain(const Gemm16Args& g, const Gemm16Pair& p, int64_t m, int64_t n, f32x4 v) {
  *reinterpret_cast<u32x2*>(p.out + m * p.ldo + n) = pack_bf16x4(v);
}

// One output of a 4-bit product in the formula's own order: for results that
// the sums of x times codes cannot tell from inf - inf.  Its pointers come one
// by one: with an argument block's address taken, every load of a kernel would
// go by flat addresses and wait for the one before.  2,048 x 4096 x 4096 with an
// infinity in every row's last column: 15 ms.
__device__ __forceinline__ float one_output(const uint16_t* x, const uint8_t* codes, const void* scales,
                                            const void* offsets, bool f32, int group_log2, int64_t k_all) {
  float y = 0.0f;
  for (int64_t k = 0; k < k_all && y == y; k += 8) {  // a NaN stays one
    const float scale = table_value(scales, f32, k >> group_log2);
    const float offset = offsets != nullptr ? table_value(offsets, f32, k >> group_log2) : -8.0f * scale;
    const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + (k >> 1));
    const u32x4 v = *reinterpret_cast<const u32x4*>(x + k);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y += bf16_to_f32(static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1)))) *
           fmaf(static_cast<float>((q >> (4 * i)) & 15), scale, offset);
  }
  return y;
}

__device__ __forceinline__ bool finite(f32x4 v) {
  return fabsf(v[0]) < INFINITY && fabsf(v[1]) < INFINITY && fabsf(v[2]) < INFINITY && fabsf(v[3]) < INFINITY;
}

// Outputs of a 4-bit product plus its bias, for any number of columns: outputs
// past the last one are left out, and rows whose length is no multiple of 4
// have no aligned group of four.
__device__ __forceinline__ void store_bias(const Gemm16Args& g, const Gemm16Pair& p, int64_t m, int64_t n, f32x4 v) {
  uint16_t* out = p.out + m * p.ldo + n;
  if (g.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.n) v[i] += table_value(g.bias, g.scales_f32, n + i);
  }
  if ((p.ldo & 3) == 0) {
    *reinterpret_cast<u32x2*>(out) = pack_bf16x4(v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < p.n) out[i] = f32_to_bf16(v[i]);
}

// Those of the four outputs stored that are not finite, once more by the formula.
__device__ __forceinline__ void store_bias_again(const Gemm16Args& g, const Gemm16Pair& p, int64_t m, int64_t n) {
  asm volatile("" ::: "memory");  // read as stored, whatever type they were stored as
#pragma unroll 1
  for (const int64_t last = n + 4 < p.n ? n + 4 : p.n; n < last; ++n) {
    uint16_t* out = p.out + m * p.ldo + n;
    if ((*out & 0x7F80) != 0x7F80) continue;
    const int64_t table = n * (g.k >> g.group_log2) * (g.scales_f32 ? 4 : 2);
    float y = one_output(p.a + m * p.lda, g.codes + n * (g.k >> 1), static_cast<const uint8_t*>(g.scales) + table,
                         g.offsets != nullptr ? static_cast<const uint8_t*>(g.offsets) + table : nullptr, g.scales_f32,
                         g.group_log2, g.k);
    if (g.bias != nullptr) y += table_value(g.bias, g.scales_f32, n);
    *out = f32_to_bf16(y);
  }
}

// h = silu(min(g, L)) clip(u, -L, L).  G and U themselves are kept in FP32
// where a gradient follows: rounded to bf16 they would put an error the size
// of the results' own rounding into every gradient.
__device__ __forceinline__ void store_swiglu(const Gemm16Args& g, const Gemm16Pair& p, int64_t m, int64_t n, f32x4 gate,
                                             f32x4 up) {
  const int64_t at = m * p.n + n;
  if (g.gate != nullptr) {
    *reinterpret_cast<f32x4*>(g.gate + at) = gate;
    *reinterpret_cast<f32x4*>(g.up + at) = up;
  }
  f32x4 h;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = clamp_gate(gate[i], g.limit);
    h[i] = c * sigmoid_f32(c) * clamp_up(up[i], g.limit);
  }
  *reinterpret_cast<u32x2*>(p.out + m * p.ldo + n) = pack_bf16x4(h);
}

// With dh: dU = dh silu(g') [|u| <= L], dG = dh u' silu'(g') [g <= L].
__device__ __forceinline__ void store_swiglu_grad(const Gemm16Args& g, const Gemm16Pair& p, int64_t m, int64_t n,
                                                  f32x4 dh, f32x4 gate, f32x4 up) {
  const int64_t at = m * p.n + n;
  f32x4 dg, du;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = clamp_gate(gate[i], g.limit), u = clamp_up(up[i], g.limit);
    const float s = sigmoid_f32(c);
    du[i] = fabsf(up[i]) > g.limit ? 0.0f : dh[i] * (c * s);
    dg[i] = gate[i] > g.limit ? 0.0f : dh[i] * u * (s * (1.0f + c * (1.0f - s)));
  }
  const u32x2 high_g = pack_bf16x4(dg), high_u = pack_bf16x4(du);
  *reinterpret_cast<u32x2*>(g.d_gate + at) = high_g;
  *reinterpret_cast<u32x2*>(g.d_up + at) = high_u;
  if (g.low != 0) {
    *reinterpret_cast<u32x2*>(g.d_gate + g.low + at) = low_bf16x4(dg, high_g);
    *reinterpret_cast<u32x2*>(g.d_up + g.low + at) = low_bf16x4(du, high_u);
  }
}

// ------------------------------------------------------------- staging ---
//
// Row form: operand tiles of 16 rows x 128 bytes, row r's 16-byte piece p in
// slot p ^ (r % 8) ^ (r / 8 % 2) of its row, the permutation the FP8 kernels
// measured at the LDS's full 16-byte read rate.  A lane reads pieces 2 (l /
// 16) and 2 (l / 16) + 1 of row l % 16, so MFMA j of a step contracts k =
// 16 (l / 16) + 8 j + 0..7.
//
// Column form: 64 rows of R columns.  ds_read_b64_tr_b16 gives lane i of each
// 16 the 4 rows x 1 column that the 16 lanes' 8 bytes hold, lane a reading
// row a / 4, columns 4 (a % 4) .. + 3.  Its 64 lanes read 32-byte pieces of 16
// rows at one column; piece c of row k lies at c ^ f(k), f(k) = k % 4 + 4 (k /
// 16 % 2), which puts the 8 rows that 32 lanes read on distinct banks.

__device__ __forceinline__ int column_swizzle(int k) { return (k & 3) | ((k >> 2) & 4); }

// A wave-uniform pointer in scalar registers, where the compiler does not see
// that it is one.
__device__ __forceinline__ const void* uniform_pointer(const void* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));  // an int: not to be sign-extended
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<const void*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// Direct global -> LDS load of 16 bytes a lane to lds_base + 16 lane.  Inline
// assembly, so that the compiler puts no wait of its own before LDS reads;
// stage_wait counts them.
__device__ __forceinline__ void load_lds16(const void* base, uint32_t off, uint32_t lds_base) {
  base = uniform_pointer(base);
  lds_base = __builtin_amdgcn_readfirstlane(lds_base);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_base)
               : "memory", "m0");
}

// All of this wavefront's LDS accesses and all but its last LEFT loads are done
// (loads return in their order), and every wavefront of the workgroup is here.
template <int LEFT>
__device__ __forceinline__ void stage_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// The share of one wavefront in staging an operand tile of R rows (row form)
// or columns (column form): loads `wave`, wave + W, ... of R / 8, 1 KB each.
template <int R, int W, bool COLUMN>
struct Stager {
  static constexpr int kLoads = R / 8 / W;
  static_assert(R % (8 * W) == 0, "whole loads a wavefront");
  static constexpr int kLanes = R / 8;  // column form: lanes a row
  uint32_t off[kLoads];                 // byte offset of this lane's piece from the tile's base

  // which row (row form) or k (column form) of the tile load i's lane holds,
  // and its first k or column
  __device__ static __forceinline__ int outer(int i, int wave, int lane) {
    const int li = wave + W * i;
    return COLUMN ? li * (64 / kLanes) + lane / kLanes : 8 * li + (lane >> 3);
  }
  __device__ static __forceinline__ int inner(int i, int wave, int lane) {
    const int li = wave + W * i;
    if (!COLUMN) return 8 * ((lane & 7) ^ (lane >> 3) ^ (li & 1));
    const int p = lane % kLanes, c = (p >> 1) ^ (column_swizzle(outer(i, wave, lane)) & (R / 16 - 1));
    return 16 * c + 8 * (p & 1);
  }
  // `left`: rows (row form) or columns (column form) of the matrix from the
  // tile's first on; what lies past them repeats the last ones and never
  // reaches an output.
  __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int64_t left) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      int o = outer(i, wave, lane), c = inner(i, wave, lane);
      if (!COLUMN && o >= left) o = static_cast<int>(left) - 1;
      if (COLUMN && c >= left) c = static_cast<int>(left) - 8;
      off[i] = static_cast<uint32_t>((o * ld + c) * 2);
    }
  }
  __device__ __forceinline__ void issue(const uint16_t* base, int wave, uint32_t lds) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_lds16(base, off[i], lds + (wave + W * i) * 1024);
  }
  // The last, partial step: k_left k's (of which the row form has a multiple
  // of 8), zeros after them.
  __device__ __forceinline__ void issue_tail(const uint16_t* base, int wave, int lane, int k_left, uint8_t* lds) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      u32x4 v = {0, 0, 0, 0};
      const int k = COLUMN ? outer(i, wave, lane) : inner(i, wave, lane);
      if (k < k_left) v = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(base) + off[i]);
      *reinterpret_cast<u32x4*>(lds + (wave + W * i) * 1024 + 16 * lane) = v;
    }
  }
};

// The bf16 values 128 + q of 8 codes, or-ed into the mantissa of 128 and so
// exact: 11 instructions.
__device__ __forceinline__ u32x4 code_values(uint32_t v) {
  const uint32_t even = v & 0x0F0F0F0Fu, odd = (v >> 4) & 0x0F0F0F0Fu;
  constexpr uint32_t kPair[4] = {0x0C040C00u, 0x0C050C01u, 0x0C060C02u, 0x0C070C03u};  // bytes i of both, zeros between
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(odd, even, kPair[i]) | 0x43004300u;
  return w;
}

// What a group's sum x (128 + q) and sum x are multiplied by: scale and base,
//   sum x (scale q + offset) = scale (sum x (128 + q)) + base (sum x).
__device__ __forceinline__ float code_base(float scale, bool offsets, float offset) {
  return offsets ? offset - 128.0f * scale : -136.0f * scale;
}

// 4-bit rows into a row-form stage of R rows by T threads: a thread takes 32
// codes (16 bytes, within one group) of a row, fetched a step ahead, and
// writes their values, and beside the stage the scale and base of their group,
// [group of GROUP columns][scale, base][R].
template <int R, int T, int GROUP, bool F32>
struct CodeStager {
  static_assert(R * 2 == T, "32 codes a thread");
  u32x4 codes;
  float scale, offset;
  const uint8_t* row;
  int64_t table;
  int at;  // byte of the row's piece 0 in the stage, without the slot
  int mix, half, r;

  __device__ __forceinline__ void init(const Gemm16Args& g, int64_t n0, int64_t n, int64_t k) {
    r = threadIdx.x >> 1;
    half = threadIdx.x & 1;
    const int64_t nr = n0 + r < n ? n0 + r : n - 1;
    row = g.codes + nr * (k >> 1);
    table = nr * (k >> g.group_log2);
    at = (r >> 4) * kOperandTile + (r & 15) * 128;
    mix = (r & 7) ^ ((r >> 3) & 1);
  }
  __device__ __forceinline__ void fetch(const Gemm16Args& g, int64_t kk) {
    const int64_t k = kk + 32 * half;
    if (k >= g.k) {  // the half step past the last k
      codes = (u32x4){0, 0, 0, 0};
      scale = offset = 0.0f;
      return;
    }
    codes = *reinterpret_cast<const u32x4*>(row + (k >> 1));
    const int64_t t = table + (k >> g.group_log2);
    scale = table_value(g.scales, F32, t);
    // without offsets: the scale, read again, so that both loads are on their
    // way before either is waited for
    offset = table_value(g.offsets != nullptr ? g.offsets : g.scales, F32, t);
  }
  __device__ __forceinline__ void write(uint8_t* stage, float* tables, bool offsets) const {
#pragma unroll
    for (int d = 0; d < 4; ++d)
      *reinterpret_cast<u32x4*>(stage + at + 16 * ((4 * half + d) ^ mix)) = code_values(codes[d]);
    if (GROUP == 32 || half == 0) {
      float* t = tables + (GROUP == 32 ? half : 0) * 2 * R + r;
      t[0] = scale;
      t[R] = code_base(scale, offsets, offset);
    }
  }
};

// MFMA operand j (0, 1) of 16-row or 16-column tile t of a stage.  HALVES (row
// form): j contracts k = 32 j + 8 (l / 16) + 0..7, a half of the step's columns,
// instead of the pieces that the staging comment names.
template <int R, bool COLUMN, bool HALVES = false>
struct Reader {
  uint32_t lo, hi;  // row form: a tile's two pieces; column form: row base and swizzle
  __device__ __forceinline__ Reader(int lane) {
    const int r = lane & 15, kq = lane >> 4;
    if (!COLUMN) {
      const int g = (r & 7) ^ (r >> 3);
      lo = 128 * r + 16 * ((HALVES ? kq : 2 * kq) ^ g);
      hi = 128 * r + 16 * ((HALVES ? 4 + kq : 2 * kq + 1) ^ g);
    } else {
      lo = (16 * kq + (r >> 2)) * (2 * R) + 8 * (r & 3);
      hi = ((r >> 2) | ((kq & 1) << 2)) & (R / 16 - 1);
    }
  }
  __device__ __forceinline__ bf16x8 operator()(const uint8_t* stage, int t, int j) const {
    if constexpr (!COLUMN) {
      return *reinterpret_cast<const bf16x8*>(stage + t * kOperandTile + (j ? hi : lo));
    } else {
      typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
      const uint8_t* p = stage + lo + 32 * (static_cast<uint32_t>(t) ^ hi) + 8 * j * (2 * R);
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p));
      const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 4 * (2 * R)));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// Tile number t of `tiles` for workgroup b: consecutive workgroups go to the
// XCDs in turn, so workgroup b takes number b / 8 of XCD b % 8's run of
// consecutive tiles, which share rows and columns in that XCD's L2.
__device__ __forceinline__ int xcd_tile(int b, int tiles) {
  const int q = tiles / 8, r = tiles % 8, x = b % 8;
  return x * q + (x < r ? x : r) + b / 8;
}

// Tile (row, column) number t of rows x cols, in bands of `group` tile rows.
__device__ __forceinline__ void band_tile(int t, int rows, int cols, int group, int& tm, int& tn) {
  const int band = t / (group * cols), first = band * group;
  const int high = rows - first < group ? rows - first : group;
  const int in = t - band * group * cols;
  tm = first + in % high;
  tn = in / high;
}

// Tiles of `size` over m or n, which are below 2^31.
__device__ __forceinline__ int tiles_of(int64_t n, int size) {
  return static_cast<int>((static_cast<uint32_t>(n) + static_cast<uint32_t>(size) - 1) / static_cast<uint32_t>(size));
}

// WM x WN wavefronts, each MT x NT MFMA tiles of 16 x 16; SUB blocks of 64 k a
// step and stage: small tiles multiply a block faster than its loads return, so
// they take two blocks between barriers.  GROUP (4-bit products): columns whose
// sums are scaled at once, 32 or 64.
template <int WM, int WN, int MT, int NT, int SUB, bool A_COLUMN, OperandForm B, Gemm16Epilogue EPI, int GROUP = 64>
struct Gemm16 {
  static constexpr int W = WM * WN, kThreads = 64 * W;
  static constexpr int BM = 16 * WM * MT, BN = 16 * WN * NT;
  static constexpr bool kAColumn = A_COLUMN, B_COLUMN = B == kColumn, kFromCodes = B == kCodes || B == kCodesF32;
  static constexpr bool kPairB = EPI == kSwiglu;           // half the tile gate columns, half up
  static constexpr int kColumns = kPairB ? BN / 2 : BN;    // output columns of a tile
  static constexpr int kStageA = BM * 128, kBlock = kStageA + BN * 128, kStage = SUB * kBlock;
  // Small tiles multiply a stage in less than its loads' way, and one workgroup
  // fills a CU's LDS anyway: a third stage, loaded two steps ahead.  Codes, which
  // pass through registers, are one step ahead.
  static constexpr int kStages = SUB == 2 && !kFromCodes ? 3 : 2;
  // 4-bit products: scales and bases of a stage's groups, behind all stages
  static constexpr bool kScaled = EPI == kBias;
  static_assert(!kScaled || kFromCodes || (B == kCodeValues && BN == 128 && kStages == 2), "tables of 128 columns");
  static constexpr int kParts = SUB * 64 / GROUP, kTable = 2 * BN;
  static constexpr int kTableStage = kScaled ? kParts * kTable * 4 : 0;
  static constexpr int kLds = kStages * (kStage + kTableStage);
  // direct loads of a wavefront and stage
  static constexpr int kStageLoads = SUB * (BM + BN) / 8 / W;

  static constexpr int kReadA = A_COLUMN ? 2 : 1, kReadB = B_COLUMN ? 2 : 1;  // LDS reads of an operand
  static constexpr int kAhead = 2;

  __device__ static __forceinline__ void schedule_step() {
    constexpr int kMfma = 0x008, kLdsRead = 0x100;
    constexpr int kGroups = MT / kAhead;
    __builtin_amdgcn_sched_group_barrier(kLdsRead, NT * kReadB + kAhead * kReadA, 0);
#pragma unroll
    for (int j = 0; j < 2 * SUB; ++j) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        if (i + 1 < kGroups)
          __builtin_amdgcn_sched_group_barrier(kLdsRead, kAhead * kReadA, 0);
        else if (j + 1 < 2 * SUB)
          __builtin_amdgcn_sched_group_barrier(kLdsRead, NT * kReadB + kAhead * kReadA, 0);
        __builtin_amdgcn_sched_group_barrier(kMfma, kAhead * NT, 0);
      }
    }
  }

  // A step of a 4-bit product: acc += scale (sum x (128 + q)) + base (sum x) for
  // each group's part of it, sums of x by an MFMA with ones.  The codes' values
  // are exact, scales and bases FP32: no weight is rounded.  A weight rounded to
  // bf16 would be off by half a step of the offset, which a group whose range is
  // small against it does not get back; the price is a quarter more MFMAs and two
  // FMAs a result and part: 2,048 x 4096 x 4096 in groups of 64 102 us instead of
  // 74, in groups of 32 129 instead of 75, 64 rows 21 instead of 20.
  template <class RA, class RB>
  __device__ static __forceinline__ void multiply_scaled(f32x4 (&acc)[MT][NT], const uint8_t* stage, const float* tables,
                                                         const RA& ra, const RB& rb, int wm, int wn, int lane) {
    constexpr int J = GROUP / 32;  // MFMAs of a part
    const u32x4 one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
    const bf16x8 ones = __builtin_bit_cast(bf16x8, one);
    const f32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const uint8_t* block = stage + part * GROUP / 64 * kBlock;
      const int j0 = J == 2 ? 0 : part & 1;
      bf16x8 a[MT][J], b[NT][J];
      f32x4 scale[NT], base[NT], sum[MT];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const float* t = tables + part * kTable + 16 * (wn * NT + c) + 4 * (lane >> 4);
        scale[c] = *reinterpret_cast<const f32x4*>(t);
        base[c] = *reinterpret_cast<const f32x4*>(t + BN);
#pragma unroll
        for (int j = 0; j < J; ++j) b[c][j] = rb(block + kStageA, wn * NT + c, j0 + j);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        sum[i] = zero;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          a[i][j] = ra(block, wm * MT + i, j0 + j);
          sum[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, a[i][j], sum[i], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          f32x4 d = zero;
#pragma unroll
          for (int j = 0; j < J; ++j) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[c][j], a[i][j], d, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][c][e] = fmaf(scale[c][e], d[e], fmaf(base[c][e], sum[i][e], acc[i][c][e]));
        }
    }
  }

  __device__ static __forceinline__ void run(const Gemm16Args& g, uint8_t* lds) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    // tile, split and problem
    const int tiles = static_cast<int>(g.tiles), unit = xcd_tile(blockIdx.x, tiles * g.splits);
    const int split = g.splits > 1 ? unit / tiles : 0;
    int t = unit - split * tiles, q = 0;
    int rows = tiles_of(g.pair[0].m, BM), cols = tiles_of(g.pair[0].n, kColumns);
    while (q + 1 < g.problems && t >= rows * cols) {
      t -= rows * cols;
      ++q;
      rows = tiles_of(g.pair[q].m, BM);
      cols = tiles_of(g.pair[q].n, kColumns);
    }
    const Gemm16Pair& p = g.pair[q];
    int tm, tn;
    band_tile(t, rows, cols, g.group_m, tm, tn);
    const int64_t m0 = static_cast<int64_t>(tm) * BM, n0 = static_cast<int64_t>(tn) * kColumns;

    // K steps of this split, counted over all segments
    constexpr int kStep = SUB * kStepK;
    const int steps = static_cast<int>((g.k + kStep - 1) / kStep), all = steps * g.segments;
    const int each = (all + g.splits - 1) / g.splits;
    const int first = split * each, last = first + each < all ? first + each : all;
    const int tail = static_cast<int>(g.k % kStep);

    Stager<BM, W, A_COLUMN> sa;
    sa.init(wave, lane, p.lda, p.m - m0);
    constexpr int kHalves = kPairB ? 2 : 1;
    Stager<BN / kHalves, W, B_COLUMN> sb;
    sb.init(wave, lane, p.ldb, p.n - n0);
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds));
    CodeStager<kFromCodes ? BN : kThreads / 2, kThreads, GROUP, B == kCodesF32> sq[SUB];
    if constexpr (kFromCodes) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) sq[u].init(g, n0, p.n, g.k);
    }
    const auto fetch_codes = [&](int step) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) sq[u].fetch(g, static_cast<int64_t>(step) * kStep + u * kStepK);
    };
    float* const tables = reinterpret_cast<float*>(lds + kStages * kStage);
    const auto table_at = [&](int slot, int part) { return (slot * kParts + part) * kTable; };
    const auto write_codes = [&](int slot) {
#pragma unroll
      for (int u = 0; u < SUB; ++u)
        sq[u].write(lds + slot * kStage + u * kBlock + kStageA, tables + table_at(slot, u * (64 / GROUP)), g.offsets != nullptr);
    };
    // Where the next step's operands start; a step on costs two additions.
    const uint16_t *pa, *pb[kHalves];
    int left;  // steps of the segment still to issue
    const auto seek = [&](int segment, int step) {
      const Gemm16Pair& o = g.pair[g.segments > 1 ? segment : q];
      const int64_t kk = static_cast<int64_t>(step) * kStep;
      pa = o.a + (A_COLUMN ? kk * p.lda + m0 : m0 * p.lda + kk);
      const int64_t b_at = B_COLUMN ? kk * p.ldb + n0 : n0 * p.ldb + kk;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) pb[h] = (kPairB ? g.pair[h].b : o.b) + b_at;
      left = steps - step;
    };
    // the column whose group's table this wavefront loads for the next step, if one
    int64_t table_k = static_cast<int64_t>(first) * kStep + wave * GROUP;
    int segment = first / steps;
    seek(segment, first - segment * steps);
    const int64_t next_a = A_COLUMN ? kStepK * p.lda : kStepK, next_b = B_COLUMN ? kStepK * p.ldb : kStepK;
    const auto issue = [&](int slot) {
      const bool partial = tail != 0 && left == 1;
      // the count that stage_wait leaves open is of direct loads: none older than
      // a partial stage, of which a wavefront may have no load at all
      if (kStages > 2 && partial) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const uint32_t at = slot * kStage + u * kBlock;
        const int k_left = tail - u * kStepK;  // in a partial step: may be none
        if (partial)
          sa.issue_tail(pa, wave, lane, k_left, lds + at);
        else
          sa.issue(pa, wave, lds_at + at);
        pa += next_a;
        if constexpr (!kFromCodes) {
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            const uint32_t b_lds = at + kStageA + h * (BN / kHalves) * 128;
            if (partial)
              sb.issue_tail(pb[h], wave, lane, k_left, lds + b_lds);
            else
              sb.issue(pb[h], wave, lds_at + b_lds);
            pb[h] += next_b;
          }
        }
      }
      if constexpr (B == kCodeValues) {
        const int64_t k = table_k < g.k ? table_k : g.k - 1;  // past the last column: any group, whose sums are zero
        if (wave < kParts)
          load_lds16(g.tables + ((k >> g.group_log2) * cols + tn) * kTable, 16 * lane,
                     lds_at + kStages * kStage + 4 * table_at(slot, wave));
        table_k += kStep;
      }
      if (--left == 0 && ++segment < g.segments) seek(segment, 0);
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int c = 0; c < NT; ++c) acc[i][c] = (f32x4){0, 0, 0, 0};
    const Reader<BM, A_COLUMN, GROUP == 32> ra(lane);
    const Reader<BN / kHalves, B_COLUMN, GROUP == 32> rb(lane);
    // LDS tile of the wavefront's column tile c: in a pair, the first half of
    // its tiles are gate columns, the others the up columns of the same outputs
    const auto b_tile = [&](int c) {
      return kPairB ? (c < NT / 2 ? wn * (NT / 2) + c : BN / 32 + wn * (NT / 2) + c - NT / 2) : wn * NT + c;
    };

    if constexpr (kFromCodes) {
      if (first < last) {
        fetch_codes(first);
        write_codes(0);
        if (first + 1 < last) fetch_codes(first + 1);
      }
    }
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s)
      if (first + s < last) issue(s);
    int slot = 0;
    for (int step = first; step < last; ++step, slot = slot + 1 < kStages ? slot + 1 : 0) {
      // the stage after this one may still be on its way
      if (kStages == 3 && step + 1 < last)
        stage_wait<kStages == 3 ? kStageLoads : 0>();
      else
        stage_wait<0>();
      if constexpr (kFromCodes) {  // codes before the direct loads: the compiler's wait for them drains both
        if (step + 1 < last) write_codes(slot ^ 1);
      }
      if (step + kStages - 1 < last) issue(slot > 0 ? slot - 1 : kStages - 1);  // the stage read a step ago
      if constexpr (kFromCodes) {
        if (step + 2 < last) fetch_codes(step + 2);
      }
      const uint8_t* stage = lds + slot * kStage;
if constexpr (kScaled) {
        multiply_scaled(acc, stage, tables + table_at(slot, 0), ra, rb, wm, wn, lane);
        continue;
      }
#pragma unroll
      for (int j = 0; j < 2 * SUB; ++j) {
        bf16x8 a[MT], b[NT];
        const uint8_t* block = stage + (j >> 1) * kBlock;
#pragma unroll
        for (int c = 0; c < NT; ++c) b[c] = rb(block + kStageA, b_tile(c), j & 1);
#pragma unroll
        for (int i = 0; i < MT; ++i) a[i] = ra(block, wm * MT + i, j & 1);
        // columns as the MFMA's rows: a lane's four results are four
        // consecutive outputs of one row
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int c = 0; c < NT; ++c)
            acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[c], a[i], acc[i][c], 0, 0, 0);
      }
      // The order of a step's LDS reads and products: rows' operands are read
      // one group of kAhead row tiles ahead of the products that take them
      // (left alone, the compiler reads each pair just before its products).
      schedule_step();
    }

    const int64_t ldp = partial_ld(p.n), plane = p.m * ldp;
    float* part = g.partial + g.partial_at[q] + split * (kPairB ? 2 : 1) * plane;
    constexpr int kOut = kPairB ? NT / 2 : NT;  // column tiles of outputs
    const auto row = [&](int i) { return m0 + 16 * (wm * MT + i) + (lane & 15); };
    const auto col = [&](int c) { return n0 + 16 * (wn * kOut + c) + 4 * (lane >> 4); };
    if constexpr (EPI == kSwigluGrad) {
      if (g.splits == 1) {
        // G and U of a row of tiles come while the row before is finished;
        // without a branch around the loads (past an edge they repeat it),
        // which would have each wait for the one before.
        f32x4 gate[2][NT], up[2][NT];
        const auto load = [&](int i) {
          const int64_t m = row(i) < p.m ? row(i) : p.m - 1;
#pragma unroll
          for (int c = 0; c < NT; ++c) {
            const int64_t at = m * p.n + (col(c) < p.n ? col(c) : p.n - 4);
            gate[i & 1][c] = *reinterpret_cast<const f32x4*>(g.gate + at);
            up[i & 1][c] = *reinterpret_cast<const f32x4*>(g.up + at);
          }
        };
        load(0);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (i + 1 < MT) load(i + 1);
#pragma unroll
          for (int c = 0; c < NT; ++c)
            if (row(i) < p.m && col(c) < p.n)
              store_swiglu_grad(g, p, row(i), col(c), acc[i][c], gate[i & 1][c], up[i & 1][c]);
        }
        return;
      }
    }
    bool all_finite = true;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t m = row(i);
      if (m >= p.m) continue;
#pragma unroll
      for (int c = 0; c < kOut; ++c) {
        const int64_t n = col(c);
        if (n >= p.n) continue;
        if (g.splits > 1) {
          *reinterpret_cast<f32x4*>(part + m * ldp + n) = acc[i][c];
          if constexpr (kPairB) *reinterpret_cast<f32x4*>(part + plane + m * ldp + n) = acc[i][c + NT / 2];
        } else if constexpr (EPI == kStore) {
          store_plain(g, p, m, n, acc[i][c]);
        } else if constexpr (EPI == kBias) {
          store_bias(g, p, m, n, acc[i][c]);
          all_finite = all_finite && finite(acc[i][c]);
        } else if constexpr (EPI == kSwiglu) {
          store_swiglu(g, p, m, n, acc[i][c], acc[i][c + NT / 2]);
        }
      }
    }
    if constexpr (EPI == kBias) {
      if (all_finite) return;
#pragma unroll 1
      for (int t = 0; t < MT * kOut; ++t) {
        const int64_t m = row(t / kOut), n = col(t % kOut);
        if (m < p.m && n < p.n) store_bias_again(g, p, m, n);
      }
    }
  }
};

template <class G>
__global__ __launch_bounds__(G::kThreads) void gemm16_kernel(Gemm16Args g) {
  extern __shared__ __align__(1024) uint8_t lds[];
  G::run(g, lds);
}

// Adds the splits' partial results, in their order, and finishes them; problem
// blockIdx.y.
template <Gemm16Epilogue EPI>
__global__ __launch_bounds__(256) void gemm16_join_kernel(Gemm16Args g) {
  const Gemm16Pair& p = g.pair[blockIdx.y];
  const float* partial = g.partial + g.partial_at[blockIdx.y];
  const int64_t ldp = partial_ld(p.n), plane = p.m * ldp, at = 4 * (blockIdx.x * int64_t{256} + threadIdx.x);
  if (at >= plane) return;
  constexpr int kPlanes = EPI == kSwiglu ? 2 : 1;
  const int64_t m = at / ldp, n = at % ldp;
  if (n >= p.n) return;
  f32x4 gate, up;
  if constexpr (EPI == kSwigluGrad) {
    gate = *reinterpret_cast<const f32x4*>(g.gate + m * p.n + n);
    up = *reinterpret_cast<const f32x4*>(g.up + m * p.n + n);
  }
  // four splits' loads on their way at once, past the last one it again
  f32x4 v[kPlanes];
#pragma unroll
  for (int h = 0; h < kPlanes; ++h) v[h] = (f32x4){0, 0, 0, 0};
  for (int s = 0; s < g.splits; s += 4) {
    f32x4 t[4][kPlanes];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < kPlanes; ++h) {
        const int one = s + i < g.splits ? s + i : g.splits - 1;
        t[i][h] = *reinterpret_cast<const f32x4*>(partial + (one * kPlanes + h) * plane + at);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < kPlanes; ++h)
        if (s + i < g.splits) v[h] += t[i][h];
  }
  if constexpr (EPI == kStore)
    store_plain(g, p, m, n, v[0]);
  else if constexpr (EPI == kBias) {
    store_bias(g, p, m, n, v[0]);
    if (!finite(v[0])) store_bias_again(g, p, m, n);
  } else if constexpr (EPI == kSwiglu)
    store_swiglu(g, p, m, n, v[0], v[1]);
  else
    store_swiglu_grad(g, p, m, n, v[0], gate, up);
}

// ---------------------------------------------------------------- host ---

enum Gemm16Tile { kTile64, kTile128, kTile256 };
struct Gemm16Plan {
  Gemm16Tile tile;
  int splits;
  int64_t partial;  // floats of the splits' partial results
  float us;         // expected time
};
// `steps` K steps in at most `splits` parts of the same number of steps, the
// last one's rest: the parts that have one.
inline int used_splits(int64_t steps, int64_t splits) {
  const int64_t each = (steps + splits - 1) / splits;
  return static_cast<int>((steps + each - 1) / each);
}
// The tile and the number of splits for g's products; pair_b: gate and up
// columns in one product.
Gemm16Plan gemm16_plan(const Gemm16Args& g, bool pair_b);
// The same for a 4-bit product of code values and tables (kCodeValues).
Gemm16Plan gemm16_plan_scaled(const Gemm16Args& g);

template <class G, Gemm16Epilogue EPI>
hipError_t gemm16_launch(Gemm16Args g, hipStream_t st) {
  constexpr int64_t kMostTiles = ((int64_t{1} << 32) - 1) / G::kThreads;  // a grid has fewer than 2^32 threads
  g.tiles = 0;
  g.group_m = 8;
  int64_t most = 0, at = 0;
  const auto tile_columns = [](const Gemm16Pair& p) { return (p.n + G::kColumns - 1) / G::kColumns; };
  for (int q = 0; q < g.problems; ++q) {
    const Gemm16Pair& p = g.pair[q];
    g.tiles += ((p.m + G::BM - 1) / G::BM) * tile_columns(p);
    const int64_t plane = p.m * partial_ld(p.n);
    g.partial_at[q] = at;
    at += plane * g.splits * (EPI == kSwiglu ? 2 : 1);
    most = most > plane ? most : plane;
  }
  if (g.splits > 1 && (at > g.room || (most + 1023) / 1024 * 256 >= (int64_t{1} << 32))) return hipErrorInvalidValue;
  if (g.tiles * g.splits > kMostTiles) {
    // One product over very many rows, whole: a launch for each band of rows.
    const int64_t columns = tile_columns(g.pair[0]), rows = g.pair[0].m, band = kMostTiles / columns * G::BM;
    if (g.problems != 1 || g.splits != 1 || band == 0) return hipErrorInvalidValue;
    for (int64_t first = 0; first < rows; first += band) {
      Gemm16Args part = g;
      for (Gemm16Pair& p : part.pair) {
        if (p.a != nullptr) p.a += G::kAColumn ? first : first * p.lda;
        if (p.out != nullptr) p.out += first * p.ldo;
        p.m = rows - first < band ? rows - first : band;
      }
      const int64_t values = first * g.pair[0].n;
      for (float** p : {&part.gate, &part.up})
        if (*p != nullptr) *p += values;
      for (uint16_t** p : {&part.d_gate, &part.d_up})
        if (*p != nullptr) *p += values;
      part.tiles = (part.pair[0].m + G::BM - 1) / G::BM * columns;
      gemm16_kernel<G><<<static_cast<uint32_t>(part.tiles), G::kThreads, G::kLds, st>>>(part);
      if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  gemm16_kernel<G><<<static_cast<uint32_t>(g.tiles * g.splits), G::kThreads, G::kLds, st>>>(g);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || g.splits == 1) return e;
  const dim3 grid(static_cast<uint32_t>((most + 1023) / 1024), static_cast<uint32_t>(g.problems));
  gemm16_join_kernel<EPI><<<grid, 256, 0, st>>>(g);
  return hipGetLastError();
}

// g's products in the plan's shape.
template <bool A_COLUMN, OperandForm B, Gemm16Epilogue EPI>
hipError_t gemm16(Gemm16Args g, const Gemm16Plan& plan, hipStream_t st) {
  g.splits = plan.splits;
  switch (plan.tile) {
    case kTile64: return gemm16_launch<Gemm16<1, 4, 4, 2, 2, A_COLUMN, B, EPI>, EPI>(g, st);  // 64 x 128
    case kTile128: return gemm16_launch<Gemm16<2, 2, 4, 4, 1, A_COLUMN, B, EPI>, EPI>(g, st);
    default: return gemm16_launch<Gemm16<2, 4, 8, 4, 1, A_COLUMN, B, EPI>, EPI>(g, st);
  }
}

}  // namespace glm53
