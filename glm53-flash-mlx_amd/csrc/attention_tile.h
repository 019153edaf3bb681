// What the attention kernels share: tiles of rows in LDS, read along their
// rows and across them, the 32 x 32 MFMA, and the parts of a softmax.
//
// A tile holds rows of DP bf16 values (head_dim, zeros up to DP) at a pitch of
// 128, 256 or 512 bytes, the 16-byte piece p of row r at slot p ^ g(r).  A row
// operand (lane l: row l % 32, 8 values from 16 j + 8 (l / 32)) reads one slot
// of 16 consecutive rows at a time, a transposed one (ds_read_b64_tr_b16: 4
// rows x 16 columns a 16 lanes) four slots of four rows: g puts both on
// distinct banks.
//
// MFMA operands, 32 x 32 x 16: lane l holds row or column l % 32 and
// contraction indexes 8 (l / 32) .. + 7; result register r of lane l is row 8
// (r / 4) + 4 (l / 32) + r % 4 of column l % 32.  A product's result X[m, n] is
// the second operand of a product that contracts m without leaving its lanes:
// registers 8 i .. 8 i + 7 as the eight values of MFMA i, whose first operand's
// values are then those of rows 16 i + 4 (l / 32) + 0..3 and 16 i + 8 + 4 (l /
// 32) + 0..3, which two transposed reads bring.
#pragma once

#include "common.h"

namespace glm53 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zero16() {
  return (f32x16){0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
}

// The row of result register r (of a 32 x 32 product) that half `h` of a wavefront holds.
__device__ __forceinline__ int result_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// Of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float both_max(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float both_sum(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}

// Eight results as an operand, rounded to nearest even, and what that leaves of them.
__device__ __forceinline__ bf16x8 operand8(const f32x16& v, int i) {
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = pack2(v[8 * i + 2 * e], v[8 * i + 2 * e + 1]);
  return __builtin_bit_cast(bf16x8, o);
}
__device__ __forceinline__ bf16x8 low_operand8(const f32x16& v, int i, bf16x8 high) {
  const u32x4 w = __builtin_bit_cast(u32x4, high);
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    o[e] = pack2(v[8 * i + 2 * e] - __uint_as_float(w[e] << 16), v[8 * i + 2 * e + 1] - __uint_as_float(w[e] & 0xFFFF0000u));
  return __builtin_bit_cast(bf16x8, o);
}

__device__ __forceinline__ u32x2 pack4(float a, float b, float c, float d) {
  return (u32x2){pack2(a, b), pack2(c, d)};
}

__device__ __forceinline__ uint32_t lds_address(const uint8_t* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)p));
}

__device__ __forceinline__ const void* uniform_address(const void* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<const void*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// Direct global -> LDS load of 4 bytes a lane, each from an address of its own, to lds + 4 lane.
__device__ __forceinline__ void load_dword_to_lds(const void* p, uint32_t lds) {
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}

// Direct global -> LDS load of 16 or 4 bytes a lane, base + off, to lds + 16 (4) lane.
template <int BYTES = 16>
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t off, uint32_t lds) {
  base = uniform_address(base);
  lds = __builtin_amdgcn_readfirstlane(lds);
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds)
                 : "memory", "m0");
}

// Has the compiler wait for a loaded value here, not in a loop that reads it: its
// wait there would be for every direct load that is under way.
template <class T>
__device__ __forceinline__ void arrived(T& v) { asm volatile("" : "+v"(v)); }

// All of this wavefront's loads are done, and every wavefront of the workgroup is here.
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ROWS rows of DP values, loaded by W wavefronts.
template <int DP, int ROWS, int W>
struct HeadTile {
  static constexpr int kPitch = DP <= 64 ? 128 : DP <= 128 ? 256 : 512;
  static constexpr int kBytes = ROWS * kPitch;
  static constexpr int kSlots = kPitch / 16;     // 16-byte pieces a row
  static constexpr int kLoadRows = 64 / kSlots;  // rows of one load instruction
  static constexpr int kLoads = ROWS / kLoadRows / W;
  static constexpr bool kEven = W * kLoadRows % 16 == 0;  // a lane's rows are a multiple of 16 apart, and have one swizzle
  static_assert(ROWS % (kLoadRows * W) == 0 && ROWS % 16 == 0, "whole loads a wavefront");

  __device__ static __forceinline__ int swizzle(int row) {
    return kPitch == 128 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
  }

  // Zeros where no load writes: the pieces from `dim` on.
  __device__ static __forceinline__ void clear(uint8_t* tile, int dim, int threads) {
    for (int i = threadIdx.x; i < kBytes / 16; i += threads) {
      const int row = i / kSlots, piece = (i % kSlots) ^ swizzle(row);
      if (8 * piece >= dim) *reinterpret_cast<u32x4*>(tile + 16 * i) = (u32x4){0, 0, 0, 0};
    }
  }

  // Rows of which the first `left` (one or more) exist, row r at byte
  // offset(r) from base; those past them repeat the last one.
  template <class Offset>
  __device__ static __forceinline__ void load(const uint16_t* base, Offset offset, int left, int dim, int wave, int lane,
                                              uint32_t lds) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int first = (wave + W * i) * kLoadRows, row = first + lane / kSlots;
      const int piece = (lane % kSlots) ^ swizzle(row);
      const uint32_t off = offset(row < left ? row : left - 1) + 16 * piece;
      if (8 * piece < dim) load_to_lds(base, off, lds + first * kPitch);
    }
  }

  // The same of rows `pitch` bytes apart.
  __device__ static __forceinline__ void load(const uint16_t* base, uint32_t pitch, int left, int dim, int wave, int lane,
                                              uint32_t lds) {
    if constexpr (kEven) {
      if (left >= ROWS) {
        load_even(base, static_cast<uint32_t>(row_of(wave, lane)) * pitch + piece_of(wave, lane), uint64_t{16} * pitch, dim,
                  wave, lane, lds);
        return;
      }
    }
    load(base, [&](int row) { return static_cast<uint32_t>(row) * pitch; }, left, dim, wave, lane, lds);
  }

  // A lane's row of a wavefront's first load, and the byte of its piece.
  __device__ static __forceinline__ int row_of(int wave, int lane) { return wave * kLoadRows + lane / kSlots; }
  __device__ static __forceinline__ int piece_of(int wave, int lane) {
    return 16 * ((lane % kSlots) ^ swizzle(row_of(wave, lane)));
  }
  // A whole tile whose rows 16 apart lie `apart` bytes apart, by one offset a lane, of its
  // first row: the rest is uniform.
  __device__ static __forceinline__ void load_even(const uint16_t* base, uint32_t off, uint64_t apart, int dim, int wave,
                                                   int lane, uint32_t lds) {
    static_assert(kEven, "rows of one lane have one swizzle");
    const uint8_t* at = reinterpret_cast<const uint8_t*>(base);
    const bool in = piece_of(wave, lane) < 2 * dim;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (in) load_to_lds(at, off, lds + (wave + W * i) * kLoadRows * kPitch);
      at += W * kLoadRows / 16 * apart;
    }
  }

  // Where a lane reads a tile's operands, from the tile at LDS address `base`: the rest of an
  // address is a constant of the read.
  struct Places {
    uint32_t row[DP / 16];       // operand j of rows 0 .. 31
    uint32_t column[DP / 32][2];  // columns 32 t .. of rows 0 .. 15, its two halves

    __device__ __forceinline__ Places(uint32_t base, int lane) {
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) {
        const int r = lane & 31, piece = 2 * j + (lane >> 5);
        row[j] = base + r * kPitch + 16 * (piece ^ swizzle(r));
        arrived(row[j]);
      }
#pragma unroll
      for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int a = lane & 15, piece = 4 * t + 2 * ((lane >> 4) & 1) + ((a & 3) >> 1);
          const int r = 8 * half + 4 * (lane >> 5) + (a >> 2);
          column[t][half] = base + r * kPitch + 16 * (piece ^ swizzle(r)) + 8 * (a & 1);
          arrived(column[t][half]);
        }
    }
    // Operand j of rows 32 b .. 32 b + 31, values 16 j .. 16 j + 15, of the tile `tile` bytes on.
    __device__ __forceinline__ bf16x8 along(int tile, int b, int j) const {
      typedef __attribute__((address_space(3))) const bf16x8* lds;
      return *reinterpret_cast<lds>(row[j] + (tile + 32 * b * kPitch));
    }
    // Values 32 t .. 32 t + 31 as the operand's rows, rows 16 i .. 16 i + 15 as its
    // contraction, in the order of a result's registers (above).
    __device__ __forceinline__ bf16x8 across(int tile, int i, int t) const {
      typedef __attribute__((address_space(3))) s16x4* lds;
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds>(column[t][0] + (tile + 16 * i * kPitch)));
      const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds>(column[t][1] + (tile + 16 * i * kPitch)));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
};

// Tiles that a mask cuts: a weight that is 0 because its place is masked must
// take nothing from the values there, not even 0 x NaN.  So the careful pass
// multiplies the values of such a tile with their infinities and NaNs replaced
// by 0 (`dirty` where there was one), and what the mask lets through of those is
// added afterwards by add_nonfinite.
// With `signs` 0 a tile stays as it is.
constexpr uint32_t kSigns = 0x80008000u;
__device__ __forceinline__ bf16x8 finite_part(bf16x8 v, uint32_t& dirty, uint32_t signs = kSigns) {
  u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t bad = ((w[i] & 0x7F807F80u) + 0x00800080u) & signs;  // exponents all ones
    dirty |= bad;
    w[i] &= ~(bad | (bad - (bad >> 15)));
  }
  return __builtin_bit_cast(bf16x8, w);
}

// To a result column's registers: the infinities and NaNs of rows first .. last -
// 1, at `at(row)`, that `seen(row)` lets through.
template <int DP, class At, class Seen>
__device__ __forceinline__ void add_nonfinite(f32x16 (&acc)[DP / 32], int first, int last, int dim, int h, At at, Seen seen) {
#pragma unroll 1
  for (int row = first; row < last; ++row) {
    if (!seen(row)) continue;
    const uint16_t* p = at(row);
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * t + result_row(r, h);
        if (d >= dim) continue;
        const u32x2 v = *reinterpret_cast<const u32x2*>(p + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = bf16_to_f32(static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1))));
          if (!(fabsf(f) < INFINITY)) acc[t][r + e] += f;
        }
      }
  }
}

// Division of numbers below 2^31 by d: two multiplications' worth.
struct Divisor {
  uint32_t d, mul, shift;
  explicit Divisor(uint32_t by) : d(by), mul(0), shift(0) {
    while ((uint64_t{1} << shift) < d) ++shift;
    mul = static_cast<uint32_t>((((uint64_t{1} << shift) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int quotient(int n) const {
    return static_cast<int>((__umulhi(mul, static_cast<uint32_t>(n)) + static_cast<uint32_t>(n)) >> shift);
  }
};

// A stretch of rows of one sequence.
struct Segment {
  int first, last;  // its rows, of all: first .. last - 1
  int number;       // the sequence, or -1: rows before the first or behind the last sequence
  int tile;         // which of its tiles
};

// Where work starts.  Rows are cut into sequences and these into tiles of `size`
// (offsets and rows are multiplied by `times`); rows before the first and behind the
// last sequence are segments too.  `t` counts the workgroups, of which there
// are rows / size + sequences + 2 for packed rows; some get no tile (`tile` negative or
// behind the segment's last row).
//
// kInOrder, kReversed: the tiles one after the other; segment i's are numbered from
// floor(first row / size) + i on, so that every one has a number of its own.
// kLastFirst, kFirstFirst: those with the most tiles of their sequence before (behind) them
// first, which of a causal sequence's row (key) tiles have the most work, so that
// the short ones fill the card's last turns.  Costs ~1.5 us a workgroup.
enum TileOrder { kInOrder, kReversed, kLastFirst, kFirstFirst };
__device__ __forceinline__ Segment find_segment(const int32_t* offsets, int sequences, int64_t rows, int times, int size, int t,
                                                int tiles, TileOrder order) {
  const int lane = threadIdx.x & 63, most = static_cast<int>(rows), segments = sequences + 2;
  const bool ranked = order >= kLastFirst && offsets != nullptr && sequences > 1 && segments < 64;
  if (order == kReversed || (order == kLastFirst && !ranked)) t = tiles - 1 - t;
  if (offsets == nullptr) return Segment{0, static_cast<int>(rows * times), 0, t};
  // boundary 0 is row 0, boundary i offsets[i - 1], boundary sequences + 2 the end
  const auto boundary = [&](int i) {
    int v = i <= 0 ? 0 : i > sequences + 1 ? most : offsets[i - 1];
    v = v < 0 ? 0 : v > most ? most : v;
    return v * times;
  };
  int s, mine = 0;
  Segment g;
  if (ranked) {
    mine = boundary(lane);
    const int next = __shfl_down(mine, 1);
    const int own = lane < segments && next > mine ? (next - mine + size - 1) / size : 0;  // tiles of segment `lane`
    // tiles with `place` or more before (behind) them; sums below 2^24 are exact
    const auto from = [&](int place) { return static_cast<int>(wave_sum(static_cast<float>(own > place ? own - place : 0))); };
    int low = 0, high = tiles;  // from(low) > t, from(high) <= t
    if (from(0) <= t) return Segment{0, 0, -1, 0};
    while (high - low > 1) {
      const int mid = (low + high) >> 1;
      if (from(mid) > t)
        low = mid;
      else
        high = mid;
    }
    const int rank = t - from(low + 1);
    const uint64_t have = __ballot(own > low);
    s = __builtin_ctzll(__ballot(own > low && __popcll(have & ((uint64_t{1} << lane) - 1)) == rank));
    g.tile = order == kLastFirst ? low : __builtin_amdgcn_readlane(own, s) - 1 - low;
  } else {
    // the last segment that starts at t or before it, of s .. s + span - 1
    s = 0;
    for (int span = segments, step;; span = step) {
      step = (span + 63) / 64;
      const int i = s + lane * step;
      mine = boundary(i);
      const uint64_t upto = __ballot(lane * step < span && i < segments && mine / size + i <= t);
      s += step * (__popcll(upto) - 1);
      if (step == 1) break;
    }
  }
  if (segments < 64) {
    g.first = __builtin_amdgcn_readlane(mine, s);
    g.last = __builtin_amdgcn_readlane(mine, s + 1);
  } else {
    g.first = __builtin_amdgcn_readfirstlane(boundary(s));
    g.last = __builtin_amdgcn_readfirstlane(boundary(s + 1));
  }
  if (!ranked) g.tile = t - g.first / size - s;
  g.number = s >= 1 && s <= sequences ? s - 1 : -1;
  return g;
}

}  // namespace glm53
