// The paged key-value cache: rows written (and quantised), rows read back,
// and the attention of one token a sequence over its pages.
#include <type_traits>

#include "attention_tile.h"
#include "kv_cache.h"

namespace glm53 {

namespace {

// ---------------------------------------------------- writing and reading ---

// Which sequence row `row` of packed rows belongs to, or -1; a wavefront asks
// for one row.
__device__ __forceinline__ int sequence_of(const int32_t* offsets, int sequences, int row) {
  const int lane = threadIdx.x & 63;
  int s = -1;  // the last one that starts at the row or before it is one of s .. s + span - 1
  for (int span = sequences + 2, step;; span = step) {
    step = (span + 63) / 64;
    const int i = s + lane * step;
    const uint64_t upto = __ballot(lane * step < span && i <= sequences && (i < 0 || offsets[i] <= row));
    s += step * (__popcll(upto) - 1);
    if (step == 1) break;
  }
  return s < sequences ? s : -1;
}

// Number of the cache row of a sequence's position, without its head: page *
// kv_heads << page_log2 and the token in the page; -1 where it has no page.
struct Place {
  int64_t page;
  int token;
};
__device__ __forceinline__ Place place_of(const CacheArgs& c, int sequence, int64_t position) {
  const int64_t n = position >> c.page_log2;
  if (position < 0 || n >= c.max_pages) return Place{-1, 0};
  const int page = c.table[sequence * c.table_stride + n];
  return Place{page >= 0 && page < c.pages ? page : -1, static_cast<int>(position & ((1 << c.page_log2) - 1))};
}

__device__ __forceinline__ int64_t cache_row(const CacheArgs& c, const Place& p, int head) {
  return ((p.page * c.kv_heads + head) << c.page_log2) + p.token;
}

// The power of two that a row whose largest finite |x| is `top` is divided by:
// the smallest 2^e with top <= 448 * 2^e, 2^-117 or more, so that the smallest
// code times it is still a normal number.
__device__ __forceinline__ int row_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e < -117 ? -117 : e;
}

// A wavefront writes one token: its rows of keys and values by groups of LANES
// lanes, 8 values a lane.  Every code is one conversion of x * 2^-e, whose
// product is exact or far below the smallest code; |x| * 2^-e <= 448, so nothing
// saturates.  Bound by the bytes; 4,096 tokens of 8 heads of 128 to E4M3: 9.4 us.
template <bool E4M3, int LANES>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const CacheArgs& c = a.cache;
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= a.tokens) return;
  int sequence = row, place = 0;
  if (a.offsets != nullptr) {
    sequence = sequence_of(a.offsets, c.sequences, row);
    if (sequence < 0) return;
    place = row - a.offsets[sequence];
  }
  const Place at = place_of(c, sequence, static_cast<int64_t>(a.lengths[sequence]) + place);
  if (at.page < 0) return;
  const int piece = lane % LANES;
  for (int i = lane / LANES; i < 2 * c.kv_heads; i += 64 / LANES) {
    const bool values = i >= c.kv_heads;
    const int head = values ? i - c.kv_heads : i;
    const Rows16& x = values ? a.rows_v : a.rows_k;
    const bool in = 8 * piece < c.dim;
    u32x4 w = {0, 0, 0, 0};
    if (in) w = *reinterpret_cast<const u32x4*>(x.p + row * x.token + head * x.head + 8 * piece);
    const int64_t to = cache_row(c, at, head);
    if constexpr (!E4M3) {
      if (in) *reinterpret_cast<u32x4*>((values ? c.v : c.k) + (to * c.dim + 8 * piece) * 2) = w;
    } else {
      float f[8], top = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = bf16_to_f32(static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1))));
        if (fabsf(f[j]) < INFINITY) top = fmaxf(top, fabsf(f[j]));
        else f[j] = NAN;
      }
#pragma unroll
      for (int s = LANES / 2; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, LANES));
      const int e = row_exponent(top);
      const float by = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      if (e == 120) {  // the next code after 240 is 2^128, no bf16 number
        const float most = 240.0f / by;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = f[j] > most ? most : f[j] < -most ? -most : f[j];
      }
      u32x2 codes = {0, 0};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        codes[j] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * j] * by, f[4 * j + 1] * by, codes[j], false);
        codes[j] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * j + 2] * by, f[4 * j + 3] * by, codes[j], true);
      }
      if (in) *reinterpret_cast<u32x2*>((values ? c.v : c.k) + to * c.dim + 8 * piece) = codes;
      if (piece == 0) (values ? c.v_scales : c.k_scales)[to] = static_cast<uint8_t>(e + 127);
    }
  }
}

// Four E4M3 codes times 2^(scale - 127) as bf16, exact.
__device__ __forceinline__ u32x2 codes_to_bf16(uint32_t codes, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false);
  const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true);
  return (u32x2){__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte << 23); }

// A wavefront reads one token.  Bound by the bytes: 34,096 tokens of 8 heads of 128
// from E4M3 33.5 us, 6.2 TB/s (partly of the last-level cache).
template <bool E4M3, int LANES>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  const CacheArgs& c = a.cache;
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int sequence = sequence_of(a.offsets, c.sequences, row);
  Place at{-1, 0};
  if (sequence >= 0) at = place_of(c, sequence, row - a.offsets[sequence]);
  const uint32_t none = sequence >= 0 ? 0x7FC07FC0u : 0u;
  const int piece = lane % LANES;
  if (8 * piece >= c.dim) return;
  for (int i = lane / LANES; i < 2 * c.kv_heads; i += 64 / LANES) {
    const bool values = i >= c.kv_heads;
    const int head = values ? i - c.kv_heads : i;
    uint16_t* to = values ? a.v : a.k;
    if (to == nullptr) continue;
    u32x4 w = {none, none, none, none};
    if (at.page >= 0) {
      const int64_t from = cache_row(c, at, head);
      const uint8_t* p = values ? c.v : c.k;
      if constexpr (!E4M3) {
        w = *reinterpret_cast<const u32x4*>(p + (from * c.dim + 8 * piece) * 2);
      } else {
        const u32x2 codes = *reinterpret_cast<const u32x2*>(p + from * c.dim + 8 * piece);
        const float scale = scale_value((values ? c.v_scales : c.k_scales)[from]);
        const u32x2 lo = codes_to_bf16(codes[0], scale), hi = codes_to_bf16(codes[1], scale);
        w = (u32x4){lo[0], lo[1], hi[0], hi[1]};
      }
    }
    *reinterpret_cast<u32x4*>(to + (static_cast<int64_t>(row) * c.kv_heads + head) * c.dim + 8 * piece) = w;
  }
}

}  // namespace

hipError_t launch_append(const AppendArgs& a, hipStream_t st) {
  const int dim = a.cache.dim;
  const uint32_t grid = static_cast<uint32_t>((a.tokens + 3) / 4);
  if (a.cache.e4m3) {
    if (dim <= 64) append_kernel<true, 8><<<grid, 256, 0, st>>>(a);
    else if (dim <= 128) append_kernel<true, 16><<<grid, 256, 0, st>>>(a);
    else append_kernel<true, 32><<<grid, 256, 0, st>>>(a);
  } else {
    if (dim <= 64) append_kernel<false, 8><<<grid, 256, 0, st>>>(a);
    else if (dim <= 128) append_kernel<false, 16><<<grid, 256, 0, st>>>(a);
    else append_kernel<false, 32><<<grid, 256, 0, st>>>(a);
  }
  return hipGetLastError();
}

hipError_t launch_read(const ReadArgs& a, hipStream_t st) {
  const int dim = a.cache.dim;
  const uint32_t grid = static_cast<uint32_t>((a.rows + 3) / 4);
  if (a.cache.e4m3) {
    if (dim <= 64) read_kernel<true, 8><<<grid, 256, 0, st>>>(a);
    else if (dim <= 128) read_kernel<true, 16><<<grid, 256, 0, st>>>(a);
    else read_kernel<true, 32><<<grid, 256, 0, st>>>(a);
  } else {
    if (dim <= 64) read_kernel<false, 8><<<grid, 256, 0, st>>>(a);
    else if (dim <= 128) read_kernel<false, 16><<<grid, 256, 0, st>>>(a);
    else read_kernel<false, 32><<<grid, 256, 0, st>>>(a);
  }
  return hipGetLastError();
}

namespace {

// ------------------------------------------------------- one token's attention ---
//
// Bound by the cache's bytes.  A wavefront, which is a workgroup of its own, streams
// TS tokens of keys and values at a time into LDS by direct loads, the next TS on
// their way while it multiplies: S^T = k q^T (16 tokens x 16 heads, the heads
// of one key head beside each other) and out^T += v^T P^T, P straight from the
// registers that S is in, values read across by the transposing LDS read.  It
// meets no barrier.
//
// The positions of every sequence and head, in chunks of TS tokens one after the
// other, are dealt to the wavefronts in equal contiguous runs, whatever the
// lengths.  A run holds the end of one (sequence, head), whole ones, which it
// finishes, and the start of another: two partial results at most, joined by a second
// launch in their order.  Workgroups of four wavefronts, a barrier a stage and a join of
// one workgroup a head took 79 us where these take 51 (131,000 tokens in bf16, 32 / 4
// heads of 128).
//
// That case reads 5.3 TB/s, 64 sequences of up to 8,192 tokens 5.7 in bf16 and 4.8 in
// E4M3 (160 us); a copy on the card reaches 5.0.  The smallest call takes 6.7 us here,
// loads that wait for each other (lengths, table, keys), and 4.9 in the join.

// Sums of weights, which reach 2^8, times values may pass FP32's range where their mean
// does not, and a weight times its row's power of two a bf16 operand's.  A head whose part of
// a run is not finite takes the run again with weights kSmaller of these, whose sum is
// below 1 over 2^31 tokens (powers of two change no bit, but of values below 2^-86 beside
// such large ones); the join takes all of its parts so.
constexpr int kHeads = 16;  // columns of the MFMA: more heads of a key head read its cache once for 16 each
constexpr float kSmaller = 0x1p-40f;

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Over the four lanes of a column.
__device__ __forceinline__ float quarter_max(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return both_max(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
}
__device__ __forceinline__ float quarter_sum(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return both_sum(__uint_as_float(x[0]) + __uint_as_float(x[1]));
}

// Sequence `s`'s tokens: 0 .. what its table holds; `whole` false where its
// length says more.
__device__ __forceinline__ int64_t tokens_of(const DecodeArgs& a, int s, bool& whole) {
  const int64_t n = a.lengths[s], most = static_cast<int64_t>(a.cache.max_pages) << a.cache.page_log2;
  whole = n <= most;
  return n < 0 ? 0 : n > most ? most : n;
}

__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
                              static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane)));
}

// How the work is dealt: units are chunks of all heads' parts of every sequence.
// Wavefronts ask; 64 sequences' numbers lie in a wavefront's lanes at a time.  More than
// 64 are 64 runs of them first, a lane's each, of which one is looked at (1,000
// sequences of 60 tokens, 32 / 8 heads: 64 us; all of them by 64: 74).
template <int WORKERS, int CHUNK>
struct Shares {
  const DecodeArgs& a;
  const int lane, head_parts, parts;  // groups of 16 heads of a key head, and of all of them
  int64_t units;                      // of all sequences
  int block;                          // sequences block .. block + 63 are in the lanes
  int64_t tokens, before;             // of the lane's sequence, and the units before it
  bool whole;
  int run;                            // sequences of a run
  int64_t run_before, run_units;      // of the lane's run

  __device__ __forceinline__ explicit Shares(const DecodeArgs& a)
      : a(a), lane(threadIdx.x & 63), head_parts((a.group + kHeads - 1) / kHeads), parts(a.cache.kv_heads * head_parts) {
    const int sequences = a.cache.sequences;
    if (sequences <= 64) {
      units = load(0, 0);
      return;
    }
    run = (sequences + 63) / 64;
    run_units = 0;
    for (int i = 0; i < run; i += 8) {
#pragma unroll
      for (int j = i; j < i + 8; ++j) {
        const int s = lane * run + j;
        bool unused;
        if (j < run && s < sequences) run_units += chunks(tokens_of(a, s, unused));
      }
    }
    run_units *= parts;
    const int64_t upto = sum_upto(run_units);
    run_before = upto - run_units;
    units = __shfl(upto, 63);
  }
  // The sum of this lane's value and of those of the lanes before it.
  __device__ __forceinline__ int64_t sum_upto(int64_t v) const {
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) {
      const int64_t left = __shfl_up(v, w);
      if (lane >= w) v += left;
    }
    return v;
  }
  __device__ __forceinline__ static int64_t chunks(int64_t tokens) { return (tokens + CHUNK - 1) / CHUNK; }
  // Takes the 64 sequences from s on, `at` units behind the start; the units behind their end.
  __device__ __forceinline__ int64_t load(int s, int64_t at) {
    block = s;
    tokens = 0;
    whole = true;
    if (s + lane < a.cache.sequences) tokens = tokens_of(a, s + lane, whole);
    const int64_t own = chunks(tokens) * parts, upto = sum_upto(own);
    before = at + upto - own;
    return at + __shfl(upto, 63);
  }
  // The sequence of unit u.
  __device__ __forceinline__ int find(int64_t u) {
    if (a.cache.sequences > 64) {
      const int in = 63 - __builtin_clzll(__ballot(run_before <= u && run_units > 0));
      int64_t end = lane_value(run_before, in);
      for (int s = in * run; s < a.cache.sequences; s += 64) {
        end = load(s, end);
        if (end > u) break;
      }
    }
    // the last one that starts at u or before it, past those without a token
    return block + 63 - __builtin_clzll(__ballot(before <= u && tokens > 0));
  }
  __device__ __forceinline__ int64_t start(int worker) const { return units * worker / WORKERS; }
  __device__ __forceinline__ int worker(int64_t u) const { return static_cast<int>(((u + 1) * WORKERS - 1) / units); }
};

// Whether not all of a lane's sums are finite.
__device__ __forceinline__ bool nonfinite(const f32x4& x) {
  return fmaf(x[0], 0.0f, x[1] * 0.0f) + fmaf(x[2], 0.0f, x[3] * 0.0f) != 0.0f;
}
template <int T>
__device__ __forceinline__ bool nonfinite(const f32x4 (&x)[T]) {
  f32x4 sum = {0, 0, 0, 0};
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[r] = fmaf(x[t][r], 0.0f, sum[r]);
  return nonfinite(sum);
}

// What a sum without a weight is divided into, with the largest scaled score: NaN of scores
// that are no FP32 numbers once scaled, 0 where there are none.
__device__ __forceinline__ float without_weights(float top) { return top == INFINITY ? NAN : 0.0f; }

// Which wavefronts have parts of one (sequence, head): first .. last, the first one its start.
struct Split {
  int sequence, part, first, last;
  int64_t units;  // of all, from which each wavefront's follow
  int64_t unused;
};

template <int DP_, bool E4M3_>
struct Decode {
  static constexpr int DP = DP_;
  static constexpr bool E4M3 = E4M3_;
  static constexpr int kRowBytes = E4M3 ? DP : 2 * DP;
  static constexpr int kPitch = kRowBytes < 128 ? 128 : kRowBytes;
  static constexpr int kSlots = kPitch / 16, kLoadRows = 64 / kSlots;
  static constexpr int TS = kPitch >= 256 ? 32 : 64, kSub = TS / 16;  // tokens of a stage, and parts of 16
  static constexpr int kTile = TS * kPitch;
  static constexpr int kStage = 2 * kTile + (E4M3 ? 128 : 0);
  static constexpr int kLds = 2 * kStage;
  // one a SIMD of 256 CUs where the LDS holds them (a fifth one a CU ends after the others:
  // 64 x 8192 tokens in bf16 470 us for 381)
  static constexpr int kWorkers = 256 * (160 * 1024 / kLds < 4 ? 160 * 1024 / kLds : 4);
  static constexpr int kLoads = 2 * (TS / kLoadRows) + E4M3;  // of a whole stage
  static constexpr int kPartial = kHeads * (DP + 2);  // floats: sums, then maximum and total of each head (negative: both kSmaller)
  static constexpr size_t kPartials = sizeof(float) * 2 * kWorkers * kPartial, kSpace = kPartials + sizeof(Split) * kWorkers;
  // What a join finds in its Split: with few (sequence, head) parts each has one, with more of them
  // each worker has that of the one which it begins and others end.
  static __device__ __forceinline__ bool by_segment(const DecodeArgs& a, int parts) {
    return static_cast<int64_t>(a.cache.sequences) * parts <= kWorkers;
  }
  static __device__ __forceinline__ Split* splits(const DecodeArgs& a) {
    return reinterpret_cast<Split*>(reinterpret_cast<uint8_t*>(a.partial) + kPartials);
  }
  using Dealt = Shares<kWorkers, TS>;

  __device__ static __forceinline__ int swizzle(int row) {
    return kPitch == 128 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
  }

  static __device__ void run(const DecodeArgs& a, uint8_t* lds) {
    const CacheArgs& c = a.cache;
    const int lane = threadIdx.x, col = lane & 15, quarter = lane >> 4;
    Dealt shares(a);
    const int worker = blockIdx.x;
    int64_t unit = shares.start(worker);
    const int64_t end = shares.start(worker + 1);
    const bool by_segment = Decode::by_segment(a, shares.parts);
    Split* splits = Decode::splits(a);
    if (!by_segment && lane == 0) splits[worker].last = -1;  // overwritten below where there is one
    if (unit >= end) return;
    int sequence = __builtin_amdgcn_readfirstlane(shares.find(unit));

    const uint32_t lds_at = lds_address(lds);
    const float sc = a.scale * 1.44269504088896340736f;
    const int row_bytes = E4M3 ? c.dim : 2 * c.dim;
    if (row_bytes < kPitch) {  // pads, where no load writes
      for (int i = lane; i < kLds / 16; i += 64) *reinterpret_cast<u32x4*>(lds + 16 * i) = (u32x4){0, 0, 0, 0};
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }

    while (unit < end) {
      if (sequence >= shares.block + 64) shares.load(shares.block + 64, unit);
      const int at = sequence - shares.block;
      const int64_t tokens = lane_value(shares.tokens, at), chunks = Dealt::chunks(tokens), base = lane_value(shares.before, at);
      if (unit >= base + chunks * shares.parts) {
        ++sequence;
        continue;
      }
      const int part = static_cast<int>((unit - base) / chunks);
      const int64_t seg = base + part * chunks;  // its first unit
      const int head = part / shares.head_parts, first_head = (part - head * shares.head_parts) * kHeads;
      const int64_t from = unit - seg, to = end - seg < chunks ? end - seg : chunks;
      bool bad = !__builtin_amdgcn_readlane(shares.whole, at);

      // The pages of the next 64 16-token parts, one a lane.
      const int32_t* table = c.table + sequence * c.table_stride;
      int pages = 0;
      const auto look_up = [&](int64_t next) {
        const int64_t first = next * TS + lane * 16;
        pages = 0;
        if (first < tokens) {
          pages = table[first >> c.page_log2];
          if (pages < 0 || pages >= c.pages) {
            bad = true;
            pages = 0;
          }
        }
      };
      look_up(from);
      // q of 16 heads as the second operand
      bf16x8 q[DP / 32];
      const int g = first_head + col;
      const uint16_t* qp = a.q.p + sequence * a.q.token + (head * a.group + (g < a.group ? g : 0)) * a.q.head;
#pragma unroll
      for (int j = 0; j < DP / 32; ++j) {
        // dims of operand j: as the keys' 16-byte pieces bring them
        const int d = E4M3 ? 64 * (j >> 1) + 16 * quarter + 8 * (j & 1) : 32 * j + 8 * quarter;
        u32x4 v = {0, 0, 0, 0};
        if (g < a.group && d < c.dim) v = *reinterpret_cast<const u32x4*>(qp + d);
        q[j] = __builtin_bit_cast(bf16x8, v);
      }
      arrived(pages);

      const auto issue = [&](int64_t next, int slot, int ahead) {
        const int64_t first = next * TS;
        const uint32_t to_stage = lds_at + slot * kStage;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // what was read here last
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          if (first + 16 * u >= tokens) break;
          const int page = __builtin_amdgcn_readlane(pages, ahead * kSub + u);
          const int64_t row0 = ((static_cast<int64_t>(page) * c.kv_heads + head) << c.page_log2) +
                               ((first + 16 * u) & ((1 << c.page_log2) - 1));
#pragma unroll
          for (int i = 0; i < 16 / kLoadRows; ++i) {
            const int row = i * kLoadRows + lane / kSlots, piece = (lane % kSlots) ^ swizzle(row);
            const uint32_t off = row * row_bytes + 16 * piece;
            const uint32_t to_lds = to_stage + (16 * u + i * kLoadRows) * kPitch;
            if (16 * piece < row_bytes) {
              load_to_lds(c.k + row0 * row_bytes, off, to_lds);
              load_to_lds(c.v + row0 * row_bytes, off, to_lds + kTile);
            }
          }
        }
        if constexpr (E4M3) {  // a stage's scales by one instruction: 4 tokens a lane, keys' and then values'
          const int u = (lane & 15) >> 2, page = __shfl(pages, ahead * kSub + u);
          const int64_t row = ((static_cast<int64_t>(page) * c.kv_heads + head) << c.page_log2) +
                              ((first + 16 * u) & ((1 << c.page_log2) - 1)) + 4 * (lane & 3);
          if (lane < 32 && u < kSub && first + 16 * u < tokens)
            load_dword_to_lds((lane < 16 ? c.k_scales : c.v_scales) + row, to_stage + 2 * kTile);
        }
      };

      issue(from, 0, 0);
#pragma unroll
      for (int j = 0; j < DP / 32; ++j) arrived(q[j]);
      float m, l, by = 1.0f;  // by: of the head's weights as operands, when the run is taken again
      f32x4 out[DP / 16];

      const auto compute = [&](int64_t stage, int slot, auto again) {
        const uint8_t* kt = lds + slot * kStage;
        const uint8_t* vt = kt + kTile;
        const int64_t left64 = tokens - stage * TS;
        const int left = left64 < TS ? static_cast<int>(left64) : TS;
#pragma unroll
        for (int u = 0; u < kSub; u += 2) {  // 32 tokens
          f32x4 s[2], vs[2];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            s[b] = (f32x4){0, 0, 0, 0};
            const uint8_t* row = kt + (16 * (u + b) + col) * kPitch;
            if constexpr (!E4M3) {
#pragma unroll
              for (int j = 0; j < DP / 32; ++j)
                s[b] = mfma16(*reinterpret_cast<const bf16x8*>(row + 16 * ((4 * j + quarter) ^ swizzle(col))), q[j], s[b]);
            } else {
#pragma unroll
              for (int j = 0; j < DP / 64; ++j) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(row + 16 * ((4 * j + quarter) ^ swizzle(col)));
                const u32x2 x0 = codes_to_bf16(w[0], 1.0f), x1 = codes_to_bf16(w[1], 1.0f);
                const u32x2 x2 = codes_to_bf16(w[2], 1.0f), x3 = codes_to_bf16(w[3], 1.0f);
                s[b] = mfma16(__builtin_bit_cast(bf16x8, (u32x4){x0[0], x0[1], x1[0], x1[1]}), q[2 * j], s[b]);
                s[b] = mfma16(__builtin_bit_cast(bf16x8, (u32x4){x2[0], x2[1], x3[0], x3[1]}), q[2 * j + 1], s[b]);
              }
              const uint32_t ks = *reinterpret_cast<const uint32_t*>(vt + kTile + 16 * (u + b) + 4 * quarter);
              const uint32_t ws = *reinterpret_cast<const uint32_t*>(vt + kTile + 64 + 16 * (u + b) + 4 * quarter);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                s[b][r] *= scale_value((ks >> (8 * r)) & 255);
                vs[b][r] = scale_value((ws >> (8 * r)) & 255);
              }
            }
          }
          const int here = left - 16 * u - 4 * quarter;  // tokens of this lane's part that exist
          if (left < TS) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (16 * b + r >= here) s[b][r] = -INFINITY;
          }
          const float top = quarter_max(fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                              fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))));
          const bool grows = top * sc > m * sc + 8.0f;  // as over packed sequences: weights reach 2^8
          if (__any(grows)) {
            const float next = grows ? top : m, alpha = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - next) * sc);
            m = next;
            l *= alpha;
#pragma unroll
            for (int t = 0; t < DP / 16; ++t)
#pragma unroll
              for (int r = 0; r < 4; ++r) out[t][r] *= alpha;
          }
          const float mc = m == -INFINITY ? 0.0f : m * sc;
          bf16x8 p;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float w = __builtin_amdgcn_exp2f(fmaf(s[b][r], sc, -mc));
              l += w;
              if constexpr (again) w *= by;
              p[4 * b + r] = static_cast<__bf16>(!E4M3 ? w : left < TS && 16 * b + r >= here ? 0.0f : w * vs[b][r]);
            }
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) {
            bf16x8 v = values(vt, u, t, lane);
            if (left < TS) {  // what lies behind the last token is no value
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (16 * (e >> 2) + (e & 3) >= here) v[e] = static_cast<__bf16>(0.0f);
            }
            out[t] = mfma16(v, p, out[t]);
          }
        }
      };

      constexpr int kAhead = 64 / kSub;  // stages of a look-up
      const auto pass = [&](auto again) {  // of stages from .. to - 1, of which the first one's loads are on their way
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) out[t] = (f32x4){0, 0, 0, 0};
        int slot = 0, ahead = 0;
        for (int64_t stage = from; stage < to; ++stage, slot ^= 1) {
          if (stage + 1 < to) {
            if (++ahead == kAhead) {
              ahead = 0;
              look_up(stage + 1);
              arrived(pages);
            }
            issue(stage + 1, slot ^ 1, ahead);
            if ((stage + 2) * TS <= tokens)
              asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
            else
              asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          }
          compute(stage, slot, again);
        }
      };
      pass(std::false_type{});
      const bool wrong = nonfinite(out);
      if (__any(wrong)) {
        if (quarter_sum(wrong ? 1.0f : 0.0f) != 0.0f) by = kSmaller;
        look_up(from);
        arrived(pages);
        issue(from, 0, 0);
        pass(std::true_type{});
      }

      if (from == 0 && lane == 0 && (by_segment || to != chunks))
        splits[by_segment ? sequence * shares.parts + part : worker] =
            Split{sequence, part, worker, to == chunks ? worker : shares.worker(seg + chunks - 1), shares.units, 0};
      l = quarter_sum(l);
      if (__any(bad)) l = NAN;
      if (g < a.group) {
        if (from == 0 && to == chunks) {
          const float inverse = l == 0.0f ? without_weights(m * sc) : 1.0f / (l * by);
          uint16_t* o = a.out + (static_cast<int64_t>(sequence) * c.kv_heads * a.group + head * a.group + g) * c.dim;
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) {
            const int d = 16 * t + 4 * quarter;
            if (d < c.dim)
              *reinterpret_cast<u32x2*>(o + d) = pack4(out[t][0] * inverse, out[t][1] * inverse, out[t][2] * inverse, out[t][3] * inverse);
          }
        } else {
          float* p = a.partial + static_cast<int64_t>(2 * worker + (from == 0 ? 1 : 0)) * kPartial;
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) *reinterpret_cast<f32x4*>(p + col * DP + 16 * t + 4 * quarter) = out[t];
          if (quarter == 0) {
            p[kHeads * DP + 2 * col] = m;
            p[kHeads * DP + 2 * col + 1] = by == 1.0f ? l : -l * by;  // the sign says by which the sums are
          }
        }
      }
      unit = seg + to;
    }
  }

  // Dims 16 t .. + 15 of 32 tokens from part u on, as a first operand whose
  // contraction is in the order of P's registers.
  __device__ static __forceinline__ bf16x8 values(const uint8_t* vt, int u, int t, int lane) {
    const int a = lane & 15, quarter = lane >> 4;
    if constexpr (!E4M3) {
      typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
      s16x4 v[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int row = 16 * (u + b) + 4 * quarter + (a >> 2), piece = 2 * t + ((a & 3) >> 1);
        v[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(vt + row * kPitch + 16 * (piece ^ swizzle(row)) + 8 * (a & 1)));
      }
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      // eight rows of 16 codes: lane a of 16 reads row a / 2, codes 8 (a % 2) .. + 7
      typedef int i32x2 __attribute__((vector_size(8)));
      typedef __attribute__((address_space(3))) i32x2* lds_i32x2;
      const int i = a >> 1, row = 16 * (u + (i >> 2)) + 4 * quarter + (i & 3);
      const auto w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2)(vt + row * kPitch + 16 * (t ^ swizzle(row)) + 8 * (a & 1)));
      const u32x2 lo = codes_to_bf16(static_cast<uint32_t>(w[0]), 1.0f), hi = codes_to_bf16(static_cast<uint32_t>(w[1]), 1.0f);
      return __builtin_bit_cast(bf16x8, (u32x4){lo[0], lo[1], hi[0], hi[1]});
    }
  }
};

template <class D>
__global__ __launch_bounds__(64) void decode_kernel(DecodeArgs a) {
  extern __shared__ __align__(1024) uint8_t lds[];
  D::run(a, lds);
}

// One head of a Split and LANES x 4 of its columns a workgroup: adds its parts where there
// are several.  Sequences without a token are written here too.  Takes 4 to 9 us, a
// launch and three loads that wait for each other; finding each head's parts from
// the lengths took 5 to 7 up to 64 sequences, 34 for 256 and 460 for 1,000.
template <class D, int LANES>
__global__ __launch_bounds__(256) void decode_join_kernel(DecodeArgs a) {
  constexpr int DP = D::DP, kGroups = 256 / LANES;  // parts at a time
  const CacheArgs& c = a.cache;
  const int heads = c.kv_heads * a.group, head_parts = (a.group + kHeads - 1) / kHeads, parts = c.kv_heads * head_parts;
  const bool by_segment = D::by_segment(a, parts);
  const Split split = D::splits(a)[blockIdx.x];
  const int hd = blockIdx.y;
  if (blockIdx.z == 0) {
    const int stride = by_segment ? c.sequences : D::kWorkers;
    for (int s = by_segment ? blockIdx.x / parts : blockIdx.x; s < c.sequences; s += stride) {
      bool whole;
      if (tokens_of(a, s, whole) != 0) continue;
      const uint32_t none = whole ? 0u : 0x7FC07FC0u;
      u32x2* o = reinterpret_cast<u32x2*>(a.out + static_cast<int64_t>(s) * heads * c.dim);
      const int row = c.dim / 4, all = heads * row;
      // a part's head, or every gridDim.y-th head
      if (by_segment) {
        const int part = blockIdx.x % parts, g = part % head_parts * kHeads + hd;
        if (g < a.group)
          for (int i = threadIdx.x; i < row; i += 256) o[(part / head_parts * a.group + g) * row + i] = (u32x2){none, none};
        return;
      }
      for (int i = hd * 256 + threadIdx.x; i < all; i += gridDim.y * 256) o[i] = (u32x2){none, none};
    }
  }
  if (by_segment) {
    bool unused;
    if (tokens_of(a, blockIdx.x / parts, unused) == 0) return;  // has no Split
  }
  if (split.last <= split.first) return;
  const int first = split.first, last = split.last, g = split.part % head_parts * kHeads + hd;
  if (split.last < 0 || g >= a.group) return;
  const int sequence = split.sequence, query_head = split.part / head_parts * a.group + g;
  const auto start = [&](int worker) { return split.units * worker / D::kWorkers; };
  const float sc = a.scale * 1.44269504088896340736f;
  const int d = 4 * (threadIdx.x % LANES + LANES * blockIdx.z), group = threadIdx.x / LANES;
  float top = -INFINITY, total = 0.0f;
  f32x4 sum = {0, 0, 0, 0};
  // Adds a part to another one, both with sums relative to their own maximum.
  const auto add = [&](float m, float l, f32x4 x) {
    const float next = fmaxf(top, m);
    const float old = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((top - next) * sc);
    const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - next) * sc);
    total = (total != total ? total : old * total) + (l != l ? l : by * l);
    sum = (old == 0.0f ? (f32x4){0, 0, 0, 0} : old * sum) + (by == 0.0f ? (f32x4){0, 0, 0, 0} : by * x);
    top = next;
  };
  constexpr int kAtOnce = 4;
  for (int w0 = first + group; w0 <= last; w0 += kAtOnce * kGroups) {
    float m[kAtOnce], l[kAtOnce];
    f32x4 x[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int w = w0 + i * kGroups;
      m[i] = -INFINITY;
      l[i] = 0.0f;
      x[i] = (f32x4){0, 0, 0, 0};
      // where there are fewer units than workers, some of these have none
      if (w > last || start(w) >= start(w + 1)) continue;
      const float* p = a.partial + static_cast<int64_t>(2 * w + (w == first ? 1 : 0)) * D::kPartial;
      m[i] = p[kHeads * DP + 2 * hd];
      l[i] = p[kHeads * DP + 2 * hd + 1];
      if (d < c.dim) x[i] = *reinterpret_cast<const f32x4*>(p + hd * DP + d);
      if (l[i] < 0.0f) x[i] = (f32x4){NAN, NAN, NAN, NAN};
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) add(m[i], l[i], x[i]);
  }
  __shared__ f32x4 sums[256];
  __shared__ float stats[256][2];
#pragma unroll
  for (int step = kGroups / 2; step > 0; step >>= 1) {
    if (group >= step && group < 2 * step) {
      sums[threadIdx.x] = sum;
      stats[threadIdx.x][0] = top;
      stats[threadIdx.x][1] = total;
    }
    __syncthreads();
    if (group < step) {
      const int other = threadIdx.x + step * LANES;
      add(stats[other][0], stats[other][1], sums[other]);
    }
  }
  if (group != 0 || d >= c.dim) return;
  if (nonfinite(sum)) {  // past FP32's range, a part with smaller weights, or no numbers: one part after the other
    top = -INFINITY;
    total = 0.0f;
    sum = (f32x4){0, 0, 0, 0};
    for (int w = first; w <= last; ++w) {
      if (start(w) >= start(w + 1)) continue;
      const float* p = a.partial + static_cast<int64_t>(2 * w + (w == first ? 1 : 0)) * D::kPartial;
      const float l = p[kHeads * DP + 2 * hd + 1], by = l < 0.0f ? 1.0f : kSmaller;
      add(p[kHeads * DP + 2 * hd], fabsf(l) * by, by * *reinterpret_cast<const f32x4*>(p + hd * DP + d));
    }
  }
  const float inverse = total == 0.0f ? without_weights(top * sc) : 1.0f / total;
  uint16_t* o = a.out + (static_cast<int64_t>(sequence) * heads + query_head) * c.dim + d;
  *reinterpret_cast<u32x2*>(o) = pack4(sum[0] * inverse, sum[1] * inverse, sum[2] * inverse, sum[3] * inverse);
}

template <class D>
hipError_t decode(const DecodeArgs& a, hipStream_t st) {
  decode_kernel<D><<<D::kWorkers, 64, D::kLds, st>>>(a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  const int most = a.group < kHeads ? a.group : kHeads, parts = a.cache.kv_heads * ((a.group + kHeads - 1) / kHeads);
  const int64_t segments = static_cast<int64_t>(a.cache.sequences) * parts, heads = a.cache.kv_heads * a.group;
  const uint32_t splits = static_cast<uint32_t>(segments < D::kWorkers ? segments : D::kWorkers);
  // A few heads may each have hundreds of parts: 16 columns a workgroup then.
  if (a.cache.sequences * heads <= 256)
    decode_join_kernel<D, 4><<<dim3(splits, most, D::DP / 16), 256, 0, st>>>(a);
  else
    decode_join_kernel<D, D::DP / 4><<<dim3(splits, most), 256, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

size_t decode_space(int dim, bool e4m3) {
  const auto of = [](auto d) { return decltype(d)::kSpace; };
  if (dim <= 64) return e4m3 ? of(Decode<64, true>{}) : of(Decode<64, false>{});
  if (dim <= 128) return e4m3 ? of(Decode<128, true>{}) : of(Decode<128, false>{});
  return e4m3 ? of(Decode<256, true>{}) : of(Decode<256, false>{});
}

hipError_t launch_decode(const DecodeArgs& a, hipStream_t st) {
  if (a.cache.e4m3) {
    if (a.cache.dim <= 64) return decode<Decode<64, true>>(a, st);
    if (a.cache.dim <= 128) return decode<Decode<128, true>>(a, st);
    return decode<Decode<256, true>>(a, st);
  }
  if (a.cache.dim <= 64) return decode<Decode<64, false>>(a, st);
  if (a.cache.dim <= 128) return decode<Decode<128, false>>(a, st);
  return decode<Decode<256, false>>(a, st);
}

}  // namespace glm53
