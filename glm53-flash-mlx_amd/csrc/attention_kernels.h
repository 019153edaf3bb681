// Attention within packed sequences, forward and backward.
//
//   S = scale q k^T over the keys a query sees, P = softmax(S), out = P v
//
// A row is one query of one head.  The `group` heads of a key head are rows
// of the same tile, token by token, so that a tile's keys and values serve all
// of them, and a key head's gradients are one contraction over its rows.
#pragma once

#include <type_traits>
#include <utility>

#include "attention.h"
#include "attention_tile.h"

namespace glm53 {

namespace {

// How a tile is multiplied: every place of it seen; some masked; or masked,
// with infinities and NaNs in masked places kept from the results.  The last is the price
// of a kernel's second pass, which follows where the first one's results are
// not all finite: they may be what 0 x NaN made of a masked place, or sums that
// passed FP32's range.
enum How { kPlain, kMasked, kCareful };
template <int N>
using Constant = std::integral_constant<int, N>;

// f(0), ..., f(N - 1) with constants: a loop that is unrolled whatever its length.
template <class F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) { (f(Constant<I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void each(F f) { each(f, std::make_integer_sequence<int, N>{}); }

// Keeps what is in front of it in front and what is behind it behind, when the
// compiler orders instructions: left alone it puts each LDS read directly
// before the product that waits for it.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// Around a run of products: its wavefront goes first on its SIMD, so that the
// other one there comes to its weights while this one multiplies (16,384 causal
// tokens, 8 / 1 heads of 128, when it was built: 505 us, without 560).
__device__ __forceinline__ void products(bool begin) {
  if (begin)
    __builtin_amdgcn_s_setprio(1);
  else
    __builtin_amdgcn_s_setprio(0);
}

constexpr float kLog2e = 1.44269504088896340736f;
// A row's maximum is kept until a new one is this many powers of two above it:
// the weights 2^(s - m) then reach 2^8, which changes no relative rounding, and
// few tiles after the first rescale their sums.  Sums of such weights times values
// may pass FP32's range where their mean does not: the second pass takes a row whose
// results were not finite with weights 2^-40 of these, whose sum is below 1 over 2^30
// keys.  Powers of two change no bit, but of values below 2^-86 beside such large ones.
constexpr float kSlack = 8.0f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Keys of the sequence that `seg` is of: first and how many.
__device__ __forceinline__ void sequence_keys(const AttentionArgs& a, const Divisor& group, const Segment& seg, int& first, int& count) {
  first = count = 0;
  if (seg.number < 0) return;
  if (a.key_offsets == nullptr) {  // the queries' own
    first = group.quotient(seg.first);
    count = group.quotient(seg.last - seg.first);
    return;
  }
  const int32_t* offsets = a.key_offsets;
  const int number = seg.number;
  const int most = static_cast<int>(a.keys);
  int lo = offsets[number], hi = offsets[number + 1];
  lo = lo < 0 ? 0 : lo > most ? most : lo;
  hi = hi < lo ? lo : hi > most ? most : hi;
  first = __builtin_amdgcn_readfirstlane(lo);
  count = __builtin_amdgcn_readfirstlane(hi - lo);
}

// Whether a causal pass over row tiles of `size` starts with those that see the most keys
// whatever their sequence, which pays for its search where sequences are long (8,192
// tokens in two, 16 heads of 64: 84 us for 94; in eleven, 32 / 8 heads of 128: 105 for 99).
__device__ __forceinline__ bool longest_first(const AttentionArgs& a, int size) {
  return a.causal && a.tokens * a.group >= int64_t{32} * size * a.sequences;
}

// Keys that the query of a row sees: a prefix of its sequence's.
struct Prefix {
  const Divisor& group;
  int first, shift, keys;
  bool causal;
  __device__ __forceinline__ Prefix(const AttentionArgs& a, const Divisor& group, const Segment& seg, int keys)
      : group(group), first(seg.first), shift(keys - group.quotient(seg.last - seg.first)), keys(keys), causal(a.causal) {}
  __device__ __forceinline__ int operator()(int row) const {
    if (!causal) return keys;
    const int n = group.quotient(row - first) + shift + 1;
    return n < 0 ? 0 : n > keys ? keys : n;
  }
};

// A row of memory as the operands that a lane of it holds, zeros from `dim` on, and
// a result's column as a row of memory.
template <int DP>
__device__ __forceinline__ void load_operand(bf16x8 (&x)[DP / 16], const uint16_t* p, int dim, int h) {
#pragma unroll
  for (int j = 0; j < DP / 16; ++j) {
    u32x4 v = {0, 0, 0, 0};
    if (16 * j + 8 * h < dim) v = *reinterpret_cast<const u32x4*>(p + 16 * j + 8 * h);
    x[j] = __builtin_bit_cast(bf16x8, v);
  }
}
template <int DP>
__device__ __forceinline__ void store_operand(uint16_t* p, const f32x16 (&x)[DP / 32], float by, int dim, int h) {
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int d = 32 * t + result_row(e, h);
      if (d < dim)
        *reinterpret_cast<u32x2*>(p + d) = pack4(x[t][e] * by, x[t][e + 1] * by, x[t][e + 2] * by, x[t][e + 3] * by);
    }
}

template <int DP>
__device__ __forceinline__ void store_sums(float* p, const f32x16 (&x)[DP / 32], int dim, int h) {
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int d = 32 * t + result_row(e, h);
      if (d < dim) *reinterpret_cast<f32x4*>(p + d) = (f32x4){x[t][e], x[t][e + 1], x[t][e + 2], x[t][e + 3]};
    }
}
__device__ __forceinline__ float* sums_of(const AttentionArgs& a, int gradient, int split) {
  return a.sums + (static_cast<int64_t>(gradient) * a.splits + split) * a.keys * a.kv_heads * a.dim;
}

template <int T>
__device__ __forceinline__ bool nonfinite(const f32x16 (&x)[T]) {
  float sum = 0.0f;
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) sum = fmaf(x[t][e], 0.0f, sum);
  return sum != 0.0f;
}

// Whether any of the workgroup's threads says so, asked when all are through with
// LDS, whose first words it takes.
template <int W>
__device__ __forceinline__ bool voted(bool mine, uint8_t* lds, int wave) {
  int* votes = reinterpret_cast<int*>(lds);
  const int own = __any(mine);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) votes[wave] = own;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) all |= votes[w];
  if (!__builtin_amdgcn_readfirstlane(all)) return false;
  __syncthreads();
  return true;
}

// Tile numbers of `rows` rows in `sequences` sequences (see find_segment).
int64_t tile_numbers(int64_t rows, bool packed, int sequences, int size) {
  return packed ? rows / size + sequences + 2 : (rows + size - 1) / size;
}

// ------------------------------------------------------------- forward ---
//
// W wavefronts of 32 rows; a tile of 64 keys is multiplied while the next one is
// loaded.  Scores are computed as S^T (keys the result's rows), so a lane holds
// 32 of its row's 64 scores, a row's maximum and sum are within a lane and its
// counterpart 32 lanes away, and the weights go into the second product (out^T
// = v^T P^T) from the registers they are in.  One pass over the keys: sums
// relative to a running maximum, in FP32; the weights are rounded to bf16 as the
// matrix instruction takes them, the result once.
//
// Bound by a SIMD's two wavefronts, which take turns at its matrix unit and its
// vector unit: a tile of 128 columns is 2,048 clocks of products for both, and the
// 32 exponentials, maxima, sums and conversions of each lane are about as many.
// 4,096 + 4,096 tokens, 16 / 4 heads of 128, all seen: 242 us, 1,138 TFLOP/s, the
// matrix unit busy half of the time (228 us without the softmax's instructions, when all took
// 254); 64 rows a wavefront, which halve the LDS reads, leave one wavefront a SIMD and
// were slower.  16,384 causal tokens, 8 / 1 heads: 477 us, 1,153 TFLOP/s.

template <int DP_, bool EXACT>
struct Forward {
  static constexpr int DP = DP_, W = 4;
  static constexpr int kRows = 32 * W, kThreads = 64 * W, kKeys = 64, T = DP / 32;
  using Tile = HeadTile<DP, kKeys, W>;
  static constexpr int kLds = 4 * Tile::kBytes;  // two stages of keys and values

  static __device__ __forceinline__ void run(const AttentionArgs& a, const Divisor& group, int tiles, uint8_t* lds) {
    const int dim = EXACT ? DP : a.dim;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.kv_heads, number = blockIdx.x / a.kv_heads;
    const Segment seg = find_segment(a.offsets, a.sequences, a.tokens, a.group, kRows, number, tiles,
                                     longest_first(a, kRows) ? kLastFirst : kReversed);
    const int row0 = seg.first + seg.tile * kRows;
    if (seg.tile < 0 || row0 >= seg.last) return;
    int key0, keys;
    sequence_keys(a, group, seg, key0, keys);
    const Prefix prefix(a, group, seg, keys);
    const int last_row = row0 + kRows < seg.last ? row0 + kRows - 1 : seg.last - 1;
    const int steps = (__builtin_amdgcn_readfirstlane(prefix(last_row)) + kKeys - 1) / kKeys;

    const int h = lane >> 5;
    if (dim < DP) {
#pragma unroll
      for (int s = 0; s < 4; ++s) Tile::clear(lds + s * Tile::kBytes, dim, kThreads);
    }
    const uint16_t* kp = a.k.p + key0 * a.k.token + head * a.k.head;
    const uint16_t* vp = a.v.p + key0 * a.v.token + head * a.v.head;
    const uint32_t lds_at = lds_address(lds);
    const auto issue = [&](int step) {
      const uint32_t to = lds_at + (step & 1) * 2 * Tile::kBytes;
      const int64_t first = static_cast<int64_t>(step) * kKeys;
      const int left = keys - step * kKeys;
      Tile::load(kp + first * a.k.token, static_cast<uint32_t>(2 * a.k.token), left, dim, wave, lane, to);
      Tile::load(vp + first * a.v.token, static_cast<uint32_t>(2 * a.v.token), left, dim, wave, lane, to + Tile::kBytes);
    };
    if (steps > 0) issue(0);

    const int row = row0 + 32 * wave + (lane & 31);
    const int r = row < seg.last ? row : seg.last - 1;  // rows past the last repeat it
    const int token = group.quotient(r), query_head = head * a.group + r - token * a.group;
    const int lim = prefix(r);
    bf16x8 q[DP / 16];
    load_operand<DP>(q, a.q.p + token * a.q.token + query_head * a.q.head, dim, h);
    const typename Tile::Places at(lds_at, lane);  // while these are on their way
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) arrived(q[j]);
    const int all_see = __builtin_amdgcn_readfirstlane(lim), some_see = __builtin_amdgcn_readlane(lim, 31);

    const float c = a.scale * kLog2e;
    f32x16 out[T];
    // whole tiles two at a time: their places in LDS are constants then
    const int whole = all_see / kKeys & ~1;
    float m, l;  // m in units of scores; l: this lane's part
    float by = 1.0f;  // of the row's weights as operands, in the second pass
    uint32_t dirty = 0;
    // `how`: kPlain, kMasked, or kCareful (see finite_part), which takes whole tiles too
    const auto compute = [&](int step, auto stage, auto how) {
      constexpr int kHow = decltype(how)::value;
      const int kt = stage * 2 * Tile::kBytes, vt = kt + Tile::kBytes;
      f32x16 s[2];
      // groups of operands: the keys' in 32 keys and 64 columns, the values' in 16 keys
      constexpr int kGroups = DP / 64, kMost = T > 4 ? T : 4;
      bf16x8 f[3][kMost];
      const auto read = [&](int n) {
        bf16x8 (&x)[kMost] = f[n % 3];
        if (n < 2 * kGroups) {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = at.along(kt, n / kGroups, 4 * (n % kGroups) + j);
        } else if (n < 2 * kGroups + 4) {
#pragma unroll
          for (int t = 0; t < T; ++t) x[t] = at.across(vt, n - 2 * kGroups, t);
        }
      };
      // the second pass reads none ahead: its registers, the most of both, would put the first one's into
      // memory (4,096 causal tokens, 16 / 4 heads of 256: 207 us, with two ahead 230; of 200: 233 and 257)
      constexpr int kAhead = kHow == kCareful ? 0 : 2;
#pragma unroll
      for (int n = 0; n < kAhead; ++n) read(n);
      products(true);
#pragma unroll
      for (int n = 0; n < 2 * kGroups; ++n) {
        fence();
        read(n + kAhead);
        f32x16& x = s[n / kGroups];
#pragma unroll
        for (int j = 0; j < 4; ++j) x = mfma32(f[n % 3][j], q[4 * (n % kGroups) + j], n % kGroups + j == 0 ? zero16() : x);
      }
      fence();
      products(false);
      if constexpr (kHow != kPlain) {
        const int left = lim - step * kKeys - 4 * h;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (32 * kb + result_row(e, 0) >= left) s[kb][e] = -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[0][e]);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[1][e]);
      top = both_max(top);
      const bool grows = top * c > m * c + kSlack;
      if (__any(grows)) {
        const float next = grows ? top : m;  // a row's bits do not depend on its neighbours in the wavefront
        const float alpha = next == -INFINITY ? 1.0f : exp2_fast((m - next) * c);
        m = next;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) out[t][e] *= alpha;
      }
      const float mc = m == -INFINITY ? 0.0f : m * c;
      bf16x8 next;
      const auto weigh = [&](int i) {  // 8 of a lane's scores
        f32x16& x = s[i >> 1];
        float sum = 0.0f;
#pragma unroll
        for (int e = 8 * (i & 1); e < 8 * (i & 1) + 8; ++e) {
          x[e] = exp2_fast(fmaf(x[e], c, -mc));
          sum += x[e];
          if constexpr (kHow == kCareful) x[e] *= by;
        }
        l += sum;
        next = operand8(x, i & 1);
      };
      weigh(0);
      products(true);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fence();
        const int n = 2 * kGroups + i;
        read(n + kAhead);
        const bf16x8 p = next;
#pragma unroll
        for (int t = 0; t < T; ++t) {
          if constexpr (kHow == kCareful) f[n % 3][t] = finite_part(f[n % 3][t], dirty, step < whole ? 0 : kSigns);
          out[t] = mfma32(f[n % 3][t], p, out[t]);
        }
        if (i < 3) weigh(i + 1);
      }
      fence();
      products(false);
    };

    const auto pass = [&](auto how) {
      m = -INFINITY;
      l = 0.0f;
#pragma unroll
      for (int t = 0; t < T; ++t) out[t] = zero16();
      int step = 0;
      for (; decltype(how)::value != kCareful && step < whole; step += 2) {
        loads_done();
        issue(step + 1);
        compute(step, Constant<0>{}, Constant<kPlain>{});
        loads_done();
        if (step + 2 < steps) issue(step + 2);
        compute(step + 1, Constant<1>{}, Constant<kPlain>{});
      }
      for (; step < steps; ++step) {
        loads_done();
        if (step + 1 < steps) issue(step + 1);
        if (step * kKeys < some_see) compute(step, step & 1, how);
      }
    };
    pass(Constant<kMasked>{});
    const bool wrong = nonfinite(out);
    if (voted<W>(wrong, lds, wave)) {
      if (both_sum(wrong ? 1.0f : 0.0f) != 0.0f) by = 0x1p-40f;
      issue(0);
      pass(Constant<kCareful>{});
      if (__any(dirty != 0))
        add_nonfinite<DP>(out, whole * kKeys, some_see, dim, h, [&](int key) { return vp + key * a.v.token; },
                          [&](int key) { return key < lim; });
    }

    // no key seen; or scores that are no FP32 numbers once scaled, which leave no weights: NaN
    const float total = both_sum(l);
    if (row >= seg.last) return;
    const float top = m * c, none = top == INFINITY ? NAN : 0.0f, inverse = total == 0.0f ? none : 1.0f / (total * by);
    const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
    store_operand<DP>(a.out + (token * heads + query_head) * dim, out, inverse, dim, h);
    if (a.lse != nullptr && h == 0)
      a.lse[static_cast<int64_t>(head) * a.tokens * a.group + row] = total == 0.0f ? none : top + __builtin_amdgcn_logf(total);
  }
};

template <class F>
__global__ __launch_bounds__(F::kThreads, F::DP == 256 ? 1 : 2) void attention_kernel(AttentionArgs a, Divisor group, int tiles) {
  extern __shared__ __align__(1024) uint8_t lds[];
  F::run(a, group, tiles, lds);
}

// ------------------------------------------------------------ backward ---
//
//   P = 2^(S log2 e - lse), dP = d_out v^T, dS = P (dP - delta), delta = sum(d_out out)
//   d_q = scale dS k,  d_k = scale dS^T q,  d_v = P^T d_out
//
// Two kernels, each with one side of the scores for its own and a loop over the other:
// no sum is shared, so every gradient is added in a fixed order, for seven
// products instead of five (8,192 tokens in three sequences, 32 / 8 heads of 128:
// 357 us and 420 us of all gradients' 777, 800 TFLOP/s of the products made).
//
// delta from the rounded `out` is off by as much as `out` is, and puts that into
// every dS of its row.  The rows' sums of dS, which are 0, say by how much:
// the first kernel adds them to delta for the second one, and carries dS in two
// bf16 parts, so that both gradients are off by one operand's rounding at most
// (relative error 0.0024 instead of 0.0026 to 0.0029).

// d_q: a lane's row as in the forward pass, a tile of 64 keys at a time.  Bound as
// that is, by four runs of products for its two.
template <int DP_, bool EXACT, bool DQ>
struct QueryGradient {
  static constexpr int DP = DP_, W = 4;
  static constexpr int kRows = 32 * W, kThreads = 64 * W, kKeys = 64, T = DP / 32;
  static constexpr int kAhead = DP >= 128 ? 1 : 2;  // the registers leave no more
  // Rows of up to 256 keys, whose `out` is no mean of many and whose delta is off by more,
  // take their sums of dS in a pass of their own first (d_q of 30 sequences of 8 to 100
  // tokens off by 0.0023 instead of 0.0029).
  static constexpr int kFewSteps = 4;
  using Tile = HeadTile<DP, kKeys, W>;
  static constexpr int kLds = 4 * Tile::kBytes;

  static __device__ __forceinline__ void run(const AttentionArgs& a, const Divisor& group, int tiles, uint8_t* lds) {
    const int dim = EXACT ? DP : a.dim;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.kv_heads, number = blockIdx.x / a.kv_heads;
    const Segment seg = find_segment(a.offsets, a.sequences, a.tokens, a.group, kRows, number, tiles,
                                     longest_first(a, kRows) ? kLastFirst : kReversed);
    const int row0 = seg.first + seg.tile * kRows;
    if (seg.tile < 0 || row0 >= seg.last) return;
    int key0, keys;
    sequence_keys(a, group, seg, key0, keys);
    const Prefix prefix(a, group, seg, keys);
    const int last_row = row0 + kRows < seg.last ? row0 + kRows - 1 : seg.last - 1;
    const int steps = (__builtin_amdgcn_readfirstlane(prefix(last_row)) + kKeys - 1) / kKeys;

    const int h = lane >> 5, row = row0 + 32 * wave + (lane & 31);
    const int r = row < seg.last ? row : seg.last - 1, token = group.quotient(r), query_head = head * a.group + r - token * a.group;
    const int lim = prefix(r);
    if (dim < DP) {
#pragma unroll
      for (int s = 0; s < 4; ++s) Tile::clear(lds + s * Tile::kBytes, dim, kThreads);
    }
    const uint16_t* kp = a.k.p + key0 * a.k.token + head * a.k.head;
    const uint16_t* vp = a.v.p + key0 * a.v.token + head * a.v.head;
    const uint32_t lds_at = lds_address(lds);
    const auto issue = [&](int step) {
      const uint32_t at = lds_at + (step & 1) * 2 * Tile::kBytes;
      const int64_t first = static_cast<int64_t>(step) * kKeys;
      const int left = keys - step * kKeys;
      Tile::load(kp + first * a.k.token, static_cast<uint32_t>(2 * a.k.token), left, dim, wave, lane, at);
      Tile::load(vp + first * a.v.token, static_cast<uint32_t>(2 * a.v.token), left, dim, wave, lane, at + Tile::kBytes);
    };

    if (steps > 0) issue(0);
    bf16x8 q[DP / 16], d_out[DP / 16];
    const uint16_t* qp = a.q.p + token * a.q.token + query_head * a.q.head;
    const uint16_t* dp = a.d_out.p + token * a.d_out.token + query_head * a.d_out.head;
    load_operand<DP>(q, qp, dim, h);
    load_operand<DP>(d_out, dp, dim, h);
    const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
    const int64_t own = (token * heads + query_head) * dim, stat = static_cast<int64_t>(head) * a.tokens * a.group + r;
    float lse = a.lse[stat], delta = 0.0f;
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      if (16 * j + 8 * h >= dim) continue;
      const bf16x8 o = *reinterpret_cast<const bf16x8*>(a.out + own + 16 * j + 8 * h);
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf(static_cast<float>(o[e]), static_cast<float>(d_out[j][e]), delta);
    }
    delta = both_sum(delta);
    arrived(lse);
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      arrived(q[j]);
      arrived(d_out[j]);
    }
    const int all_see = __builtin_amdgcn_readfirstlane(lim), some_see = __builtin_amdgcn_readlane(lim, 31);

    const typename Tile::Places at(lds_at, lane);
    const float c = a.scale * kLog2e;
    float sum;  // of dS
    f32x16 d_q[T];
    // `results`: d_q's products too, not the sums of dS alone
    const auto compute = [&](int step, auto stage, auto how, auto results) {
      constexpr int kHow = decltype(how)::value;
      constexpr bool kResults = decltype(results)::value;
      const int kt = stage * 2 * Tile::kBytes, vt = kt + Tile::kBytes;
      // groups of operands, read ahead of the products that take them: of 32 keys those of
      // scores, 16 columns and two operands at a time, then those of 16 keys, 32 columns each
      constexpr int kOf = DP == 256 ? 4 : 2, kScores = DP / 8 / kOf, kAcross = T / kOf;
      constexpr int kPart = kScores + (kResults ? 2 * kAcross : 0), kAll = 2 * kPart;
      bf16x8 f[kAhead + 1][kOf];
      const auto read = [&](int n) {
        if (n >= kAll) return;
        bf16x8 (&x)[kOf] = f[n % (kAhead + 1)];
        const int kb = n / kPart, g = n % kPart, turn = g - kScores;
#pragma unroll
        for (int i = 0; i < kOf; ++i) {
          if (g >= kScores)
            x[i] = at.across(kt, 2 * kb + turn / kAcross, kOf * (turn % kAcross) + i);
          else
            x[i] = at.along(i & 1 ? vt : kt, kb, kOf / 2 * g + i / 2);
        }
      };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) read(n);
      f32x16 s, p;
      bf16x8 ds, low;
      products(true);
      each<kAll>([&](auto number) {
        constexpr int n = decltype(number)::value, kb = n / kPart, g = n % kPart, turn = g - kScores;
        fence();
        read(n + kAhead);
        bf16x8 (&x)[kOf] = f[n % (kAhead + 1)];
        if (g == 0) {
          s = zero16();
#pragma unroll
          for (int e = 0; e < 16; ++e) p[e] = -delta;
        }
        if constexpr (g < kScores) {
#pragma unroll
          for (int i = 0; i < kOf; i += 2) {
            s = mfma32(x[i], q[(kOf * g + i) / 2], s);
            p = mfma32(x[i + 1], d_out[(kOf * g + i) / 2], p);
          }
        } else {
          if (turn % kAcross == 0) {
            ds = operand8(s, turn / kAcross);
            low = low_operand8(s, turn / kAcross, ds);
          }
#pragma unroll
          for (int i = 0; i < kOf; ++i) {
            // a key that holds an infinity or NaN gives them to the dS of the rows that see it
            uint32_t unused = 0;
            if constexpr (kHow == kCareful) x[i] = finite_part(x[i], unused);
            f32x16& sum_q = d_q[kOf * (turn % kAcross) + i];
            sum_q = mfma32(x[i], ds, sum_q);
            sum_q = mfma32(x[i], low, sum_q);
          }
        }
        if constexpr (g == kScores - 1) {
          fence();
          products(false);
          const int left = lim - step * kKeys - 32 * kb - 4 * h;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
#pragma clang fp contract(off)  // the same sum whether or not dS is needed for itself
            s[e] = exp2_fast(fmaf(s[e], c, -lse)) * p[e];
            if (kHow != kPlain && result_row(e, 0) >= left) s[e] = 0.0f;
            sum += s[e];
          }
          products(true);
        }
      });
      fence();
      products(false);
    };
    const int whole = all_see / kKeys & ~1;
    const auto masked = [&](int step, auto how, auto results) {
      loads_done();
      if (step + 1 < steps) issue(step + 1);
      if (step * kKeys < some_see) compute(step, step & 1, how, results);
    };
    const auto pass = [&](auto how) {
      sum = 0.0f;
#pragma unroll
      for (int t = 0; t < T; ++t) d_q[t] = zero16();
      int step = 0;
      for (; step < whole; step += 2) {
        loads_done();
        issue(step + 1);
        compute(step, Constant<0>{}, Constant<kPlain>{}, Constant<DQ>{});
        loads_done();
        if (step + 2 < steps) issue(step + 2);
        compute(step + 1, Constant<1>{}, Constant<kPlain>{}, Constant<DQ>{});
      }
      for (; step < steps; ++step) masked(step, how, Constant<DQ>{});
    };
    const bool few = DQ && steps > 0 && steps <= kFewSteps;
    if (few) {
      sum = 0.0f;
      for (int step = 0; step < steps; ++step) masked(step, Constant<kMasked>{}, Constant<false>{});
      delta += both_sum(sum);
      __syncthreads();
      issue(0);
    }
    pass(Constant<kMasked>{});
    if constexpr (DQ) {
      if (voted<W>(nonfinite(d_q), lds, wave)) {
        issue(0);
        pass(Constant<kCareful>{});
      }
    }
    sum = few ? 0.0f : both_sum(sum);  // the joint call's starts are those of d_k's alone
    if (row >= seg.last) return;
    if (h == 0) {  // where the second kernel's products start
      a.starts[stat] = lse * (-1.0f / c);
      a.starts[stat + heads * a.tokens] = -(delta + sum);
    }
    if constexpr (DQ) store_operand<DP>(a.d_q + own, d_q, a.scale, dim, h);
  }
};

// d_k and d_v: a lane's key and a tile of rows at a time.  Scores are computed
// with rows the result's rows, so that P and dS are the second operands of
// d_v^T += d_out^T P and d_k^T += q^T dS as they are.  A wavefront has 32 keys
// and all of a tile's rows (RW = 1), or two wavefronts share 32 keys, each with half
// of a tile's rows, and add up at the end (RW = 2): a workgroup has 64 keys then and
// half as many turns, so that the first keys of a causal sequence, which all rows
// see, do not outlast the rest (wide_key_tiles has both sides).  With few keys and heads
// the turns of a tile are split over workgroups, whose FP32 sums key_gradient_join_kernel
// adds in their order (attention_row_splits).  Bound by
// its one wavefront a SIMD, which has the gradients' sums in 128 registers of a lane
// and no other one to multiply beside its weights, and by LDS: loading the
// tiles costs 18% of it.
template <int DP_, bool EXACT, int NB_, int RW_, bool DK, bool DV>
struct KeyGradient {
  static constexpr int DP = DP_, NB = NB_, RW = RW_;  // NB blocks of 32 rows a wavefront and turn, RW wavefronts' rows a tile
  static constexpr int W = 4, KW = W / RW, kKeys = 32 * KW, kThreads = 64 * W, RT = RW * NB * 32, T = DP / 32;
  using Tile = HeadTile<DP, RT, W>;
  static constexpr int kStats = 4 * 64 * ((RT + 63) / 64);      // bytes of lse, and of delta
  static constexpr int kStage = 2 * Tile::kBytes + 2 * kStats;  // q, d_out, lse, delta
  static constexpr int kSums = RW == 2 ? (DK + DV) * T / 2 * 4096 : 0;  // of one wavefront, exchanged at the end
  static constexpr int kLds = 2 * kStage > 4 * kSums ? 2 * kStage : 4 * kSums;

  static __device__ __forceinline__ void run(const AttentionArgs& a, const Divisor& group, int tiles, uint8_t* lds) {
    const int dim = EXACT ? DP : a.dim;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = wave / KW;  // whose rows of a tile
    const int head = blockIdx.x % a.kv_heads, split = blockIdx.x / a.kv_heads % a.splits, number = blockIdx.x / a.kv_heads / a.splits;
    const Segment seg = find_segment(a.key_offsets != nullptr ? a.key_offsets : a.offsets, a.sequences, a.keys, 1, kKeys, number,
                                     tiles, a.causal ? kFirstFirst : kInOrder);
    const int key0 = seg.first + seg.tile * kKeys;
    if (seg.tile < 0 || key0 >= seg.last) return;
    // the sequence's rows
    int first_row = 0, last_row = 0;
    if (seg.number >= 0) {
      if (a.key_offsets == nullptr) {  // the keys' own
        first_row = seg.first * a.group;
        last_row = seg.last * a.group;
      } else {
        const int most = static_cast<int>(a.tokens);
        int lo = a.offsets[seg.number], hi = a.offsets[seg.number + 1];
        lo = lo < 0 ? 0 : lo > most ? most : lo;
        hi = hi < lo ? lo : hi > most ? most : hi;
        first_row = __builtin_amdgcn_readfirstlane(lo) * a.group;
        last_row = __builtin_amdgcn_readfirstlane(hi) * a.group;
      }
    }
    const int shift = seg.last - seg.first - group.quotient(last_row - first_row);
    // the first row that sees a key
    const auto sees = [&](int key) {
      const int n = a.causal ? key - seg.first - shift : 0;
      return n <= 0 ? first_row : first_row + n * a.group;
    };
    const int h = lane >> 5, key = key0 + 32 * (wave % KW) + (lane & 31), k = key < seg.last ? key : seg.last - 1;
    const int from = sees(k), from_all = __builtin_amdgcn_readlane(from, 31), from_some = __builtin_amdgcn_readfirstlane(from);
    int start = __builtin_amdgcn_readfirstlane(sees(key0));
    int steps = start < last_row ? (last_row - start + RT - 1) / RT : 0;
    if (a.splits > 1) {  // this workgroup's share of the turns, in as many parts as have kLeastTurns
      const int64_t all = steps;
      const int parts = steps >= 2 * kLeastTurns ? (steps / kLeastTurns < a.splits ? steps / kLeastTurns : a.splits) : 1;
      const int first = static_cast<int>(split < parts ? all * split / parts : all);
      const int end = static_cast<int>(split < parts ? all * (split + 1) / parts : all);
      if (end < all) last_row = start + end * RT;
      start += first * RT;
      steps = end - first;
    }

    if (dim < DP) {
#pragma unroll
      for (int s = 0; s < 4; ++s) Tile::clear(lds + (s >> 1) * kStage + (s & 1) * Tile::kBytes, dim, kThreads);
    }
    const uint32_t lds_at = lds_address(lds);
    const int64_t stat = static_cast<int64_t>(head) * a.tokens * a.group, heads = static_cast<int64_t>(a.kv_heads) * a.group;
    const float* lse = (DK ? a.starts : a.lse) + stat;
    const float* delta = a.starts + heads * a.tokens + stat;
    const bool even = 16 % a.group == 0;  // rows 16 apart are whole tokens apart
    const int own = Tile::row_of(wave, lane), own_token = group.quotient(own), own_head = own - own_token * a.group;
    const uint32_t q_off = static_cast<uint32_t>(2 * (own_token * a.q.token + own_head * a.q.head)) + Tile::piece_of(wave, lane);
    const uint32_t o_off = static_cast<uint32_t>(2 * (own_token * a.d_out.token + own_head * a.d_out.head)) + Tile::piece_of(wave, lane);
    const auto issue = [&](int step) {
      const uint32_t at = lds_at + (step & 1) * kStage;
      const int row0 = start + step * RT, left = last_row - row0;
      const int token0 = group.quotient(row0);
      const uint16_t* qp = a.q.p + token0 * a.q.token + head * a.group * a.q.head;
      const uint16_t* op = a.d_out.p + token0 * a.d_out.token + head * a.group * a.d_out.head;
      // row0 may lie inside token0 where a group does not divide RT, so that every row's token and
      // head are found; load_even needs whole tokens a tile, which `even` says
      const auto offset = [&](const Rows16& x) {
        return [&](int n) {
          const int token = group.quotient(row0 + n), g = row0 + n - token * a.group;
          return static_cast<uint32_t>(token - token0) * static_cast<uint32_t>(2 * x.token) + static_cast<uint32_t>(g) * static_cast<uint32_t>(2 * x.head);
        };
      };
      bool done = false;
      if constexpr (Tile::kEven) {
        if (even && left >= RT) {
          const uint64_t apart = 16 / a.group;
          Tile::load_even(qp, q_off, 2 * apart * a.q.token, dim, wave, lane, at);
          Tile::load_even(op, o_off, 2 * apart * a.d_out.token, dim, wave, lane, at + Tile::kBytes);
          done = true;
        }
      }
      if (!done) {
        Tile::load(qp, offset(a.q), left, dim, wave, lane, at);
        Tile::load(op, offset(a.d_out), left, dim, wave, lane, at + Tile::kBytes);
      }
      if (wave < kStats / 256) {
        const int n = 64 * wave + lane;
        const uint32_t off = 4 * (n < left ? n : left - 1), to = at + 2 * Tile::kBytes + 256 * wave;
        load_to_lds<4>(lse + row0, off, to);
        if (DK) load_to_lds<4>(delta + row0, off, to + kStats);
      }
    };

    if (steps > 0) issue(0);
    bf16x8 kf[DP / 16], vf[DP / 16];
    const uint16_t* kp = a.k.p + k * a.k.token + head * a.k.head;
    const uint16_t* vp = a.v.p + k * a.v.token + head * a.v.head;
    load_operand<DP>(kf, kp, dim, h);
    if (DK) load_operand<DP>(vf, vp, dim, h);
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      arrived(kf[j]);
      if (DK) arrived(vf[j]);
    }
    const typename Tile::Places at(lds_at + half * (NB * 32 * Tile::kPitch), lane);
    const float c = a.scale * kLog2e, start_scale = -1.0f / c;
    f32x16 d_k[T], d_v[T];
    uint32_t dirty = 0;
    const auto compute = [&](int step, auto stage, auto how) {
      constexpr int kHow = decltype(how)::value;
      const int qt = stage * kStage, ot = qt + Tile::kBytes;
      const float* stats = reinterpret_cast<const float*>(lds + stage * kStage + 2 * Tile::kBytes) + half * (NB * 32);
      f32x16 s[NB], p[NB];
      const auto begin = [&](int b) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const f32x4 l = *reinterpret_cast<const f32x4*>(stats + 32 * b + result_row(e, h));
          const f32x4 d = *reinterpret_cast<const f32x4*>(stats + (DK ? kStats / 4 : 0) + 32 * b + result_row(e, h));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[b][e + i] = DK ? l[i] : l[i] * start_scale;  // as the first kernel has it
            p[b][e + i] = d[i];
          }
        }
      };
      // w = P, p = dS of results first .. first + 7 of a block
      const auto weigh = [&](int b, int first) {
#pragma unroll
        for (int e = first; e < first + 8; ++e) {
          const float w = exp2_fast(s[b][e] * c);
          s[b][e] = w;
          p[b][e] *= w;
          if constexpr (kHow != kPlain) {
            const int row = start + step * RT + half * (NB * 32) + 32 * b + 4 * h + result_row(e, 0);
            if (row < from || row >= last_row) s[b][e] = p[b][e] = 0.0f;
          }
        }
      };
      // Operands are read two groups ahead of the products that take them (a block's scores
      // over 64 columns, the sums over 16 rows), and the weights of a block are made beside
      // the products of the other one.
      constexpr int kGroups = DP / 64, kScores = NB * kGroups, kAll = kScores + 2 * NB;
      constexpr int kAhead = 2, kOf = DK + DV, kMost = kOf * T > 8 ? kOf * T : 8;
      bf16x8 f[kAhead + 1][kMost];
      const auto read = [&](int n) {
        if (n >= kAll) return;
        bf16x8 (&x)[kMost] = f[n % (kAhead + 1)];
        if (n < kScores) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[2 * j] = at.along(qt, n / kGroups, 4 * (n % kGroups) + j);
            if (DK) x[2 * j + 1] = at.along(ot, n / kGroups, 4 * (n % kGroups) + j);
          }
        } else {
#pragma unroll
          for (int t = 0; t < T; ++t) {
            if (DV) x[kOf * t] = at.across(ot, n - kScores, t);
            if (DK) x[kOf * t + DV] = at.across(qt, n - kScores, t);
          }
        }
      };
#pragma unroll
      for (int b = 0; b < NB; ++b) begin(b);
#pragma unroll
      for (int n = 0; n < kAhead; ++n) read(n);
      each<kAll>([&](auto number) {
        constexpr int n = decltype(number)::value;
        if constexpr (DP > 64) fence();
        read(n + kAhead);
        bf16x8 (&x)[kMost] = f[n % (kAhead + 1)];
        if constexpr (n < kScores) {
          constexpr int b = n / kGroups;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[b] = mfma32(x[2 * j], kf[4 * (n % kGroups) + j], s[b]);
            if (DK) p[b] = mfma32(x[2 * j + 1], vf[4 * (n % kGroups) + j], p[b]);
          }
        } else {
          constexpr int i = n - kScores;
          const bf16x8 w = operand8(s[i >> 1], i & 1), ds = operand8(p[i >> 1], i & 1);
#pragma unroll
          for (int t = 0; t < T; ++t) {
            if constexpr (DV) {
              if constexpr (kHow == kCareful) x[kOf * t] = finite_part(x[kOf * t], dirty);
              d_v[t] = mfma32(x[kOf * t], w, d_v[t]);
            }
            if constexpr (DK) {
              // a query that holds an infinity or NaN gives them to the dS of the keys it sees
              uint32_t unused = 0;
              if constexpr (kHow == kCareful) x[kOf * t + DV] = finite_part(x[kOf * t + DV], unused);
              d_k[t] = mfma32(x[kOf * t + DV], ds, d_k[t]);
            }
          }
        }
        // block b's weights beside the products behind its scores
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int from_group = (b + 1) * kGroups - (NB == 1 ? 1 : 0);
          if (kGroups == 1 && b + 1 < NB) {
            if (n == from_group) {
              weigh(b, 0);
              weigh(b, 8);
            }
          } else if (NB == 1) {
            if (n == from_group) {
              weigh(b, 0);
              weigh(b, 8);
            }
          } else if (n == from_group || n == from_group + 1) {
            weigh(b, 8 * (n - from_group));
          }
        }
      });
      if constexpr (DP > 64) fence();
    };
    const int first_own = start + half * (NB * 32);  // this wavefront's first row
    // turns whose rows all exist and see every key of the wavefront, two at a time
    int lead = from_all > start ? (from_all - start + RT - 1) / RT : 0;
    lead += lead & 1;
    lead = lead < steps ? lead : steps;
    const int end = (last_row - start) / RT, tail = end > lead ? lead + ((end - lead) & ~1) : lead;
    const auto pass = [&](auto how) {
#pragma unroll
      for (int t = 0; t < T; ++t) d_k[t] = d_v[t] = zero16();
      const auto masked = [&](int step) {
        loads_done();
        if (step + 1 < steps) issue(step + 1);
        if (first_own + step * RT + NB * 32 > from_some && first_own + step * RT < last_row) compute(step, step & 1, how);
      };
      int step = 0;
      for (; step < lead; ++step) masked(step);
      for (; step < tail; step += 2) {
        loads_done();
        issue(step + 1);
        compute(step, Constant<0>{}, Constant<kPlain>{});
        loads_done();
        if (step + 2 < steps) issue(step + 2);
        compute(step + 1, Constant<1>{}, Constant<kPlain>{});
      }
      for (; step < steps; ++step) masked(step);
    };
    pass(Constant<kMasked>{});
    if (voted<W>((DK && nonfinite(d_k)) || (DV && nonfinite(d_v)), lds, wave)) {
      issue(0);
      pass(Constant<kCareful>{});
      if (DV && __any(dirty != 0)) {
        const auto place = [&](int row) {
          const int token = group.quotient(row);
          return a.d_out.p + token * a.d_out.token + (head * a.group + row - token * a.group) * a.d_out.head;
        };
        const auto seen = [&](int row) { return row >= from; };
        const int until = start + lead * RT < last_row ? start + lead * RT : last_row;
        add_nonfinite<DP>(d_v, start, until, dim, h, place, seen);
        add_nonfinite<DP>(d_v, start + tail * RT > until ? start + tail * RT : until, last_row, dim, h, place, seen);
      }
    }

    const int64_t o = (static_cast<int64_t>(key) * a.kv_heads + head) * dim;
    if constexpr (RW == 1) {
      if (key >= seg.last) return;
      if (a.splits > 1) {
        if (DK) store_sums<DP>(sums_of(a, 0, split) + o, d_k, dim, h);
        if (DV) store_sums<DP>(sums_of(a, 1, split) + o, d_v, dim, h);
        return;
      }
      if (DK) store_operand<DP>(a.d_k + o, d_k, a.scale, dim, h);
      if (DV) store_operand<DP>(a.d_v + o, d_v, 1.0f, dim, h);
      return;
    }
    // Each of two wavefronts finishes half of the columns that both have sums of.
    __syncthreads();
    const auto sums = [&](int of, int n) { return reinterpret_cast<f32x4*>(lds + of * kSums + n * 4096) + 4 * lane; };
    const auto give = [&](const f32x16 (&x)[T], int slot) {
#pragma unroll
      for (int t = 0; t < T; ++t)
        if ((t >= T / 2) == (half == 0))
#pragma unroll
          for (int e = 0; e < 4; ++e) sums(wave, slot + t % (T / 2))[e] = (f32x4){x[t][4 * e], x[t][4 * e + 1], x[t][4 * e + 2], x[t][4 * e + 3]};
    };
    if (DK) give(d_k, 0);
    if (DV) give(d_v, DK ? T / 2 : 0);
    __syncthreads();
    if (key >= seg.last) return;
    const auto finish = [&](const f32x16 (&x)[T], int slot, float scale, uint16_t* to, float* partial) {
#pragma unroll
      for (int t = 0; t < T; ++t)
        if ((t < T / 2) == (half == 0))
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x4 y = sums(wave ^ KW, slot + t % (T / 2))[e];
            const int d = 32 * t + result_row(4 * e, h);
            if (d >= dim) continue;
            if (a.splits > 1)
              *reinterpret_cast<f32x4*>(partial + o + d) = (f32x4){x[t][4 * e], x[t][4 * e + 1], x[t][4 * e + 2], x[t][4 * e + 3]} + y;
            else
              *reinterpret_cast<u32x2*>(to + o + d) = pack4((x[t][4 * e] + y[0]) * scale, (x[t][4 * e + 1] + y[1]) * scale,
                                                            (x[t][4 * e + 2] + y[2]) * scale, (x[t][4 * e + 3] + y[3]) * scale);
          }
    };
    if (DK) finish(d_k, 0, a.scale, a.d_k, sums_of(a, 0, split));
    if (DV) finish(d_v, DK ? T / 2 : 0, 1.0f, a.d_v, sums_of(a, 1, split));
  }
};

template <class F>
__global__ __launch_bounds__(F::kThreads, F::DP == 256 ? 1 : 2) void query_gradient_kernel(AttentionArgs a, Divisor group, int tiles) {
  extern __shared__ __align__(1024) uint8_t lds[];
  F::run(a, group, tiles, lds);
}
template <class F>
__global__ __launch_bounds__(F::kThreads, F::DP == 64 ? 2 : 1) void key_gradient_kernel(AttentionArgs a, Divisor group, int tiles) {
  extern __shared__ __align__(1024) uint8_t lds[];
  F::run(a, group, tiles, lds);
}

template <class F>
hipError_t launch_query_gradient(const AttentionArgs& a, hipStream_t st) {
  if (a.tokens == 0) return hipSuccess;
  const int64_t tiles = tile_numbers(a.tokens * a.group, a.offsets != nullptr, a.sequences, F::kRows);
  query_gradient_kernel<F><<<static_cast<uint32_t>(tiles * a.kv_heads), F::kThreads, F::kLds, st>>>(a, Divisor(a.group), static_cast<int>(tiles));
  return hipGetLastError();
}
template <class F>
hipError_t launch_key_gradient(const AttentionArgs& a, hipStream_t st) {
  if (a.keys == 0) return hipSuccess;
  const int64_t tiles = tile_numbers(a.keys, a.offsets != nullptr, a.sequences, F::kKeys);
  key_gradient_kernel<F><<<static_cast<uint32_t>(tiles * a.kv_heads * a.splits), F::kThreads, F::kLds, st>>>(a, Divisor(a.group), static_cast<int>(tiles));
  return hipGetLastError();
}

// Adds the parts of d_k (blockIdx.y 0) or d_v in their order: four values a thread.  Bound
// by the bytes of the parts.
__global__ __launch_bounds__(256) void key_gradient_join_kernel(AttentionArgs a) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4, all = a.keys * a.kv_heads * a.dim;
  uint16_t* to = blockIdx.y == 0 ? a.d_k : a.d_v;
  if (i >= all || to == nullptr) return;
  const float* p = sums_of(a, blockIdx.y, 0) + i;
  f32x4 sum = *reinterpret_cast<const f32x4*>(p);
#pragma unroll 4
  for (int s = 1; s < a.splits; ++s) sum += *reinterpret_cast<const f32x4*>(p + s * all);
  const float by = blockIdx.y == 0 ? a.scale : 1.0f;
  *reinterpret_cast<u32x2*>(to + i) = pack4(sum[0] * by, sum[1] * by, sum[2] * by, sum[3] * by);
}

hipError_t join_key_gradients(const AttentionArgs& a, hipStream_t st) {
  if (a.splits == 1 || a.keys == 0) return hipSuccess;
  const int64_t quads = a.keys * a.kv_heads * a.dim / 4;
  key_gradient_join_kernel<<<dim3(static_cast<uint32_t>((quads + 255) / 256), 2), 256, 0, st>>>(a);
  return hipGetLastError();
}

// Whether to take 128 keys a workgroup, which load each row half as often as 64: where
// they are enough for every CU, and twice as many in causal sequences, whose tiles have
// different amounts of work (8,192 tokens in two sequences, 16 / 4 heads, all seen: 927 us
// with 128 keys, 1026 with 64; 4,096 causal tokens, 16 / 4 heads of 96: 556 and 401).  With
// 32,768 keys of all heads, of up to 64 values and all seen, their rows are split too (all
// gradients of 4,096 tokens, 32 / 8 heads: 528 us; unsplit 536, split with 64 keys 545).
bool wide_key_tiles(const AttentionArgs& a) { return a.keys * a.kv_heads / 128 >= (a.causal ? 512 : 256); }

template <int DP, bool EXACT, int NB>
hipError_t backward(const AttentionArgs& a, hipStream_t st) {
  hipError_t e = hipSuccess;
  if (a.d_q != nullptr)
    e = launch_query_gradient<QueryGradient<DP, EXACT, true>>(a, st);
  else if (a.d_k != nullptr)
    e = launch_query_gradient<QueryGradient<DP, EXACT, false>>(a, st);  // for delta
  if (e != hipSuccess) return e;
  // both gradients of 256 columns at once would not leave a lane registers for the scores
  if constexpr (DP < 256) {
    if (a.d_k != nullptr && a.d_v != nullptr) {
      e = wide_key_tiles(a) ? launch_key_gradient<KeyGradient<DP, EXACT, NB, 1, true, true>>(a, st)
                            : launch_key_gradient<KeyGradient<DP, EXACT, NB, 2, true, true>>(a, st);
      return e != hipSuccess ? e : join_key_gradients(a, st);
    }
  }
  if (a.d_k != nullptr)
    if (e = launch_key_gradient<KeyGradient<DP, EXACT, NB, 2, true, false>>(a, st); e != hipSuccess) return e;
  if (a.d_v != nullptr)
    if (e = launch_key_gradient<KeyGradient<DP, EXACT, NB, 2, false, true>>(a, st); e != hipSuccess) return e;
  return a.d_k != nullptr || a.d_v != nullptr ? join_key_gradients(a, st) : hipSuccess;
}

template <class F>
hipError_t launch_forward(const AttentionArgs& a, hipStream_t st) {
  const int64_t tiles = tile_numbers(a.tokens * a.group, a.offsets != nullptr, a.sequences, F::kRows);
  attention_kernel<F><<<static_cast<uint32_t>(tiles * a.kv_heads), F::kThreads, F::kLds, st>>>(a, Divisor(a.group), static_cast<int>(tiles));
  return hipGetLastError();
}

}  // namespace

}  // namespace glm53
