// Attention within packed sequences, forward and backward.
//
//   S = scale q k^T over the keys a query sees, P = softmax(S), out = P v
//
// A row is one query of one head.  The `group` heads of a key head are rows
// of the same tile, token by token, so that a tile's keys and values serve all
// of them, and a key head's gradients are one contraction over its rows.
#pragma once

#include <type_traits>

#include "attention.h"
#include "attention_tile.h"

namespace glm53 {

namespace {

#ifndef QAHEAD
#define QAHEAD 1
#endif
#ifndef KAHEAD64
#define KAHEAD64 2
#endif
// Keeps what is in front of it in front and what is behind it behind, when the
// compiler orders instructions: left alone it puts each LDS read directly
// before the product that waits for it.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// Around a run of products: its wavefront goes first on its SIMD, so that the
// other one there comes to its weights while this one multiplies (16,384 causal
// tokens, 8 heads of 128: 505 us, without 560).
__device__ __forceinline__ void products(bool begin) {
  if (begin)
    __builtin_amdgcn_s_setprio(1);
  else
    __builtin_amdgcn_s_setprio(0);
}

constexpr float kLog2e = 1.44269504088896340736f;
// A row's maximum is kept until a new one is this many powers of two above it:
// the weights 2^(s - m) then reach 2^8, which changes no relative rounding, and
// few tiles after the first rescale their sums.
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

// Tile numbers of `rows` rows in `sequences` sequences (see find_segment).
int64_t tile_numbers(int64_t rows, bool packed, int sequences, int size) {
  return packed ? rows / size + sequences + 2 : (rows + size - 1) / size;
}

// ------------------------------------------------------------- forward ---
//
// W wavefronts of RB x 32 rows; a tile of 64 keys is multiplied while the next
// one is loaded.  Scores are computed as S^T (keys the result's rows), so a
// lane holds 32 of its row's 64 scores, a row's maximum and sum are within a
// lane and its counterpart 32 lanes away, and the weights go into the second
// product (out^T = v^T P^T) from the registers they are in.

template <int DP_, bool EXACT, int RB_, int W_>
struct Forward {
  static constexpr int DP = DP_, RB = RB_, W = W_;
  static constexpr int kRows = 32 * RB * W, kThreads = 64 * W, kKeys = 64, T = DP / 32;
  using Tile = HeadTile<DP, kKeys, W>;
  static constexpr int kLds = 4 * Tile::kBytes;  // two stages of keys and values

  static __device__ __forceinline__ void run(const AttentionArgs& a, const Divisor& group, int tiles, uint8_t* lds) {
    const int dim = EXACT ? DP : a.dim;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.kv_heads, number = tiles - 1 - blockIdx.x / a.kv_heads;
    const Segment seg = find_segment(a.offsets, a.sequences, a.tokens, a.group, kRows, number);
    const int row0 = seg.first + seg.tile * kRows;
    if (seg.tile < 0 || row0 >= seg.last) return;

    int key0, keys;
    sequence_keys(a, group, seg, key0, keys);
    // keys that the query of row r sees: a prefix
    const int shift = keys - group.quotient(seg.last - seg.first);
    const auto limit = [&](int row) {
      if (!a.causal) return keys;
      const int n = group.quotient(row - seg.first) + shift + 1;
      return n < 0 ? 0 : n > keys ? keys : n;
    };
    const int last_row = row0 + kRows < seg.last ? row0 + kRows - 1 : seg.last - 1;
    const int steps = (__builtin_amdgcn_readfirstlane(limit(last_row)) + kKeys - 1) / kKeys;

    const int h = lane >> 5;
    if (dim < DP) {
#pragma unroll
      for (int s = 0; s < 4; ++s) Tile::clear(lds + s * Tile::kBytes, dim, kThreads);
    }
    const uint16_t* kp = a.k.p + static_cast<int64_t>(key0) * a.k.token + static_cast<int64_t>(head) * a.k.head;
    const uint16_t* vp = a.v.p + static_cast<int64_t>(key0) * a.v.token + static_cast<int64_t>(head) * a.v.head;
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds));
    const auto issue = [&](int step) {
      const uint32_t at = lds_at + (step & 1) * 2 * Tile::kBytes;
      const int64_t first = static_cast<int64_t>(step) * kKeys;
      const int left = keys - step * kKeys;
      Tile::load(kp + first * a.k.token, static_cast<uint32_t>(2 * a.k.token), left, dim, wave, lane, at);
      Tile::load(vp + first * a.v.token, static_cast<uint32_t>(2 * a.v.token), left, dim, wave, lane, at + Tile::kBytes);
    };

    if (steps > 0) issue(0);
    int row[RB], lim[RB];
    bf16x8 q[RB][DP / 16];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      row[b] = row0 + 32 * (RB * wave + b) + (lane & 31);
      const int r = row[b] < seg.last ? row[b] : seg.last - 1;  // rows past the last repeat it
      lim[b] = limit(r);
      const int token = group.quotient(r);
      const uint16_t* p = a.q.p + token * a.q.token + (head * a.group + r - token * a.group) * a.q.head;
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) {
        u32x4 v = {0, 0, 0, 0};
        if (16 * j + 8 * h < dim) v = *reinterpret_cast<const u32x4*>(p + 16 * j + 8 * h);
        q[b][j] = __builtin_bit_cast(bf16x8, v);
      }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) arrived(q[b][j]);
    const int all_see = __builtin_amdgcn_readfirstlane(lim[0]);                  // every row of the wavefront
    const int some_see = __builtin_amdgcn_readlane(lim[RB - 1], 31);             // its last row

    const typename Tile::Places at(lds_at, lane);
    const float c = a.scale * kLog2e;
    f32x16 out[RB][DP / 32];
    float m[RB], l[RB];  // m in units of scores; l: this lane's part
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      m[b] = -INFINITY;
      l[b] = 0.0f;
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) out[b][t] = zero16();
    }

    uint32_t dirty = 0;
    const auto compute = [&](int step, auto stage, auto masked) {
      constexpr bool kMasked = decltype(masked)::value;
      const int kt = stage * 2 * Tile::kBytes, vt = kt + Tile::kBytes;
      f32x16 s[RB][2];
      // groups of operands: the keys' in kb and 64 columns, the values' in 16 keys
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
      read(0);
      read(1);
      products(true);
#pragma unroll
      for (int n = 0; n < 2 * kGroups; ++n) {
        fence();
        read(n + 2);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int b = 0; b < RB; ++b)
            s[b][n / kGroups] = mfma32(f[n % 3][j], q[b][4 * (n % kGroups) + j], n % kGroups + j == 0 ? zero16() : s[b][n / kGroups]);
      }
      fence();
      products(false);
      float mc[RB];
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        if constexpr (kMasked) {
          const int left = lim[b] - step * kKeys - 4 * h;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (32 * kb + result_row(r, 0) >= left) s[b][kb][r] = -INFINITY;
        }
        float top = s[b][0][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[b][0][r]);
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][1][r]);
        top = both_max(top);
        if (__any(top * c > m[b] * c + kSlack)) {
          const float next = fmaxf(m[b], top);
          const float alpha = next == -INFINITY ? 1.0f : exp2_fast((m[b] - next) * c);
          m[b] = next;
          l[b] *= alpha;
#pragma unroll
          for (int t = 0; t < T; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[b][t][r] *= alpha;
        }
        mc[b] = m[b] == -INFINITY ? 0.0f : m[b] * c;
      }
      bf16x8 p[RB], next[RB];
      const auto weigh = [&](int i) {  // 8 of a lane's scores
#pragma unroll
        for (int b = 0; b < RB; ++b) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            s[b][i >> 1][8 * (i & 1) + e] = exp2_fast(fmaf(s[b][i >> 1][8 * (i & 1) + e], c, -mc[b]));
          float sum = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += s[b][i >> 1][8 * (i & 1) + e];
          l[b] += sum;
          next[b] = operand8(s[b][i >> 1], i & 1);
        }
      };
      weigh(0);
      products(true);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fence();
        const int n = 2 * kGroups + i;
        read(n + 2);
#pragma unroll
        for (int b = 0; b < RB; ++b) p[b] = next[b];
#pragma unroll
        for (int t = 0; t < T; ++t) {
          if constexpr (kMasked) f[n % 3][t] = finite_part(f[n % 3][t], dirty);
#pragma unroll
          for (int b = 0; b < RB; ++b) out[b][t] = mfma32(f[n % 3][t], p[b], out[b][t]);
        }
        if (i < 3) weigh(i + 1);
      }
      fence();
      products(false);
    };

    // whole tiles two at a time: their places in LDS are constants then
    const int whole = all_see / kKeys & ~1;
    int step = 0;
    for (; step < whole; step += 2) {
      loads_done();
      issue(step + 1);
      compute(step, std::integral_constant<int, 0>{}, std::false_type{});
      loads_done();
      if (step + 2 < steps) issue(step + 2);
      compute(step + 1, std::integral_constant<int, 1>{}, std::false_type{});
    }
    for (; step < steps; ++step) {
      loads_done();
      if (step + 1 < steps) issue(step + 1);
      if (step * kKeys < some_see) compute(step, step & 1, std::true_type{});
    }

    if (__any(dirty != 0)) {
#pragma unroll
      for (int b = 0; b < RB; ++b)
        add_nonfinite<DP>(out[b], whole * kKeys, some_see, dim, h,
                          [&](int key) { return vp + key * a.v.token; }, [&](int key) { return key < lim[b]; });
    }
    const int64_t heads = static_cast<int64_t>(a.kv_heads) * a.group;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const float total = both_sum(l[b]);
      const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
      if (row[b] >= seg.last) continue;
      const int token = group.quotient(row[b]);
      uint16_t* o = a.out + (token * heads + head * a.group + row[b] - token * a.group) * dim;
#pragma unroll
      for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int d = 32 * t + result_row(r, h);
          if (d < dim)
            *reinterpret_cast<u32x2*>(o + d) = pack4(out[b][t][r] * inverse, out[b][t][r + 1] * inverse,
                                                     out[b][t][r + 2] * inverse, out[b][t][r + 3] * inverse);
        }
      if (a.lse != nullptr && h == 0)
        a.lse[static_cast<int64_t>(head) * a.tokens * a.group + row[b]] =
            total == 0.0f ? 0.0f : m[b] * c + __builtin_amdgcn_logf(total);
    }
  }
};

template <class F>
__global__ __launch_bounds__(F::kThreads, F::DP == 256 || F::RB == 2 ? 1 : F::W == 8 ? 1 : 2) void attention_kernel(AttentionArgs a, Divisor group, int tiles) {
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
// products instead of five.
//
// delta from the rounded `out` is off by as much as `out` is, and puts that into
// every dS of its row.  The rows' sums of dS, which are 0, say by how much:
// the first kernel adds them to delta for the second one, and carries dS in two
// bf16 parts, so that both gradients are off by one operand's rounding at most
// (relative error 0.0024 instead of 0.0026 to 0.0029).

// d_q: a lane's row as in the forward pass, a tile of 64 keys at a time.
template <int DP_, bool EXACT, int W_, bool DQ>
struct QueryGradient {
  static constexpr int DP = DP_, W = W_;
  static constexpr int kRows = 32 * W, kThreads = 64 * W, kKeys = 64, T = DP / 32;
  using Tile = HeadTile<DP, kKeys, W>;
  static constexpr int kLds = 4 * Tile::kBytes;

  static __device__ __forceinline__ void run(const AttentionArgs& a, const Divisor& group, int tiles, uint8_t* lds) {
    const int dim = EXACT ? DP : a.dim;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.kv_heads, number = tiles - 1 - blockIdx.x / a.kv_heads;
    const Segment seg = find_segment(a.offsets, a.sequences, a.tokens, a.group, kRows, number);
    const int row0 = seg.first + seg.tile * kRows;
    if (seg.tile < 0 || row0 >= seg.last) return;
    int key0, keys;
    sequence_keys(a, group, seg, key0, keys);
    const int shift = keys - group.quotient(seg.last - seg.first);
    const auto limit = [&](int row) {
      if (!a.causal) return keys;
      const int n = group.quotient(row - seg.first) + shift + 1;
      return n < 0 ? 0 : n > keys ? keys : n;
    };
    const int last_row = row0 + kRows < seg.last ? row0 + kRows - 1 : seg.last - 1;
    const int steps = (__builtin_amdgcn_readfirstlane(limit(last_row)) + kKeys - 1) / kKeys;

    const int h = lane >> 5, row = row0 + 32 * wave + (lane & 31);
    const int r = row < seg.last ? row : seg.last - 1, token = group.quotient(r), query_head = head * a.group + r - token * a.group;
    const int lim = limit(r);
    if (dim < DP) {
#pragma unroll
      for (int s = 0; s < 4; ++s) Tile::clear(lds + s * Tile::kBytes, dim, kThreads);
    }
    const uint16_t* kp = a.k.p + key0 * a.k.token + head * a.k.head;
    const uint16_t* vp = a.v.p + key0 * a.v.token + head * a.v.head;
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds));
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
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
      if (16 * j + 8 * h < dim) {
        x = *reinterpret_cast<const u32x4*>(qp + 16 * j + 8 * h);
        y = *reinterpret_cast<const u32x4*>(dp + 16 * j + 8 * h);
      }
      q[j] = __builtin_bit_cast(bf16x8, x);
      d_out[j] = __builtin_bit_cast(bf16x8, y);
    }
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
    float sum = 0.0f;  // of dS
    f32x16 d_q[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) d_q[t] = zero16();
    const auto compute = [&](int step, auto stage, auto masked) {
      constexpr bool kMasked = decltype(masked)::value;
      const int kt = stage * 2 * Tile::kBytes, vt = kt + Tile::kBytes;
      // groups of operands, read ahead of the products that take them: of 32 keys
      // those of 32 columns of scores at a time, then those of 16 keys
      constexpr int kGroups = DP / 32, kAhead = QAHEAD, kPart = kGroups + (DQ ? 2 : 0), kAll = 2 * kPart, kMost = T > 4 ? T : 4;
      bf16x8 f[kAhead + 1][kMost];
      const auto read = [&](int n) {
        if (n >= kAll) return;
        bf16x8 (&x)[kMost] = f[n % (kAhead + 1)];
        const int kb = n / kPart, g = n % kPart;
        if (g < kGroups) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            x[2 * j] = at.along(kt, kb, 2 * g + j);
            x[2 * j + 1] = at.along(vt, kb, 2 * g + j);
          }
        } else {
#pragma unroll
          for (int t = 0; t < T; ++t) x[t] = at.across(kt, 2 * kb + g - kGroups, t);
        }
      };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) read(n);
      f32x16 s, p;
      products(true);
#pragma unroll
      for (int n = 0; n < kAll; ++n) {
        const int kb = n / kPart, g = n % kPart;
        fence();
        read(n + kAhead);
        bf16x8 (&x)[kMost] = f[n % (kAhead + 1)];
        if (g == 0) {
          s = zero16();
#pragma unroll
          for (int e = 0; e < 16; ++e) p[e] = -delta;
        }
        if (g < kGroups) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s = mfma32(x[2 * j], q[2 * g + j], s);
            p = mfma32(x[2 * j + 1], d_out[2 * g + j], p);
          }
        } else {
          const bf16x8 ds = operand8(s, g - kGroups), low = low_operand8(s, g - kGroups, ds);
#pragma unroll
          for (int t = 0; t < T; ++t) {
            // a key that holds an infinity or NaN gives them to the dS of the rows that see it
            uint32_t unused = 0;
            if constexpr (kMasked) x[t] = finite_part(x[t], unused);
            d_q[t] = mfma32(x[t], ds, d_q[t]);
            d_q[t] = mfma32(x[t], low, d_q[t]);
          }
        }
        if (g == kGroups - 1) {
          fence();
          products(false);
          const int left = lim - step * kKeys - 32 * kb - 4 * h;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[e] = exp2_fast(fmaf(s[e], c, -lse)) * p[e];
            if (kMasked && result_row(e, 0) >= left) s[e] = 0.0f;
            sum += s[e];
          }
          products(true);
        }
      }
      fence();
      products(false);
    };
    // whole tiles two at a time: their places in LDS are constants then
    const int whole = all_see / kKeys & ~1;
    int step = 0;
    for (; step < whole; step += 2) {
      loads_done();
      issue(step + 1);
      compute(step, std::integral_constant<int, 0>{}, std::false_type{});
      loads_done();
      if (step + 2 < steps) issue(step + 2);
      compute(step + 1, std::integral_constant<int, 1>{}, std::false_type{});
    }
    for (; step < steps; ++step) {
      loads_done();
      if (step + 1 < steps) issue(step + 1);
      if (step * kKeys < some_see) compute(step, step & 1, std::true_type{});
    }
    sum = both_sum(sum);
    if (row >= seg.last) return;
    if (h == 0) {  // where the second kernel's products start
      a.starts[stat] = -lse / c;
      a.starts[stat + heads * a.tokens] = -(delta + sum);
    }
    if (!DQ) return;
    uint16_t* o = a.d_q + own;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = 32 * t + result_row(e, h);
        if (d < dim)
          *reinterpret_cast<u32x2*>(o + d) =
              pack4(d_q[t][e] * a.scale, d_q[t][e + 1] * a.scale, d_q[t][e + 2] * a.scale, d_q[t][e + 3] * a.scale);
      }
  }
};

// d_k and d_v: a lane's key and a tile of rows at a time.  Scores are computed
// with rows the result's rows, so that P and dS are the second operands of
// d_v^T += d_out^T P and d_k^T += q^T dS as they are.  Of the four wavefronts two
// and two share 32 keys, each with half of a tile's rows, and add up at the end: a
// workgroup has 64 keys and half as many turns, so that the first keys of a
// causal sequence, which all rows see, take no longer than the card takes for the
// rest (8,192 tokens in three sequences, 8 key heads: DKDV us; 128 keys a
// workgroup: 777).
template <int DP_, bool EXACT, int NB_, bool DK, bool DV>
struct KeyGradient {
  static constexpr int DP = DP_, NB = NB_;  // NB blocks of 32 rows a wavefront and turn
  static constexpr int W = 4, kKeys = 64, kThreads = 64 * W, RT = 2 * NB * 32, T = DP / 32;
  using Tile = HeadTile<DP, RT, W>;
  static constexpr int kStats = 4 * 64 * ((RT + 63) / 64);      // bytes of lse, and of delta
  static constexpr int kStage = 2 * Tile::kBytes + 2 * kStats;  // q, d_out, lse, delta
  static constexpr int kSums = (DK + DV) * T / 2 * 4096;        // of one wavefront, exchanged at the end
  static constexpr int kLds = 2 * kStage > 4 * kSums ? 2 * kStage : 4 * kSums;

  static __device__ __forceinline__ void run(const AttentionArgs& a, const Divisor& group, uint8_t* lds) {
    const int dim = EXACT ? DP : a.dim;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = wave >> 1;  // of a tile's rows
    const int head = blockIdx.x % a.kv_heads, number = blockIdx.x / a.kv_heads;
    const Segment seg = find_segment(a.key_offsets != nullptr ? a.key_offsets : a.offsets, a.sequences, a.keys, 1, kKeys, number);
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
    const int h = lane >> 5, key = key0 + 32 * (wave & 1) + (lane & 31), k = key < seg.last ? key : seg.last - 1;
    const int from = sees(k), from_all = __builtin_amdgcn_readlane(from, 31), from_some = __builtin_amdgcn_readfirstlane(from);
    const int start = __builtin_amdgcn_readfirstlane(sees(key0));
    const int steps = start < last_row ? (last_row - start + RT - 1) / RT : 0;

    if (dim < DP) {
#pragma unroll
      for (int s = 0; s < 4; ++s) Tile::clear(lds + (s >> 1) * kStage + (s & 1) * Tile::kBytes, dim, kThreads);
    }
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds));
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
      const auto offset = [&](const Rows16& x) {  // start, and so row0, is a token's first row
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
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
      if (16 * j + 8 * h < dim) {
        x = *reinterpret_cast<const u32x4*>(kp + 16 * j + 8 * h);
        if (DK) y = *reinterpret_cast<const u32x4*>(vp + 16 * j + 8 * h);
      }
      kf[j] = __builtin_bit_cast(bf16x8, x);
      vf[j] = __builtin_bit_cast(bf16x8, y);
    }
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      arrived(kf[j]);
      if (DK) arrived(vf[j]);
    }
    const typename Tile::Places at(lds_at + half * (NB * 32 * Tile::kPitch), lane);
    const float c = a.scale * kLog2e, start_scale = -1.0f / c;
    f32x16 d_k[T], d_v[T];
#pragma unroll
    for (int t = 0; t < T; ++t) d_k[t] = d_v[t] = zero16();
    uint32_t dirty = 0;
    const auto compute = [&](int step, auto stage, auto masked) {
      constexpr bool kMasked = decltype(masked)::value;
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
            s[b][e + i] = DK ? l[i] : l[i] * start_scale;
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
          if constexpr (kMasked) {
            const int row = start + step * RT + half * (NB * 32) + 32 * b + 4 * h + result_row(e, 0);
            if (row < from || row >= last_row) s[b][e] = p[b][e] = 0.0f;
          }
        }
      };
      if constexpr (DK && DV && NB == 2 && !kMasked) {
        // Operands are read two groups ahead of the products that take them, and the weights
        // of a block are made beside the products of the other one.
        constexpr int kGroups = DP / 64;  // of a block's scores
        constexpr int kAhead = DP == 64 ? KAHEAD64 : 2;
        bf16x8 f[kAhead + 1][8];
        const auto read_scores = [&](bf16x8 (&x)[8], int n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[2 * j] = at.along(qt, n / kGroups, 4 * (n % kGroups) + j);
            x[2 * j + 1] = at.along(ot, n / kGroups, 4 * (n % kGroups) + j);
          }
        };
        const auto scores = [&](const bf16x8 (&x)[8], int n) {
          const int b = n / kGroups;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[b] = mfma32(x[2 * j], kf[4 * (n % kGroups) + j], s[b]);
            p[b] = mfma32(x[2 * j + 1], vf[4 * (n % kGroups) + j], p[b]);
          }
        };
        const auto read_across = [&](bf16x8 (&x)[8], int n) {
#pragma unroll
          for (int t = 0; t < T; ++t) {
            x[2 * t] = at.across(ot, n, t);
            x[2 * t + 1] = at.across(qt, n, t);
          }
        };
        const auto add = [&](const bf16x8 (&x)[8], int n) {
          const bf16x8 w = operand8(s[n >> 1], n & 1), ds = operand8(p[n >> 1], n & 1);
#pragma unroll
          for (int t = 0; t < T; ++t) {
            d_v[t] = mfma32(x[2 * t], w, d_v[t]);
            d_k[t] = mfma32(x[2 * t + 1], ds, d_k[t]);
          }
        };
        constexpr int kAll = 2 * kGroups + 4;
        const auto read = [&](int n) { n < 2 * kGroups ? read_scores(f[n % (kAhead + 1)], n) : read_across(f[n % (kAhead + 1)], n - 2 * kGroups); };
        begin(0);
        begin(1);
#pragma unroll
        for (int n = 0; n < kAhead; ++n) read(n);
#pragma unroll
        for (int n = 0; n < kAll; ++n) {
          fence();
          if (n + kAhead < kAll) read(n + kAhead);
          if (n < 2 * kGroups) scores(f[n % (kAhead + 1)], n);
          else add(f[n % (kAhead + 1)], n - 2 * kGroups);
          // block 0's weights beside block 1's scores, block 1's beside block 0's sums
          if (n >= kGroups && n < 2 * kGroups) {
            weigh(0, kGroups == 2 ? 8 * (n - kGroups) : 0);
            if (kGroups == 1) weigh(0, 8);
          }
          if (n >= 2 * kGroups && n < 2 * kGroups + 2) weigh(1, 8 * (n - 2 * kGroups));
        }
        fence();
        return;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        begin(b);
#pragma unroll
        for (int j = 0; j < DP / 16; ++j) {
          s[b] = mfma32(at.along(qt, b, j), kf[j], s[b]);
          if (DK) p[b] = mfma32(at.along(ot, b, j), vf[j], p[b]);
        }
        weigh(b, 0);
        weigh(b, 8);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bf16x8 w = operand8(s[b], i), ds = operand8(p[b], i);
#pragma unroll
          for (int t = 0; t < T; ++t) {
            if constexpr (DV) {
              bf16x8 f = at.across(ot, 2 * b + i, t);
              if constexpr (kMasked) f = finite_part(f, dirty);
              d_v[t] = mfma32(f, w, d_v[t]);
            }
            if constexpr (DK) {
              bf16x8 f = at.across(qt, 2 * b + i, t);
              // a query that holds an infinity or NaN gives them to the dS of the keys it sees
              uint32_t unused = 0;
              if constexpr (kMasked) f = finite_part(f, unused);
              d_k[t] = mfma32(f, ds, d_k[t]);
            }
          }
        }
    };
    const int first_own = start + half * (NB * 32);  // this wavefront's first row
    const auto masked = [&](int step) {
      loads_done();
      if (step + 1 < steps) issue(step + 1);
      if (first_own + step * RT + NB * 32 > from_some && first_own + step * RT < last_row) compute(step, step & 1, std::true_type{});
    };
    // turns whose rows all exist and see every key of the wavefront, two at a time
    int lead = from_all > start ? (from_all - start + RT - 1) / RT : 0;
    lead += lead & 1;
    const int end = (last_row - start) / RT;
    int step = 0;
    for (; step < (lead < steps ? lead : steps); ++step) masked(step);
    for (; step + 2 <= end; step += 2) {
      loads_done();
      issue(step + 1);
      compute(step, std::integral_constant<int, 0>{}, std::false_type{});
      loads_done();
      if (step + 2 < steps) issue(step + 2);
      compute(step + 1, std::integral_constant<int, 1>{}, std::false_type{});
    }
    const int tail = start + step * RT;
    for (; step < steps; ++step) masked(step);
    if (DV && __any(dirty != 0)) {
      const auto place = [&](int row) {
        const int token = group.quotient(row);
        return a.d_out.p + token * a.d_out.token + (head * a.group + row - token * a.group) * a.d_out.head;
      };
      const auto seen = [&](int row) { return row >= from; };
      const int until = start + lead * RT < last_row ? start + lead * RT : last_row;
      add_nonfinite<DP>(d_v, start, until, dim, h, place, seen);
      add_nonfinite<DP>(d_v, tail > until ? tail : until, last_row, dim, h, place, seen);
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
    const int64_t o = (static_cast<int64_t>(key) * a.kv_heads + head) * dim;
    const auto finish = [&](const f32x16 (&x)[T], int slot, float scale, uint16_t* to) {
#pragma unroll
      for (int t = 0; t < T; ++t)
        if ((t < T / 2) == (half == 0))
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x4 y = sums(wave ^ 2, slot + t % (T / 2))[e];
            const int d = 32 * t + result_row(4 * e, h);
            if (d < dim)
              *reinterpret_cast<u32x2*>(to + o + d) = pack4((x[t][4 * e] + y[0]) * scale, (x[t][4 * e + 1] + y[1]) * scale,
                                                            (x[t][4 * e + 2] + y[2]) * scale, (x[t][4 * e + 3] + y[3]) * scale);
          }
    };
    if (DK) finish(d_k, 0, a.scale, a.d_k);
    if (DV) finish(d_v, DK ? T / 2 : 0, 1.0f, a.d_v);
  }
};

template <class F>
__global__ __launch_bounds__(F::kThreads, F::DP == 256 ? 1 : 2) void query_gradient_kernel(AttentionArgs a, Divisor group, int tiles) {
  extern __shared__ __align__(1024) uint8_t lds[];
  F::run(a, group, tiles, lds);
}
template <class F>
__global__ __launch_bounds__(F::kThreads, F::DP == 64 ? 2 : 1) void key_gradient_kernel(AttentionArgs a, Divisor group) {
  extern __shared__ __align__(1024) uint8_t lds[];
  F::run(a, group, lds);
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
  key_gradient_kernel<F><<<static_cast<uint32_t>(tiles * a.kv_heads), F::kThreads, F::kLds, st>>>(a, Divisor(a.group));
  return hipGetLastError();
}

template <int DP, bool EXACT, int NB>
hipError_t backward(const AttentionArgs& a, hipStream_t st) {
  hipError_t e = hipSuccess;
  if (a.d_q != nullptr)
    e = launch_query_gradient<QueryGradient<DP, EXACT, 4, true>>(a, st);
  else if (a.d_k != nullptr)
    e = launch_query_gradient<QueryGradient<DP, EXACT, 4, false>>(a, st);  // for delta
  if (e != hipSuccess) return e;
  // both gradients of 256 columns at once would not leave a lane registers for the scores
  if (DP < 256 && a.d_k != nullptr && a.d_v != nullptr) return launch_key_gradient<KeyGradient<DP, EXACT, NB, DP < 256, true>>(a, st);
  if (a.d_k != nullptr)
    if (e = launch_key_gradient<KeyGradient<DP, EXACT, NB, true, false>>(a, st); e != hipSuccess) return e;
  if (a.d_v != nullptr) return launch_key_gradient<KeyGradient<DP, EXACT, NB, false, true>>(a, st);
  return hipSuccess;
}

template <class F>
hipError_t launch_forward(const AttentionArgs& a, hipStream_t st) {
  const int64_t tiles = tile_numbers(a.tokens * a.group, a.offsets != nullptr, a.sequences, F::kRows);
  attention_kernel<F><<<static_cast<uint32_t>(tiles * a.kv_heads), F::kThreads, F::kLds, st>>>(a, Divisor(a.group), static_cast<int>(tiles));
  return hipGetLastError();
}

}  // namespace

}  // namespace glm53
