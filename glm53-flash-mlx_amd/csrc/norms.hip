// Norms before and after a block, fused with the block's gate and residual
// scale, and their gradients.
//
//   s = o r_o p,  r_o = (mean o^2 + eps)^-1/2     (without a post norm: s = o)
//   x' = x + a g s
//   y = x' r' w,  r' = (mean x'^2 + eps)^-1/2
//
// One workgroup holds a row in registers from its load to its store, so that
// each tensor crosses HBM once in a pass: over many rows the kernels are bound by
// those bytes.  Beside them the gradients write and read partial column sums, which
// over few rows are as many (norm_backward_kernel), and past 8,192 columns
// their registers spill.  All values between load and store are fp32; y is made
// of the x' that has not been rounded yet.  Squares are summed as they are: rows
// of values past 2^63 sum to infinity, and their norm is 0.
#include "common.h"
#include "norms.h"

namespace glm53 {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kVec = 8;  // elements a thread loads at once

// 16 bytes at any element's address: rows of odd widths, and views, start
// anywhere, and the memory takes such loads whole.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;

struct Raw {
  u32x4 lo, hi;
};

// How a row's last elements are taken where the width is no multiple of kVec.
// kWhole: it is one.  kOverlap: the last load is the row's last kVec elements,
// whose first ones another thread has too: both compute and store the same
// values for them, and one of the two leaves them out of the row's sums (8,192
// x 2,050 forward: 52 us, 108 with single elements).
// kSingly (rows shorter than kVec): one by one.
enum Ends { kWhole, kOverlap, kSingly };

// kVec elements from element index i, as stored (kSingly: `left` of them, the
// others 0); converted by to_float once every load of the row is on its way.
template <Ends E>
__device__ __forceinline__ Raw load_raw(const Tensor& t, int64_t i, int64_t left) {
  Raw r{};
  if constexpr (E == kSingly) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (e >= left) break;
      if (t.f32) {
        const uint32_t v = static_cast<const uint32_t*>(t.p)[i + e];
        if (e < 4)
          r.lo[e] = v;
        else
          r.hi[e - 4] = v;
      } else {
        r.lo[e / 2] |= static_cast<uint32_t>(static_cast<const uint16_t*>(t.p)[i + e]) << (16 * (e & 1));
      }
    }
  } else if (t.f32) {
    const u32x4_any* p = reinterpret_cast<const u32x4_any*>(static_cast<const float*>(t.p) + i);
    r.lo = p[0];
    r.hi = p[1];
  } else {
    r.lo = *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(t.p) + i);
  }
  return r;
}

__device__ __forceinline__ void to_float(const Raw& r, bool f32, float* v) {
  if (f32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = __uint_as_float(r.lo[e]);
      v[4 + e] = __uint_as_float(r.hi[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(r.lo[e] << 16);
      v[2 * e + 1] = __uint_as_float(r.lo[e] & 0xFFFF0000u);
    }
  }
}

__device__ __forceinline__ void store_one(const Tensor& t, int64_t i, float v) {
  if (t.f32)
    static_cast<float*>(t.p)[i] = v;
  else
    static_cast<uint16_t*>(t.p)[i] = f32_to_bf16(v);
}

template <Ends E>
__device__ __forceinline__ void store(const Tensor& t, int64_t i, int64_t left, const float* v) {
  if constexpr (E == kSingly) {
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if (e < left) store_one(t, i + e, v[e]);
  } else if (t.f32) {
    u32x4_any* p = reinterpret_cast<u32x4_any*>(static_cast<float*>(t.p) + i);
    u32x4 lo, hi;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = __float_as_uint(v[e]);
      hi[e] = __float_as_uint(v[4 + e]);
    }
    p[0] = lo;
    p[1] = hi;
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = f32_to_bf16(v[2 * e]) | static_cast<uint32_t>(f32_to_bf16(v[2 * e + 1])) << 16;
    *reinterpret_cast<u32x4_any*>(static_cast<uint16_t*>(t.p) + i) = w;
  }
}

__device__ __forceinline__ float scalar(const Tensor& t, int64_t i) {
  return t.f32 ? static_cast<const float*>(t.p)[i] : bf16_to_f32(static_cast<const uint16_t*>(t.p)[i]);
}

// Sum over the T threads of a row, in every one of them.  `turn` alternates
// between two sets of LDS words, so one barrier a sum is enough.
template <int T>
__device__ __forceinline__ float row_sum(float v, float (*words)[T / kWave], int& turn) {
  v = wave_sum(v);
  if constexpr (T == kWave) return v;
  float* w = words[turn];
  turn ^= 1;
  if ((threadIdx.x & (kWave - 1)) == 0) w[threadIdx.x / kWave] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < T / kWave; ++i) s += w[i];
  return s;
}

// A row's threads and how its elements lie on them: T threads, C chunks of
// kVec consecutive elements each, chunk c of thread t at (c T + t) kVec.
template <int T, int C, Ends E>
struct Row {
  static constexpr int kN = kVec * C;
  __device__ static __forceinline__ int64_t chunk(int c) { return (static_cast<int64_t>(c) * T + threadIdx.x) * kVec; }
  // where chunk c starts, in a row that has it
  __device__ static __forceinline__ int64_t at(int c, int64_t width) {
    const int64_t i = chunk(c);
    return E == kOverlap && i + kVec > width ? width - kVec : i;
  }
  // whether element e counts in a row's sum: it is no second copy
  __device__ static __forceinline__ bool counts(int e, int64_t width) {
    if (E != kOverlap) return true;
    const int64_t i = chunk(e / kVec);
    return i + kVec <= width || e % kVec >= i + kVec - width;
  }

  // Row elements [base, base + width) of t; elements past the width read 0.
  __device__ static __forceinline__ void raw(const Tensor& t, int64_t base, int64_t width, Raw (&r)[C]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      r[c] = Raw{};
      if (t.p != nullptr && chunk(c) < width) r[c] = load_raw<E>(t, base + at(c, width), width - chunk(c));
    }
  }
  __device__ static __forceinline__ void floats(const Raw (&r)[C], const Tensor& t, float (&v)[kN]) {
#pragma unroll
    for (int c = 0; c < C; ++c) to_float(r[c], t.f32, v + c * kVec);
  }
  __device__ static __forceinline__ void put(const Tensor& t, int64_t base, int64_t width, const float (&v)[kN]) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (chunk(c) < width) store<E>(t, base + at(c, width), width - chunk(c), v + c * kVec);
  }
  // Every thread has its part of the row before any thread stores over it: the
  // overlapping ends belong to two.
  __device__ static __forceinline__ void all_loaded() {
    if (E == kOverlap && T > kWave) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
  }
  // sum_e v_e w_e over the row's elements of this thread
  __device__ static __forceinline__ float dot(const float (&v)[kN], const float (&w)[kN], int64_t width) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < kN; ++e) s += counts(e, width) ? v[e] * w[e] : 0.0f;
    return s;
  }
  // Column values of a weight that may be absent (1).
  __device__ static __forceinline__ void weight(const Tensor& t, int64_t base, int64_t width, float (&v)[kN]) {
    if (t.p == nullptr) {
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = 1.0f;
      return;
    }
    Raw r[C];
    raw(t, base, width, r);
    floats(r, t, v);
  }
};

__device__ __forceinline__ int64_t gate_base(const NormArgs& a, int64_t row) {
  return a.gate_kind == kGateFull ? row * a.width : row / a.rows_per_gate * a.width;
}

template <class R>
__device__ __forceinline__ void gate_values(const NormArgs& a, int64_t row, float (&g)[R::kN]) {
  if (a.gate_kind == kGateRows) {
    const float v = scalar(a.gate, row);
#pragma unroll
    for (int e = 0; e < R::kN; ++e) g[e] = v;
  } else if (a.gate_kind == kGateNone) {
#pragma unroll
    for (int e = 0; e < R::kN; ++e) g[e] = 1.0f;
  } else {
    R::weight(a.gate, gate_base(a, row), a.width, g);
  }
}

// One row a workgroup.  Bound by its bytes from about 1,000 rows on: 2,048 x
// 4096, FP32 in and bf16 out, 10.9 us, 4.6 TB/s; 8,192 x 4096 bf16 behind a block
// 57 to 63 us, 4.3 to 4.7 TB/s (a 4 GiB copy: 4.7).  One row costs a launch and
// the way of two dependent sums, 5.2 us.
template <int T, int C, Ends E, bool POST>
__global__ __launch_bounds__(T) void norm_forward_kernel(NormArgs a, int64_t first) {
  using R = Row<T, C, E>;
  constexpr int N = R::kN;
  __shared__ float words[2][T / kWave];
  int turn = 0;
  const float inv_width = 1.0f / static_cast<float>(a.width);
  const int64_t row = first + blockIdx.x, base = row * a.width;
  Raw rx[C], ro[C];
  R::raw(a.residual, base, a.width, rx);
  if (POST) R::raw(a.out, base, a.width, ro);
  float x[N];
  R::floats(rx, a.residual, x);
  R::all_loaded();
  if (POST) {
    float o[N], g[N];
    R::floats(ro, a.out, o);
    gate_values<R>(a, row, g);
    float r_o = 1.0f;
    if (a.post_norm) {
      float p[N];
      R::weight(a.post, 0, a.width, p);
      r_o = 1.0f / sqrtf(row_sum<T>(R::dot(o, o, a.width), words, turn) * inv_width + a.eps);
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = o[e] * r_o * p[e];
    }
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] += a.scale * g[e] * o[e];
    R::put(a.new_residual, base, a.width, x);
    if (a.stats != nullptr && threadIdx.x == 0) a.stats[2 * row] = r_o;
  }
  if (a.y.p == nullptr) return;
  float w[N];
  R::weight(a.next, 0, a.width, w);
  const float r = 1.0f / sqrtf(row_sum<T>(R::dot(x, x, a.width), words, turn) * inv_width + a.eps);  // x past the width: 0
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = x[e] * r * w[e];
  R::put(a.y, base, a.width, x);
  if (a.stats != nullptr && threadIdx.x == 0) a.stats[2 * row + 1] = r;
}

// Rows [first, last) of backward workgroup `slice`, which lie in one gate group.
struct Slice {
  int64_t first, last;
};
__device__ __forceinline__ Slice slice_rows(int64_t rows, int64_t groups, int64_t slices, int64_t slice) {
  const int64_t per = rows / groups, each = slices / groups, chunk = (per + each - 1) / each;
  const int64_t g = slice / each, s = slice % each;
  const int64_t first = g * per + min(s * chunk, per);
  return {first, g * per + min((s + 1) * chunk, per)};
}

// Each workgroup takes a run of rows and keeps the column sums of d_post,
// d_gate (kGateColumns) and d_next in registers, written once as one row of
// fp32 partial sums: 3 width floats beside the six bf16 or fp32 rows of each row
// that it has, 16 of 8,192 x 4096 and one of 512 x 4096, where the sums, written
// and read again, are twice the tensors' bytes; a workgroup whose run begins past
// its group's last row writes zeros.  The order of the sums is the rows',
// whatever runs when.
// bf16 with all gradients, us without the join: 8,192 x 4096 85 to 96, 403 MB at
// 4.2 to 4.7 TB/s; 4,096 x 4096 49; 2,048 29; 512 17.  4,096 x 8192 120, 3.4 TB/s.
// Odd widths above 2,048 take 256 registers, one workgroup a CU: x 3001 72, x 5000
// 82.  Past 8,192 columns 1,024 threads have 128 registers each, and 178 (220
// in odd rows) of a thread's values spill: x 9001 602, x 12288 551, 1.1 TB/s, x
// 16384 637.
template <int T, int C, Ends E, bool POST>
__global__ __launch_bounds__(T) void norm_backward_kernel(NormArgs a, int64_t groups, int64_t slices) {
  using R = Row<T, C, E>;
  constexpr int N = R::kN;
  __shared__ float words[2][T / kWave];
  int turn = 0;
  const float inv_width = 1.0f / static_cast<float>(a.width);
  float s_next[N], s_post[N], s_gate[N];
#pragma unroll
  for (int e = 0; e < N; ++e) s_next[e] = s_post[e] = s_gate[e] = 0.0f;
  const Slice rows = slice_rows(a.rows, groups, slices, blockIdx.x);
  // The next row's tensors are on their way while a row is worked on (with two
  // loads a thread and tensor they would take the registers of half the
  // wavefronts).
  constexpr bool kAhead = C == 1;
  struct {
    Raw x[C], o[C], n[C], y[C];
    float r_o, r;
  } f;
  const auto fetch = [&](int64_t row) {
    const int64_t base = row * a.width;
    R::raw(a.residual, base, a.width, f.x);
    if (POST) R::raw(a.out, base, a.width, f.o);
    R::raw(a.d_new, base, a.width, f.n);
    R::raw(a.d_y, base, a.width, f.y);
    f.r_o = a.stats[2 * row];
    f.r = a.stats[2 * row + 1];
  };
  if (kAhead && rows.first < rows.last) fetch(rows.first);
  for (int64_t row = rows.first; row < rows.last; ++row) {
    const int64_t base = row * a.width;
    if (!kAhead) fetch(row);
    const float r_o = POST && a.post_norm ? f.r_o : 1.0f, r = f.r;
    float x[N], o[N], g[N], p[N], d[N], dy[N];
    R::floats(f.x, a.residual, x);
    R::floats(f.n, a.d_new, d);
    R::floats(f.y, a.d_y, dy);
    if (POST) R::floats(f.o, a.out, o);
    R::all_loaded();
    if (kAhead && row + 1 < rows.last) fetch(row + 1);
    if (POST) {
      gate_values<R>(a, row, g);
      R::weight(a.post, 0, a.width, p);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        o[e] *= r_o;
        x[e] += a.scale * g[e] * (o[e] * p[e]);
      }
    }
    if (a.d_y.p != nullptr) {
      float w[N];
      R::weight(a.next, 0, a.width, w);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x[e] *= r;
        s_next[e] += dy[e] * x[e];
        dy[e] *= w[e];
      }
      const float m = row_sum<T>(R::dot(dy, x, a.width), words, turn) * inv_width;
#pragma unroll
      for (int e = 0; e < N; ++e) d[e] += r * (dy[e] - x[e] * m);
    }
    if (a.d_residual.p != nullptr) R::put(a.d_residual, base, a.width, d);
    if (!POST) continue;
    if (a.d_gate.p != nullptr) {
      float dg[N];
#pragma unroll
      for (int e = 0; e < N; ++e) dg[e] = a.scale * (o[e] * p[e]) * d[e];
      if (a.gate_kind == kGateColumns) {
#pragma unroll
        for (int e = 0; e < N; ++e) s_gate[e] += dg[e];
      } else if (a.gate_kind == kGateFull) {
        R::put(a.d_gate, base, a.width, dg);
      } else {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) sum += R::counts(e, a.width) ? dg[e] : 0.0f;
        sum = row_sum<T>(sum, words, turn);
        if (threadIdx.x == 0) store_one(a.d_gate, row, sum);
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) d[e] *= a.scale * g[e];
    if (a.post_norm) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        s_post[e] += d[e] * o[e];
        d[e] *= p[e];
      }
      const float m = row_sum<T>(R::dot(d, o, a.width), words, turn) * inv_width;
#pragma unroll
      for (int e = 0; e < N; ++e) d[e] = r_o * (d[e] - o[e] * m);
    }
    if (a.d_out.p != nullptr) R::put(a.d_out, base, a.width, d);
  }
  const Tensor part = {a.partial, true};
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kNormSums * a.width;
  if (a.d_next.p != nullptr) R::put(part, at, a.width, s_next);
  if (a.d_post.p != nullptr) R::put(part, at + a.width, a.width, s_post);
  if (a.d_gate.p != nullptr && a.gate_kind == kGateColumns) R::put(part, at + 2 * a.width, a.width, s_gate);
}

// Adds the partial rows: out[v][column] = sum over rows first_v .. of sum v,
// blockIdx.y = 0 d_next, 1 d_post, 2 + g d_gate of gate group g.  16 row
// slices of 64 columns a workgroup, joined in LDS in their order.  512 slices of
// 4096 columns: 5.4 us.
constexpr int kJoin = 16;
__global__ __launch_bounds__(kWave* kJoin) void norm_join_kernel(NormArgs a, int64_t groups, int64_t slices) {
  __shared__ float part[kJoin][kWave];
  const int v = blockIdx.y < 2 ? blockIdx.y : 2;
  const Tensor out = v == 0 ? a.d_next : v == 1 ? a.d_post : a.d_gate;
  if (out.p == nullptr || (v == 2 && a.gate_kind != kGateColumns)) return;
  const int64_t each = slices / groups, g = v == 2 ? blockIdx.y - 2 : 0;
  const int64_t first = v == 2 ? g * each : 0, count = v == 2 ? each : slices;
  const int lane = threadIdx.x & (kWave - 1), slot = threadIdx.x / kWave;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kWave + lane;
  float sum = 0.0f;
  if (col < a.width)
#pragma unroll 8
    for (int64_t s = slot; s < count; s += kJoin) sum += a.partial[((first + s) * kNormSums + v) * a.width + col];
  part[slot][lane] = sum;
  __syncthreads();
  if (slot != 0 || col >= a.width) return;
  sum = part[0][lane];
#pragma unroll
  for (int i = 1; i < kJoin; ++i) sum += part[i][lane];
  store_one(out, g * a.width + col, sum);
}

template <int T, int C, Ends E>
hipError_t launch_shape(const NormArgs& a, bool backward, int64_t groups, int64_t slices, hipStream_t st) {
  const bool post = a.out.p != nullptr;
  if (!backward) {
    constexpr int64_t kMost = (int64_t{1} << 31) / T;  // a grid has fewer than 2^32 threads
    for (int64_t first = 0; first < a.rows; first += kMost) {
      const dim3 grid(static_cast<uint32_t>(a.rows - first < kMost ? a.rows - first : kMost));
      if (post)
        norm_forward_kernel<T, C, E, true><<<grid, T, 0, st>>>(a, first);
      else
        norm_forward_kernel<T, C, E, false><<<grid, T, 0, st>>>(a, first);
    }
  } else {
    const dim3 grid(static_cast<uint32_t>(slices));
    if (post)
      norm_backward_kernel<T, C, E, true><<<grid, T, 0, st>>>(a, groups, slices);
    else
      norm_backward_kernel<T, C, E, false><<<grid, T, 0, st>>>(a, groups, slices);
  }
  return hipGetLastError();
}

// Threads a row, so that each holds one or two loads of every tensor: more
// threads leave lanes without elements, more loads a thread take the registers
// of half the wavefronts.  Narrow rows on 64 and 128 threads, the next row read
// ahead, against 256 threads: 8,192 x 256 backward 46 -> 25 us, x 1,024 59 -> 38.
int row_threads(int64_t width) { return width <= 512 ? 64 : width <= 1024 ? 128 : width <= 4096 ? 256 : width <= 8192 ? 512 : 1024; }

template <Ends E>
hipError_t launch_any(const NormArgs& a, bool backward, int64_t groups, int64_t slices, hipStream_t st) {
  switch (row_threads(a.width)) {
    case 64: return launch_shape<64, 1, E>(a, backward, groups, slices, st);
    case 128: return launch_shape<128, 1, E>(a, backward, groups, slices, st);
    case 256:
      if (a.width <= 2048) return launch_shape<256, 1, E>(a, backward, groups, slices, st);
      return launch_shape<256, 2, E>(a, backward, groups, slices, st);
    case 512: return launch_shape<512, 2, E>(a, backward, groups, slices, st);
    default: return launch_shape<1024, 2, E>(a, backward, groups, slices, st);
  }
}

hipError_t launch(const NormArgs& a, bool backward, int64_t groups, int64_t slices, hipStream_t st) {
  if (a.width < kVec) return launch_shape<64, 1, kSingly>(a, backward, groups, slices, st);
  return a.width % kVec ? launch_any<kOverlap>(a, backward, groups, slices, st) : launch_any<kWhole>(a, backward, groups, slices, st);
}

// Workgroups of 256 threads or more: two a CU, where 256 threads have 218
// registers each; odd rows, and the 512 and 1,024 threads of wider ones, are one
// a CU at a time.
constexpr int64_t kNormSlices = 512;

int64_t gate_groups(const NormArgs& a) {
  return a.gate_kind == kGateColumns && a.rows > 0 ? a.rows / a.rows_per_gate : 1;
}

}  // namespace

int64_t norm_slices(int64_t rows, int64_t groups, int64_t width) {
  const int64_t per = rows / groups, threads = row_threads(width);
  const int64_t each = (threads < 256 ? kNormSlices * 256 / threads : kNormSlices) / groups;
  return groups * (each < 1 ? 1 : each > per ? per : each);
}

hipError_t launch_norm_forward(const NormArgs& a, hipStream_t st) { return launch(a, false, 1, 1, st); }

hipError_t launch_norm_backward(const NormArgs& a, hipStream_t st) {
  const int64_t groups = gate_groups(a), slices = norm_slices(a.rows, groups, a.width);
  if (slices > 0)  // without rows the sums are zero
    if (hipError_t e = launch(a, true, groups, slices, st); e != hipSuccess) return e;
  const bool gates = a.d_gate.p != nullptr && a.gate_kind == kGateColumns;
  if (a.d_next.p == nullptr && a.d_post.p == nullptr && !gates) return hipSuccess;
  const dim3 grid(static_cast<uint32_t>((a.width + kWave - 1) / kWave), static_cast<uint32_t>(2 + (gates ? groups : 0)));
  norm_join_kernel<<<grid, kWave * kJoin, 0, st>>>(a, groups, slices);
  return hipGetLastError();
}

}  // namespace glm53
