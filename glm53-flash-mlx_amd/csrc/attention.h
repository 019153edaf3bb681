// Attention over packed sequences and its gradients: argument block and launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace glm53 {

constexpr int64_t kMaxHeadDim = 256;
// Elements from one token, or one head, to the next: a tile's rows lie within
// 32-bit byte offsets of its first one.
constexpr int64_t kMaxRowStride = int64_t{1} << 22;
constexpr int64_t kMaxHeadSpan = int64_t{1} << 30;  // a token's heads, together

// Rows of one head each: element d of head h of token t at p + t * token + h * head + d.
struct Rows16 {
  const uint16_t* p;
  int64_t token, head;
};

// Queries [tokens, kv_heads * group], keys and values [keys, kv_heads], rows
// of `dim`; query head h reads key head h / group.  Sequence s holds queries
// offsets[s] .. offsets[s + 1] - 1 and keys key_offsets[s] .. ; no offsets: all
// of them are one sequence.
struct AttentionArgs {
  Rows16 q, k, v;
  const int32_t* offsets;      // [sequences + 1] or null
  const int32_t* key_offsets;  // [sequences + 1] or null
  int64_t tokens, keys;
  int sequences, kv_heads, group, dim;
  bool causal;                 // query i of n sees keys up to i + (keys of the sequence) - n
  float scale;
  uint16_t* out;               // [tokens, heads, dim]
  float* lse;                  // [kv_heads, tokens * group]: log2 of each row's sum of 2^(score log2 e); null: not kept
  // backward
  Rows16 d_out;
  uint16_t *d_q, *d_k, *d_v;   // contiguous; null: not wanted
  float* starts;               // [2, kv_heads, tokens * group]: -lse / (scale log2 e), -delta
  int splits;                  // of the rows that a workgroup of d_k and d_v takes
  float* sums;                 // [splits, keys, kv_heads, dim] of d_k, then the same of d_v; where splits > 1
};

// Into how many parts the rows of one tile of keys are best cut, at most: each has
// kLeastTurns turns of a workgroup.
constexpr int kLeastTurns = 16;
int attention_row_splits(const AttentionArgs& a);

hipError_t launch_attention(const AttentionArgs& a, hipStream_t st);
hipError_t launch_attention_backward(const AttentionArgs& a, hipStream_t st);
// The same for heads of more than 128 values.
hipError_t launch_attention_wide(const AttentionArgs& a, hipStream_t st);
hipError_t launch_attention_backward_wide(const AttentionArgs& a, hipStream_t st);

}  // namespace glm53
