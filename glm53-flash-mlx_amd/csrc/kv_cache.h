// A paged key-value cache: writing, reading back, and one token's attention
// over it.  Argument blocks and launchers.
#pragma once

#include "attention.h"

namespace glm53 {

// Row (page, head, token) of a page at ((page * kv_heads + head) << page_log2) + token.
struct CacheArgs {
  uint8_t *k, *v;              // bf16 or E4M3 rows of `dim`
  uint8_t *k_scales, *v_scales;  // one byte a row, 127 + e; null in a bf16 cache
  const int32_t* table;        // [sequences, table_stride]
  int64_t pages, table_stride;
  int sequences, max_pages, kv_heads, dim, page_log2;
  bool e4m3;
};

struct AppendArgs {
  CacheArgs cache;
  Rows16 rows_k, rows_v;
  int64_t tokens;
  const int32_t* offsets;  // null: one token a sequence
  const int32_t* lengths;
};

struct ReadArgs {
  CacheArgs cache;
  const int32_t* offsets;
  int64_t rows;
  uint16_t *k, *v;  // [rows, kv_heads, dim]; null: not wanted
};

struct DecodeArgs {
  CacheArgs cache;
  Rows16 q;              // [sequences, kv_heads * group]
  const int32_t* lengths;
  int group;
  float scale;
  uint16_t* out;         // [sequences, kv_heads * group, dim]
  float* partial;        // decode_space bytes
};

hipError_t launch_append(const AppendArgs& a, hipStream_t st);
hipError_t launch_read(const ReadArgs& a, hipStream_t st);
size_t decode_space(int dim, bool e4m3);
hipError_t launch_decode(const DecodeArgs& a, hipStream_t st);

}  // namespace glm53
