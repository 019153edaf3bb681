// Linear with 4-bit weights and group scales: argument block and launcher.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace glm53 {

struct Int4Args {
  const uint16_t* x;      // [rows, K] bf16
  const uint8_t* codes;   // [N, K / 2], even k in the low half
  const void* scales;     // [N, K / group]
  const void* offsets;    // or null: -8 scale
  const void* bias;       // [N] or null
  bool tables_f32;        // scales, offsets and bias are FP32, not bf16
  int group_log2;         // 5, 6 or 7
  int64_t rows, N, K;
  uint16_t* y;            // [rows, N]
  void* space;            // int4_space bytes or more
  size_t space_bytes;
};

size_t int4_space(int64_t rows, int64_t N, int64_t K);
hipError_t launch_int4(const Int4Args& a, hipStream_t st);

}  // namespace glm53
