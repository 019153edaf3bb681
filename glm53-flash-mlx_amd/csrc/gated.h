// Gated MLP in bf16 weights: argument block and launchers of its products.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace glm53 {

struct GatedArgs {
  const uint16_t* x;      // [rows, hidden]
  const uint16_t* wg;     // [inter, hidden]
  const uint16_t* wu;     // [inter, hidden]
  const uint16_t* wd;     // [hidden, inter]
  int64_t rows, hidden, inter;
  float limit;            // +inf: no clamp
  uint16_t* y;            // [rows, hidden]
  float* gate;            // [rows, inter] kept for the gradient, or null
  float* up;
  uint16_t* h;            // [rows, inter] kept with them; up to 16 rows [2, rows, inter], high and low parts
  // backward: gradients that are not wanted are null
  const uint16_t* dy;
  uint16_t* dx;
  uint16_t* d_wg;
  uint16_t* d_wu;
  uint16_t* d_wd;
  void* space;            // workspace of gated_space bytes or more, 256-byte aligned
  size_t space_bytes;
};

size_t gated_space(int64_t rows, int64_t hidden, int64_t inter, bool backward);
hipError_t launch_gated(const GatedArgs& a, hipStream_t st);
hipError_t launch_gated_backward(const GatedArgs& a, hipStream_t st);

}  // namespace glm53
