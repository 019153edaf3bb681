// Norms before and after a block: argument blocks and launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace glm53 {

// A bf16 or fp32 tensor.
struct Tensor {
  void* p;
  bool f32;
};

enum GateKind : int { kGateNone = 0, kGateColumns = 1, kGateRows = 2, kGateFull = 3 };

// residual_norm over rows of `width`, and rms_norm where out.p is null.
// Null tensors are absent: post (no norm of out), gate, next (weight 1) and y
// (no norm of the new residual).
struct NormArgs {
  Tensor residual;  // [rows, width]
  Tensor out;       // [rows, width]
  Tensor post;      // [width]
  Tensor gate;      // kGateColumns: [rows / rows_per_gate, width], kGateRows: [rows], kGateFull: [rows, width]
  Tensor next;      // [width]
  GateKind gate_kind;
  bool post_norm;   // norm of out, whether or not post is given
  int64_t rows_per_gate;
  float scale, eps;
  int64_t rows, width;
  Tensor new_residual;  // [rows, width], residual's type
  Tensor y;             // [rows, width]
  float* stats;         // [rows, 2]: 1 / rms of out and of the new residual; null in a forward that keeps none
  // backward: gradients given (null: zero) and wanted (null: not written)
  Tensor d_new, d_y;
  Tensor d_residual, d_out, d_post, d_gate, d_next;
  float* partial;       // [norm_slices, kNormSums, width]
};

constexpr int64_t kNormMaxWidth = 16384;  // rows whose values a workgroup holds in registers

// Workgroups of a backward pass over `rows` rows in `groups` equal groups,
// each writing one row of kNormSums column sums.
int64_t norm_slices(int64_t rows, int64_t groups, int64_t width);
constexpr int kNormSums = 3;

hipError_t launch_norm_forward(const NormArgs& a, hipStream_t st);
hipError_t launch_norm_backward(const NormArgs& a, hipStream_t st);

}  // namespace glm53
