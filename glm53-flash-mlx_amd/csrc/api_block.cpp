// C ABI of the dense feed-forward block (declared in include/glm53_moe.h):
// the norms around it.
#include "api_util.h"
#include "norms.h"

using namespace glm53;

// -------------------------------------------------------------- norms -----

namespace {

// Elements of gate rows a norm's column sums are kept apart for; 1 where the
// gate has one row, and where it has none.
int64_t gate_groups(const glm53_norm* n) {
  return n->gate_kind == GLM53_GATE_COLUMNS && n->rows > 0 ? n->rows / n->rows_per_gate : 1;
}

// Checks a descriptor and makes the kernels' argument block of it.
int norm_args(const glm53_norm* n, bool backward, NormArgs& a, bool& vec) {
  CHECK_ARG(n != nullptr, "norm descriptor is null");
  CHECK_ARG(n->rows >= 0 && n->rows < (int64_t{1} << 31) && n->width > 0, "invalid shape rows=%lld width=%lld",
            (long long)n->rows, (long long)n->width);
  CHECK_ARG(n->width <= kNormMaxWidth, "width %lld exceeds %lld", (long long)n->width, (long long)kNormMaxWidth);
  CHECK_ARG(n->eps >= 0.0f, "eps must not be negative");
  CHECK_ARG((n->f32_mask & ~63) == 0, "unknown bits in f32_mask");
  CHECK_ARG(n->gate_kind >= GLM53_GATE_NONE && n->gate_kind <= GLM53_GATE_FULL, "unknown gate kind %d", n->gate_kind);
  CHECK_ARG((n->gate != nullptr) == (n->gate_kind != GLM53_GATE_NONE), "gate and gate_kind disagree");
  CHECK_ARG(n->out != nullptr || (n->gate == nullptr && n->post_weight == nullptr && !n->post_norm),
            "a norm without a block output has no gate and no post norm");
  CHECK_ARG(n->post_norm || n->post_weight == nullptr, "post_weight without post_norm");
  if (n->gate_kind == GLM53_GATE_COLUMNS && n->rows > 0) {
    CHECK_ARG(n->rows_per_gate > 0 && n->rows % n->rows_per_gate == 0, "rows_per_gate %lld does not divide %lld rows",
              (long long)n->rows_per_gate, (long long)n->rows);
    CHECK_ARG(gate_groups(n) <= 65533, "more than 65533 gate rows");
  }
  const auto tensor = [&](const void* p, int bit) { return Tensor{const_cast<void*>(p), (n->f32_mask & bit) != 0}; };
  a = NormArgs{};
  a.residual = tensor(n->residual, GLM53_NORM_F32_RESIDUAL);
  a.out = tensor(n->out, GLM53_NORM_F32_OUT);
  a.post = tensor(n->post_weight, GLM53_NORM_F32_POST);
  a.gate = tensor(n->gate, GLM53_NORM_F32_GATE);
  a.next = tensor(n->next_weight, GLM53_NORM_F32_NEXT);
  a.gate_kind = static_cast<GateKind>(n->gate_kind);
  a.post_norm = n->post_norm != 0;
  a.rows_per_gate = n->gate_kind == GLM53_GATE_COLUMNS ? n->rows_per_gate : 1;
  a.scale = n->scale;
  a.eps = n->eps;
  a.rows = n->rows;
  a.width = n->width;
  a.stats = n->stats;
  if (!backward) {
    a.new_residual = tensor(n->out != nullptr ? n->new_residual : nullptr, GLM53_NORM_F32_RESIDUAL);
    a.y = tensor(n->y, GLM53_NORM_F32_Y);
    CHECK_ARG(n->rows == 0 || (a.residual.p && (n->out == nullptr || a.new_residual.p)), "null pointer argument");
    CHECK_ARG(n->out != nullptr || n->y != nullptr, "nothing to compute: neither a block output nor y");
  } else {
    a.d_new = tensor(n->d_new_residual, GLM53_NORM_F32_RESIDUAL);
    a.d_y = tensor(n->d_y, GLM53_NORM_F32_Y);
    a.d_residual = tensor(n->d_residual, GLM53_NORM_F32_RESIDUAL);
    a.d_out = tensor(n->d_out, GLM53_NORM_F32_OUT);
    a.d_post = tensor(n->d_post_weight, GLM53_NORM_F32_POST);
    a.d_gate = tensor(n->d_gate, GLM53_NORM_F32_GATE);
    a.d_next = tensor(n->d_next_weight, GLM53_NORM_F32_NEXT);
    CHECK_ARG(n->rows == 0 || (a.residual.p && a.stats), "null pointer argument");
    CHECK_ARG(a.d_gate.p == nullptr || n->gate != nullptr, "d_gate without a gate");
    CHECK_ARG(a.d_post.p == nullptr || n->post_norm, "d_post_weight without a post norm");
    CHECK_ARG(a.d_out.p == nullptr || n->out != nullptr, "d_out without a block output");
    const size_t need = glm53_residual_norm_workspace_bytes(n->rows, n->width, gate_groups(n));
    CHECK_ARG(need == 0 || (n->workspace && n->workspace_bytes >= need && aligned(n->workspace, 16)),
              "norm gradients need a 16-byte aligned workspace of %zu bytes", need);
    a.partial = static_cast<float*>(n->workspace);
  }
  const void* every[] = {a.residual.p, a.out.p, a.post.p, a.gate_kind == kGateRows ? nullptr : a.gate.p, a.next.p,
                         a.new_residual.p, a.y.p, a.d_new.p, a.d_y.p, a.d_residual.p, a.d_out.p};
  vec = n->width % 8 == 0;
  for (const void* p : every) vec = vec && aligned(p, 16);
  if (a.gate_kind != kGateRows) vec = vec && aligned(a.d_gate.p, 16);
  CHECK_ARG(vec || n->width <= kNormMaxScalarWidth,
            "a width above %lld must be a multiple of 8 with 16-byte aligned tensors", (long long)kNormMaxScalarWidth);
  return GLM53_OK;
}

}  // namespace

extern "C" {

size_t glm53_residual_norm_workspace_bytes(int64_t rows, int64_t width, int64_t gate_rows) {
  if (rows <= 0 || width <= 0 || gate_rows <= 0 || gate_rows > rows) return 0;
  return sizeof(float) * static_cast<size_t>(norm_slices(rows, gate_rows)) * kNormSums * static_cast<size_t>(width);
}

int glm53_residual_norm(const glm53_norm* norm, void* stream) {
  NormArgs a;
  bool vec;
  if (int rc = norm_args(norm, false, a, vec)) return rc;
  if (a.rows == 0) return GLM53_OK;
  HIP_TRY(launch_norm_forward(a, vec, S(stream)), "norm launch");
  return GLM53_OK;
}

int glm53_residual_norm_backward(const glm53_norm* norm, void* stream) {
  NormArgs a;
  bool vec;
  if (int rc = norm_args(norm, true, a, vec)) return rc;
  HIP_TRY(launch_norm_backward(a, vec, S(stream)), "norm gradient launch");
  return GLM53_OK;
}

}  // extern "C"
