// C ABI of the dense feed-forward block (declared in include/glm53_moe.h):
// the norms around it, the gated MLP and the 4-bit linear.
#include "api_util.h"
#include "gated.h"
#include "int4.h"
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
int norm_args(const glm53_norm* n, bool backward, NormArgs& a) {
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
    const auto over = [](const Tensor& result, const Tensor& input) {
      return result.p != nullptr && result.p == input.p && result.f32 != input.f32;
    };
    CHECK_ARG(!over(a.new_residual, a.out) && !over(a.y, a.out) && !over(a.y, a.residual),
              "a result in an input's place must have its type");
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
  return GLM53_OK;
}

}  // namespace

extern "C" {

size_t glm53_residual_norm_workspace_bytes(int64_t rows, int64_t width, int64_t gate_rows) {
  if (rows <= 0 || width <= 0 || gate_rows <= 0 || gate_rows > rows) return 0;
  return sizeof(float) * static_cast<size_t>(norm_slices(rows, gate_rows, width)) * kNormSums * static_cast<size_t>(width);
}

int glm53_residual_norm(const glm53_norm* norm, void* stream) {
  NormArgs a;
  if (int rc = norm_args(norm, false, a)) return rc;
  if (a.rows == 0) return GLM53_OK;
  HIP_TRY(launch_norm_forward(a, S(stream)), "norm launch");
  return GLM53_OK;
}

int glm53_residual_norm_backward(const glm53_norm* norm, void* stream) {
  NormArgs a;
  if (int rc = norm_args(norm, true, a)) return rc;
  HIP_TRY(launch_norm_backward(a, S(stream)), "norm gradient launch");
  return GLM53_OK;
}

}  // extern "C"

// ----------------------------------------------------------- gated MLP ----

namespace {

constexpr int64_t kGatedMaxWidth = int64_t{1} << 22;  // 256 rows of a tile within 32-bit byte offsets

int gated_args(const glm53_gated_mlp_desc* d, GatedArgs& a) {
  CHECK_ARG(d != nullptr, "gated MLP descriptor is null");
  CHECK_ARG(d->rows >= 0 && d->rows < (int64_t{1} << 31) && d->hidden > 0 && d->intermediate > 0,
            "invalid shape rows=%lld hidden=%lld intermediate=%lld", (long long)d->rows, (long long)d->hidden,
            (long long)d->intermediate);
  CHECK_ARG(d->hidden % 8 == 0 && d->intermediate % 8 == 0, "hidden %lld and intermediate %lld must be multiples of 8",
            (long long)d->hidden, (long long)d->intermediate);
  CHECK_ARG(d->hidden <= kGatedMaxWidth && d->intermediate <= kGatedMaxWidth, "widths above %lld",
            (long long)kGatedMaxWidth);
  CHECK_ARG(d->limit > 0.0f, "limit must be positive (infinity: no clamp)");
  a = GatedArgs{};
  a.x = static_cast<const uint16_t*>(d->x);
  a.wg = static_cast<const uint16_t*>(d->gate_weight);
  a.wu = static_cast<const uint16_t*>(d->up_weight);
  a.wd = static_cast<const uint16_t*>(d->down_weight);
  a.rows = d->rows;
  a.hidden = d->hidden;
  a.inter = d->intermediate;
  a.limit = d->limit;
  a.y = static_cast<uint16_t*>(d->y);
  a.gate = d->gate;
  a.up = d->up;
  a.h = static_cast<uint16_t*>(d->h);
  a.dy = static_cast<const uint16_t*>(d->d_y);
  a.dx = static_cast<uint16_t*>(d->d_x);
  a.d_wg = static_cast<uint16_t*>(d->d_gate_weight);
  a.d_wu = static_cast<uint16_t*>(d->d_up_weight);
  a.d_wd = static_cast<uint16_t*>(d->d_down_weight);
  a.space = d->workspace;
  a.space_bytes = d->workspace_bytes;
  const void* every[] = {a.x, a.wg, a.wu, a.wd, a.y, a.gate, a.up, a.h, a.dy, a.dx, a.d_wg, a.d_wu, a.d_wd};
  for (const void* p : every) CHECK_ARG(aligned(p, 16), "gated MLP tensors must be 16-byte aligned");
  CHECK_ARG((a.gate == nullptr) == (a.up == nullptr) && (a.gate == nullptr) == (a.h == nullptr),
            "gate, up and h are kept together");
  return GLM53_OK;
}

}  // namespace

extern "C" {

size_t glm53_gated_mlp_workspace_bytes(int64_t rows, int64_t hidden, int64_t intermediate) {
  if (rows <= 0 || hidden <= 0 || intermediate <= 0) return 0;
  return gated_space(rows, hidden, intermediate, false);
}

size_t glm53_gated_mlp_backward_workspace_bytes(int64_t rows, int64_t hidden, int64_t intermediate) {
  if (rows <= 0 || hidden <= 0 || intermediate <= 0) return 0;
  return gated_space(rows, hidden, intermediate, true);
}

int glm53_gated_mlp(const glm53_gated_mlp_desc* desc, void* stream) {
  GatedArgs a;
  if (int rc = gated_args(desc, a)) return rc;
  if (a.rows == 0) return GLM53_OK;
  CHECK_ARG(a.x && a.wg && a.wu && a.wd && a.y, "null pointer argument");
  const size_t need = glm53_gated_mlp_workspace_bytes(a.rows, a.hidden, a.inter);
  CHECK_ARG(a.space && desc->workspace_bytes >= need && aligned(a.space, 256),
            "the gated MLP needs a 256-byte aligned workspace of %zu bytes", need);
  HIP_TRY(launch_gated(a, S(stream)), "gated MLP launch");
  return GLM53_OK;
}

int glm53_gated_mlp_backward(const glm53_gated_mlp_desc* desc, void* stream) {
  GatedArgs a;
  if (int rc = gated_args(desc, a)) return rc;
  CHECK_ARG(a.rows > 0, "gradients of an MLP over no rows are zero: nothing to compute");
  CHECK_ARG(a.x && a.wg && a.wu && a.wd && a.gate && a.up && a.dy, "null pointer argument");
  const size_t need = glm53_gated_mlp_backward_workspace_bytes(a.rows, a.hidden, a.inter);
  CHECK_ARG(a.space && desc->workspace_bytes >= need && aligned(a.space, 256),
            "the gated MLP's gradients need a 256-byte aligned workspace of %zu bytes", need);
  HIP_TRY(launch_gated_backward(a, S(stream)), "gated MLP gradient launch");
  return GLM53_OK;
}

}  // extern "C"

// --------------------------------------------------------- 4-bit linear ---

extern "C" {

size_t glm53_int4_linear_workspace_bytes(int64_t rows, int64_t out_features, int64_t in_features) {
  if (rows <= 0 || out_features <= 0 || in_features <= 0) return 0;
  return int4_space(rows, out_features, in_features);
}

int glm53_int4_linear(const glm53_int4_weight* w, const void* x, int64_t rows, void* y, void* workspace,
                      size_t workspace_bytes, void* stream) {
  CHECK_ARG(w != nullptr, "4-bit weight is null");
  const int64_t N = w->out_features, K = w->in_features;
  CHECK_ARG(rows >= 0 && rows < (int64_t{1} << 31) && N > 0 && K > 0, "invalid shape rows=%lld out=%lld in=%lld",
            (long long)rows, (long long)N, (long long)K);
  CHECK_ARG(w->group == 32 || w->group == 64 || w->group == 128, "group must be 32, 64 or 128, got %d", w->group);
  CHECK_ARG(K % w->group == 0, "in_features %lld is not a multiple of the group %d", (long long)K, w->group);
  CHECK_ARG(K <= kGatedMaxWidth && N <= kGatedMaxWidth, "weight too large: widths above %lld", (long long)kGatedMaxWidth);
  if (rows == 0) return GLM53_OK;
  CHECK_ARG(w->codes && w->scales && x && y, "null pointer argument");
  CHECK_ARG(aligned(w->codes, 16) && aligned(x, 16) && aligned(y, 16), "codes, x and y must be 16-byte aligned");
  const size_t need = glm53_int4_linear_workspace_bytes(rows, N, K);
  CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 256)),
            "the 4-bit linear needs a 256-byte aligned workspace of %zu bytes", need);
  Int4Args a{};
  a.x = static_cast<const uint16_t*>(x);
  a.codes = w->codes;
  a.scales = w->scales;
  a.offsets = w->offsets;
  a.bias = w->bias;
  a.tables_f32 = w->tables_f32 != 0;
  a.group_log2 = w->group == 32 ? 5 : w->group == 64 ? 6 : 7;
  a.rows = rows;
  a.N = N;
  a.K = K;
  a.y = static_cast<uint16_t*>(y);
  a.space = workspace;
  a.space_bytes = workspace_bytes;
  HIP_TRY(launch_int4(a, S(stream)), "4-bit linear launch");
  return GLM53_OK;
}

}  // extern "C"
