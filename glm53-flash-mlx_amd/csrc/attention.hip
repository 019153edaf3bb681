// Attention over heads of up to 128 values.
#include "attention_kernels.h"

namespace glm53 {

hipError_t launch_attention(const AttentionArgs& a, hipStream_t st) {
  if (a.dim > 128) return launch_attention_wide(a, st);
  if (a.dim == 128) return launch_forward<Forward<128, true, 4>>(a, st);
  if (a.dim == 64) return launch_forward<Forward<64, true, 4>>(a, st);
  if (a.dim > 64) return launch_forward<Forward<128, false, 4>>(a, st);
  return launch_forward<Forward<64, false, 4>>(a, st);
}

hipError_t launch_attention_backward(const AttentionArgs& a, hipStream_t st) {
  if (a.dim > 128) return launch_attention_backward_wide(a, st);
  if (a.dim == 128) return backward<128, true, 2>(a, st);
  if (a.dim == 64) return backward<64, true, 2>(a, st);
  if (a.dim > 64) return backward<128, false, 2>(a, st);
  return backward<64, false, 2>(a, st);
}

}  // namespace glm53
