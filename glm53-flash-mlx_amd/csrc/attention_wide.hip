// Attention over heads of more than 128 values: a translation unit of its own, as its
// kernels, of up to 512 registers, take as long to compile as all of the others.
#include "attention_kernels.h"

namespace glm53 {

hipError_t launch_attention_wide(const AttentionArgs& a, hipStream_t st) {
  if (a.dim == 256) return launch_forward<Forward<256, true>>(a, st);
  return launch_forward<Forward<256, false>>(a, st);
}

hipError_t launch_attention_backward_wide(const AttentionArgs& a, hipStream_t st) {
  if (a.dim == 256) return backward<256, true, 1>(a, st);
  return backward<256, false, 1>(a, st);
}

}  // namespace glm53
