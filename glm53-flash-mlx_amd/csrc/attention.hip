// Attention over heads of up to 128 values.
#include "attention_kernels.h"

namespace glm53 {

hipError_t launch_attention(const AttentionArgs& a, hipStream_t st) {
  if (a.dim > 128) return launch_attention_wide(a, st);
  if (a.dim == 128) return launch_forward<Forward<128, true>>(a, st);
  if (a.dim == 64) return launch_forward<Forward<64, true>>(a, st);
  if (a.dim > 64) return launch_forward<Forward<128, false>>(a, st);
  return launch_forward<Forward<64, false>>(a, st);
}

int attention_row_splits(const AttentionArgs& a) {
  // Up to 1,024 workgroups of 64 keys and all of a sequence's rows, 128 (of more than 128
  // columns 64) a turn: with fewer than one a CU, and causal ones among them of different
  // lengths, the card waits for the longest.  All gradients of causal tokens, in us, split
  // and not: 8,192 of 8 / 1 heads of 128 684 and 1,296, 16,384 2,259 and 3,147, 2 x 2,693 of
  // 16 / 2 heads of 256 808 and 1,265, 4,096 of 16 / 4 heads of 128 (256 tiles) 405 and 423,
  // of 16 / 8 (512, in two) 380 and 316; heads of 64, two workgroups a CU: 8,192 of 16 / 4
  // (512 tiles) 566 and 622.  Sequences too short for two parts pay for
  // parts that are 0, so that few turns a sequence are not split.
  const int64_t tiles = (a.keys + 63) / 64 * a.kv_heads, turns = a.tokens * a.group / (a.dim > 128 ? 64 : 128);
  if (tiles == 0 || tiles > (a.dim <= 64 ? 512 : 256) || turns < 20 * a.sequences) return 1;
  const int64_t most = turns / kLeastTurns < 16 ? turns / kLeastTurns : 16, splits = 1024 / tiles;
  return static_cast<int>(splits < most ? splits : most < 1 ? 1 : most);
}

hipError_t launch_attention_backward(const AttentionArgs& a, hipStream_t st) {
  if (a.dim > 128) return launch_attention_backward_wide(a, st);
  if (a.dim == 128) return backward<128, true, 2>(a, st);
  if (a.dim == 64) return backward<64, true, 2>(a, st);
  if (a.dim > 64) return backward<128, false, 2>(a, st);
  return backward<64, false, 2>(a, st);
}

}  // namespace glm53
