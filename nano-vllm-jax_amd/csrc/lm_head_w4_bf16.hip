// LM head with 4-bit weights (lm_head_w4.h): bf16 activations.
#include "lm_head_w4.h"

namespace nvjsel {

template <int MODE>
static int pass(const W4Args& a, int group, hipStream_t s) {
  if (a.B <= 16) return launch_w4_group<DT_BF16, 1, 1, MODE>(a, group, s);
  if (a.B <= 32) return launch_w4_group<DT_BF16, 1, 2, MODE>(a, group, s);
  return launch_w4_group<DT_BF16, 1, 4, MODE>(a, group, s);
}

int w4_pass_bf16(int mode, const W4Args& a, int group, hipStream_t s) {
  return mode == MODE_GREEDY ? pass<MODE_GREEDY>(a, group, s) : pass<MODE_LOGITS>(a, group, s);
}

}  // namespace nvjsel
