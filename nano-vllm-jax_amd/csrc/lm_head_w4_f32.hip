// LM head with 4-bit weights (lm_head_w4.h): f32 activations, as three bf16 terms.
#include "lm_head_w4.h"

namespace nvjsel {

template <int MODE>
static int pass(const W4Args& a, int group, hipStream_t s) {
  if (a.B <= 16) return launch_w4_group<DT_BF16, 3, 1, MODE>(a, group, s);
  return launch_w4_group<DT_BF16, 3, 2, MODE>(a, group, s);
}

int w4_pass_f32(int mode, const W4Args& a, int group, hipStream_t s) {
  return mode == MODE_GREEDY ? pass<MODE_GREEDY>(a, group, s) : pass<MODE_LOGITS>(a, group, s);
}

}  // namespace nvjsel
