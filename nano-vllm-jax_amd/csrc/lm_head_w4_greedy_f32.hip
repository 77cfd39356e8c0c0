// LM head with 4-bit weights (lm_head_w4.h): greedy top-1, f32 activations, as three bf16 terms.
#include "lm_head_w4.h"

int nvjsel::w4_greedy_f32(const W4Args& a, int group, hipStream_t s) {
  return w4_pass<DT_BF16, 3, MODE_GREEDY>(a, group, s);
}
