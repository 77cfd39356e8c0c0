// LM head with 4-bit weights (lm_head_w4.h): greedy top-1, f16 activations.
#include "lm_head_w4.h"

int nvjsel::w4_greedy_f16(const W4Args& a, int group, hipStream_t s) {
  return w4_pass<DT_F16, 1, MODE_GREEDY>(a, group, s);
}
