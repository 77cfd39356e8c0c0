// LM head with 4-bit weights (lm_head_w4.h): logits, bf16 activations.
#include "lm_head_w4.h"

int nvjsel::w4_logits_bf16(const W4Args& a, int group, hipStream_t s) {
  return w4_pass<DT_BF16, 1, MODE_LOGITS>(a, group, s);
}
