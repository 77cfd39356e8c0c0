// LM head with 4-bit weights (lm_head_w4.h): logits, f32 activations, as three bf16 terms.
#include "lm_head_w4.h"

int nvjsel::w4_logits_f32(const W4Args& a, int group, hipStream_t s) {
  return w4_pass<DT_BF16, 3, MODE_LOGITS>(a, group, s);
}
