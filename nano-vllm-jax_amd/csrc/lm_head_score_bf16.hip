#include "lm_head_score.h"

int nvjsel::launch_score_bf16(const LmArgs& a, const ScoreArgs& sc, const RowAnswers& w, int block_rows, bool entropy, bool cast,
                             hipStream_t s) {
  return launch_score<DT_BF16, 1>(a, sc, w, block_rows, entropy, cast, s);
}
