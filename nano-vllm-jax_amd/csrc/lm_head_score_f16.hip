#include "lm_head_score.h"

int nvjsel::launch_score_f16(const LmArgs& a, const ScoreArgs& sc, const RowAnswers& w, int block_rows, bool entropy, bool cast,
                             hipStream_t s) {
  return launch_score<DT_F16, 1>(a, sc, w, block_rows, entropy, cast, s);
}
