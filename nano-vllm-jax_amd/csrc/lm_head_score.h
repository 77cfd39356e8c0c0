// Launches of the scoring staged GEMM, instantiated by types in
// lm_head_score_{bf16,f16,f32}.hip.
#pragma once
#include "lm_head_ring.h"

namespace nvjsel {

// Rows a block takes (32, 64, 128 or 256; f32 hidden 32 or 64), with the entropy, of logits rounded to the weight's type.
int launch_score_bf16(const LmArgs& a, const ScoreArgs& sc, const RowAnswers& w, int block_rows, bool entropy, bool cast,
                      hipStream_t s);
int launch_score_f16(const LmArgs& a, const ScoreArgs& sc, const RowAnswers& w, int block_rows, bool entropy, bool cast,
                     hipStream_t s);
int launch_score_f32(const LmArgs& a, const ScoreArgs& sc, const RowAnswers& w, int block_rows, bool entropy, bool cast,
                     hipStream_t s);
int launch_score_split(const LmArgs& a, const ScoreArgs& sc, hipStream_t s);
int launch_score_finish(const RowAnswers& answers, const ScoreArgs& sc, int rows, int vocab, hipStream_t s);

template <int WT, int MODE, int NBR, int NS>
static int launch_score_rows(const LmArgs& a, ScoreArgs sc, const RowAnswers& answers, hipStream_t s) {
  const int rows = ring_share(a.V, device_cu_count() / sc.row_blocks);
  sc.shares = (a.V + rows - 1) / rows;
  hipLaunchKernelGGL((lm_head_ring_kernel<WT, MODE, NBR, NS>), dim3((unsigned)(sc.shares * sc.row_blocks)),
                     dim3(RingShape<MODE, NBR, NS>::NW * 64), 0, s, a, rows, sc);
  NVJSEL_CHECK_LAUNCH("lm_head_ring_kernel");
  return launch_score_finish(answers, sc, a.B, a.V, s);
}

template <int WT, int NS, int MODE>
static int launch_score_mode(const LmArgs& a, const ScoreArgs& sc, const RowAnswers& w, int block_rows, hipStream_t s) {
  if (block_rows == 32) return launch_score_rows<WT, MODE, 32, NS>(a, sc, w, s);
  if constexpr (NS == 3) {
    if (sc.terms && block_rows == 64) {
      const int rc = launch_score_split(a, sc, s);
      return rc != NVJSEL_OK ? rc : launch_score_rows<WT, MODE + SCORE_TERMS, 64, NS>(a, sc, w, s);
    }
  } else {
    if (block_rows == 128) return launch_score_rows<WT, MODE, 128, NS>(a, sc, w, s);
    if (block_rows == 256) return launch_score_rows<WT, MODE, 256, NS>(a, sc, w, s);
  }
  return launch_score_rows<WT, MODE, 64, NS>(a, sc, w, s);
}
template <int WT, int NS>
static int launch_score(const LmArgs& a, const ScoreArgs& sc, const RowAnswers& w, int block_rows, bool entropy, bool cast,
                        hipStream_t s) {
  if constexpr (NS == 1) {
    if (cast)
      return entropy ? launch_score_mode<WT, NS, MODE_SCORE + SCORE_ENTROPY + SCORE_CAST>(a, sc, w, block_rows, s)
                     : launch_score_mode<WT, NS, MODE_SCORE + SCORE_CAST>(a, sc, w, block_rows, s);
  }
  return entropy ? launch_score_mode<WT, NS, MODE_SCORE + SCORE_ENTROPY>(a, sc, w, block_rows, s)
                 : launch_score_mode<WT, NS, MODE_SCORE + 0>(a, sc, w, block_rows, s);
}

}  // namespace nvjsel
