// Log probabilities of given tokens from the hidden states: the staged GEMM of
// lm_head_ring.h, whose tiles end in sums of exponentials instead of logits.
//
//   l[n, v] = x[n] . W[v],   logprob = (l[n, t] - m) - ln S,   entropy = ln S - T / S   (row_sums.h)
//
// The logits never leave the registers: 2048 rows of 248,320 would be 1 GB written and read
// (bf16; 2 GB f32) beside a product of 1.04 TFLOP.  A lane holds 16 logits of one column (batch row) per
// 32-row tile, so that the sums cross no lanes until a block's share of the vocabulary
// ends; a share's parts are joined by a second kernel, a wave a row.
//
// Bound: the products, at the clock that the card's power leaves.  2048 bf16 rows x 1024, 248,320 tokens, with
// entropies: 874-928 us by card, 1.12-1.19 PFLOP/s (a library's bare product of these sizes, which writes
// 1 GB of logits, 919); the tiles' products without their sums 881: matrix pipes 67% busy of 1.51 M cycles, some 1.7 GHz of
// 2.4.  Logits rounded to the weight's type, the default of 16-bit hidden rows, take 4% more there (920 beside 886 on one
// card: each is rounded where it is compared, summed and taken), 1-2% for 64 and 256 rows, nothing for few.
// 24 rows 79 us, the stream of W (508 MB) at 6.4 TB/s.  300 f32 rows x 768 (three products each)
// of 50,257 tokens 75-77 us, 0.90 PFLOP/s: four tiles a block, three launches; 2048 x 1024, 248,320 tokens 2.62 ms, 1.19 PFLOP/s.
#include "lm_head_score.h"

namespace nvjsel {

__global__ void __launch_bounds__(256) score_finish_kernel(RowAnswers answers, const float* token_logits, const RowPart* parts,
                                                           int rows, int shares, int vocab) {
  const int row = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
  if (row >= rows) return;
  // all on their way together: the parts, the token and its logit (whatever lies there where none is asked)
  const int64_t t = row_token(answers, row);
  const float x = token_logits[row];
  const RowPart* p = parts + (size_t)row * shares;
  constexpr int KEPT = 4;
  RowPart q[KEPT];
#pragma unroll
  for (int u = 0; u < KEPT; ++u) q[u] = p[min(lane + 64 * u, shares - 1)];
  float m = -INFINITY;
#pragma unroll
  for (int u = 0; u < KEPT; ++u) m = fmaxf(m, q[u].max);
  for (int i = lane + 64 * KEPT; i < shares; i += 64) m = fmaxf(m, p[i].max);
  m = wave_max_f32(m);
  RowSum r{0.0, 0.0};
#pragma unroll
  for (int u = 0; u < KEPT; ++u)
    if (lane + 64 * u < shares) row_join(r, RowSum{q[u].sum, q[u].ent}, q[u].max, m);
  for (int i = lane + 64 * KEPT; i < shares; i += 64) row_join(r, RowSum{p[i].sum, p[i].ent}, p[i].max, m);
  r.sum = wave_sum_f64(r.sum);
  r.ent = wave_sum_f64(r.ent);
  if (lane != 0) return;
  const bool asked = t >= 0 && t < vocab;
  row_answer(answers, row, asked, asked ? x : 0.0f, m, r, row_log_sum(r.sum));
}

// f32 hidden rows as their three bf16 terms, [row][term][H], eight values a thread: once for a launch, where
// the GEMM's blocks would each split them again for every tile (calls of 300 rows x 768 and 50,257 tokens 85 -> 77
// us, 64 x 1024 and 248,320 124 -> 108, 40 x 768 and 8000 26 -> 24, 2048 x 1024 and 248,320 3455 -> 2622).
__global__ void __launch_bounds__(256) score_split_kernel(const float* hidden, uint16_t* terms, int H, int64_t pieces) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= pieces) return;
  const int each = H / 8;
  const int64_t row = i / each;
  const int k = (int)(i - row * each) * 8;
  const u32x4_t* x = (const u32x4_t*)(hidden + i * 8);
  float v[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const u32x4_t r = x[h];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[h][j] = __uint_as_float(r[j]);
  }
#pragma unroll
  for (int t = 0; t < 3; ++t) {
    const uint2 lo = next_term(v[0]), hi = next_term(v[1]);
    *(u32x4_t*)(terms + (row * 3 + t) * H + k) = u32x4_t{lo.x, lo.y, hi.x, hi.y};
  }
}

int launch_score_split(const LmArgs& a, const ScoreArgs& sc, hipStream_t s) {
  const int64_t pieces = (int64_t)a.B * (a.H / 8);
  hipLaunchKernelGGL(score_split_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, (const float*)a.hidden,
                     sc.terms, a.H, pieces);
  NVJSEL_CHECK_LAUNCH("score_split_kernel");
  return NVJSEL_OK;
}

int launch_score_finish(const RowAnswers& answers, const ScoreArgs& sc, int rows, int vocab, hipStream_t s) {
  hipLaunchKernelGGL(score_finish_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, answers,
                     (const float*)sc.token_logits, (const RowPart*)sc.parts, rows, sc.shares, vocab);
  NVJSEL_CHECK_LAUNCH("score_finish_kernel");
  return NVJSEL_OK;
}

// Rows of a block: 256 while more than 128 are left (64 of f32 activations, three products each).
static int score_block_rows(bool f32, int64_t left) {
  if (f32) return left > 32 ? 64 : 32;
  return left > 128 ? 256 : left > 64 ? 128 : left > 32 ? 64 : 32;
}

// Row blocks of the next launch: a call of n blocks is cut so that the rounds of tiles, half a tile for a
// launch, are fewest over all (every CU has one block: 5 of 51 shares each fill 255 CUs, 29 of 8
// fill 232, 16 and 13 256 and 247).
static constexpr int kScoreBlocks = 32;  // of a launch at most
static int score_row_blocks(int64_t left, int vocab, int cus) {
  const int most = cus < kScoreBlocks ? cus : kScoreBlocks;
  double cost[kScoreBlocks + 1], total[2 * kScoreBlocks + 1];
  int first[2 * kScoreBlocks + 1];
  int whole = 1;  // the launch of most rows a round, while more than two of the largest are left
  for (int r = 1; r <= most; ++r) {
    cost[r] = 0.5 + ring_tiles(ring_share(vocab, cus / r));
    if (r * cost[whole] >= whole * cost[r]) whole = r;
  }
  if (left > 2 * most) return whole;
  total[0] = 0.0;
  for (int n = 1; n <= (int)left; ++n) {
    first[n] = 1;
    total[n] = 1e30;
    for (int r = 1; r <= most && r <= n; ++r)
      if (cost[r] + total[n - r] <= total[n]) {
        total[n] = cost[r] + total[n - r];
        first[n] = r;
      }
  }
  return first[left];
}

// Hidden values whose terms are kept, for calls of more than 32 f32 rows.
static constexpr int kScoreTermsHidden = 16384;
static bool score_terms(bool f32, int64_t rows, int H) { return f32 && rows > 32 && H <= kScoreTermsHidden; }
static size_t score_parts_bytes(int64_t rows, int cus) {  // parts: at most `cus` shares x row blocks of 256 rows
  return align_up((size_t)rows * 4, 16) + (size_t)cus * 256 * sizeof(RowPart);
}
static size_t score_bytes(bool f32, int64_t rows, int H, int cus) {
  const int64_t most = rows < kScoreBlocks * 64 ? rows : kScoreBlocks * 64;  // of a launch
  return score_parts_bytes(rows, cus) + (score_terms(f32, rows, H) ? (size_t)most * 3 * H * 2 : 0);
}

}  // namespace nvjsel

using namespace nvjsel;

static int score_check(int hidden_dtype, int weight_dtype, int layout, int64_t rows, int H, int V) {
  if (rows <= 0 || H <= 0 || V <= 0) {
    set_error("lm_head_token_logprobs requires non-empty dimensions (rows=%lld hidden=%d vocab=%d)", (long long)rows, H, V);
    return NVJSEL_EINVAL;
  }
  if (!valid_dtype(hidden_dtype) || !valid_dtype(weight_dtype)) {
    set_error("lm_head_token_logprobs: unsupported dtype (hidden=%d weight=%d)", hidden_dtype, weight_dtype);
    return NVJSEL_EINVAL;
  }
  if (layout != NVJSEL_W_VH && layout != NVJSEL_W_HV) {
    set_error("lm_head_token_logprobs: bad weight layout %d", layout);
    return NVJSEL_EINVAL;
  }
  if (rows > 1 << 23) return fail(NVJSEL_EINVAL, "lm_head_token_logprobs: at most 2^23 rows");
  const bool types = weight_dtype != NVJSEL_F32 && (hidden_dtype == weight_dtype ||
                                                    (hidden_dtype == NVJSEL_F32 && weight_dtype == NVJSEL_BF16));
  if (layout != NVJSEL_W_VH || !types || H % kRingKC != 0 || H > (1 << 20) || V >= 0x7FFFFF00) {
    set_error("lm_head_token_logprobs: takes a 16-bit weight [V, H], H a multiple of 64, hidden of its type or f32 beside bf16");
    return NVJSEL_EUNSUPPORTED;
  }
  return NVJSEL_OK;
}

extern "C" size_t nvjsel_lm_head_token_logprobs_workspace_size(int hidden_dtype, int weight_dtype, int weight_layout,
                                                               int64_t rows, int hidden_dim, int vocab) {
  clear_error();
  if (score_check(hidden_dtype, weight_dtype, weight_layout, rows, hidden_dim, vocab) != NVJSEL_OK) return 0;
  return score_bytes(hidden_dtype == NVJSEL_F32, rows, hidden_dim, device_cu_count());
}

extern "C" int nvjsel_lm_head_token_logprobs(const void* hidden, int hidden_dtype, const void* weight, int weight_dtype,
                                             int weight_layout, int64_t rows, int hidden_dim, int vocab, int reduce_cast,
                                             const void* tokens, int token_bytes, float* out_logprobs, float* out_entropy,
                                             void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const int rc = score_check(hidden_dtype, weight_dtype, weight_layout, rows, hidden_dim, vocab);
  if (rc != NVJSEL_OK) return rc;
  if (!hidden || !weight || !tokens || !out_logprobs) return fail(NVJSEL_EINVAL, "lm_head_token_logprobs: null pointer");
  if (reduce_cast < 0 || reduce_cast > 2) return fail(NVJSEL_EINVAL, "lm_head_token_logprobs: reduce_cast must be 0, 1 or 2");
  if (reduce_cast && reduce_cast != (hidden_dtype == NVJSEL_F32 ? 0 : weight_dtype))
    return fail(NVJSEL_EUNSUPPORTED, "lm_head_token_logprobs: reduce_cast must be 0 or the type of 16-bit operands");
  if ((token_bytes != 4 && token_bytes != 8) || ((uintptr_t)tokens & (token_bytes - 1)))
    return fail(NVJSEL_EINVAL, "lm_head_token_logprobs: tokens must be int32 or int64, aligned");
  if ((((uintptr_t)hidden) | ((uintptr_t)weight)) & 15)
    return fail(NVJSEL_EUNSUPPORTED, "lm_head_token_logprobs: hidden and weight must be 16-byte aligned");
  const int cus = device_cu_count();
  const bool f32 = hidden_dtype == NVJSEL_F32;
  const size_t need = score_bytes(f32, rows, hidden_dim, cus);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) {
    set_error("lm_head_token_logprobs: workspace %zu bytes (16-byte aligned) < required %zu", workspace_bytes, need);
    return NVJSEL_EWORKSPACE;
  }
  std::lock_guard<std::mutex> lock(launch_mutex());
  hipStream_t s = (hipStream_t)stream;
  int64_t n = 0;
  for (int64_t r0 = 0; r0 < rows; r0 += n) {
    const int64_t left = rows - r0;
    const int block_rows = score_block_rows(f32, left);
    ScoreArgs sc{};
    // a last block that a smaller shape takes is left to the next launch
    const int64_t blocks = block_rows == 256 ? (left + 127) / 256 : (left + block_rows - 1) / block_rows;
    sc.row_blocks = score_row_blocks(blocks, vocab, cus);
    n = (int64_t)sc.row_blocks * block_rows < left ? (int64_t)sc.row_blocks * block_rows : left;
    sc.tokens = (const char*)tokens + r0 * token_bytes;
    sc.token64 = token_bytes == 8;
    sc.token_logits = (float*)workspace + r0;
    sc.parts = (RowPart*)((char*)workspace + align_up((size_t)rows * 4, 16));
    sc.terms = score_terms(f32, rows, hidden_dim) ? (uint16_t*)((char*)workspace + score_parts_bytes(rows, cus)) : nullptr;
    LmArgs a{};
    a.W = weight;
    a.hidden = (const char*)hidden + (size_t)r0 * hidden_dim * dtype_size(hidden_dtype);
    a.hidden_dtype = hidden_dtype;
    a.act_dtype = hidden_dtype;
    a.weight_dtype = weight_dtype;
    a.layout = weight_layout;
    a.B = (int)n;
    a.H = hidden_dim;
    a.V = vocab;
    a.reduce_cast = reduce_cast;
    const RowAnswers answers{sc.tokens, sc.token64, out_logprobs + r0, out_entropy ? out_entropy + r0 : nullptr, nullptr};
    const int st = hidden_dtype == NVJSEL_F32    ? launch_score_f32(a, sc, answers, block_rows, out_entropy, false, s)
                   : weight_dtype == NVJSEL_BF16 ? launch_score_bf16(a, sc, answers, block_rows, out_entropy, reduce_cast, s)
                                                 : launch_score_f16(a, sc, answers, block_rows, out_entropy, reduce_cast, s);
    if (st != NVJSEL_OK) return st;
  }
  return NVJSEL_OK;
}
