// Log probabilities of given tokens, with the rows' entropies and top alternatives,
// and their gradient.  Row n with logits l, token t:
//
//   m = max_v l[v],  S = sum_v exp(l[v] - m),  T = sum_v exp(l[v] - m) (l[v] - m)
//   logprob = (l[t] - m) - ln S,   entropy = -sum_v p[v] ln p[v] = ln S - T / S
//   dl[v] = g (1[v = t] - p[v]) - h p[v] (ln p[v] + entropy),   p[v] = exp((l[v] - m) - ln S)
//
// One pass over the logits takes m, S and T together (row_sums.h): without alternatives
// by row_sums_kernel, with them by beam search's scan and join of rows of one beam
// (beam_select.h), whose candidates' scores are log probabilities.  The gradient is a
// second pass, elementwise, from the row's m, ln S and entropy.
#include "beam_select.h"

namespace nvjsel {

static constexpr int kRowVecs = 4;                       // 16-byte pieces per lane and chunk
static constexpr int kRowThreads = 256, kRowBlockWaves = kRowThreads / 64;
static constexpr int kRowWaves = 16;                     // per CU that a call is split into
static constexpr int kRowBlocks = 64;                    // of a row at most: one lane each joins them
static constexpr int kRowTickets = 4096;                 // rows of several blocks, in 16 KB at a workspace's start
static constexpr int64_t kTopRows = 8192;                // rows of one scan and join
static constexpr int64_t kLaunchBlocks = 1 << 23;        // of 256 threads: a launch has less than 2^32

struct RowArgs {
  const void* logits;
  int vocab;
  int64_t row_stride;
  int share;               // elements of a wave's share (whole chunks)
  int blocks;              // of a row
  unsigned int* tickets;   // [rows], zero at rest: a row's blocks that have finished
  RowPart* parts;          // [rows blocks]
  RowAnswers answers;
};

// Bound: the stream and, beside it, an exponential a logit: 1000 rows of 151,936 bf16 logits (304
// MB) 50 us, 6.1 TB/s, with entropies; 7.0 is this card's streaming read.  8 to 28 waves per CU, two to four
// chunks in registers and chunks half as long took as much (31-33 us at 512 rows), 40 and 64 waves more (36-37).
// A block's four waves take consecutive shares of one row, the next chunk on its way in
// registers, lanes with a maximum and sums of their own; the waves' sums meet in LDS, and
// where a row has several blocks the last one to finish joins them, a lane each.
template <int DT, bool ENT>
__global__ void __launch_bounds__(kRowThreads, 4) row_sums_kernel(RowArgs a) {
  using E = RowElems<DT>;
  constexpr int N = E::N, CHUNK = 64 * kRowVecs * N, DEPTH = 2;
  __shared__ RowPart parts[kRowBlockWaves];
  __shared__ int last;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = (int64_t)blockIdx.x / a.blocks;
  const int part = ((int)(blockIdx.x % a.blocks)) * kRowBlockWaves + wave;
  const size_t es = DT == DT_F32 ? 4 : 2;
  const char* base = (const char*)a.logits + row * a.row_stride * (int64_t)es;
  const int64_t first = (int64_t)part * a.share;
  const int e0 = (int)(first < a.vocab ? first : a.vocab), e1 = (int)(first + a.share < a.vocab ? first + a.share : a.vocab);
  const int full = (e1 - e0) / CHUNK;

  float m = -INFINITY, ref = row_ref(-INFINITY);
  RowSum sum{0.0, 0.0};
  auto take = [&](const row_u32x4 (&w)[kRowVecs]) NVJSEL_INLINE {
    float x = -INFINITY;
#pragma unroll
    for (int j = 0; j < kRowVecs; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) x = __builtin_elementwise_maximum(x, E::get(w[j], e));
    row_add<DT, ENT>(w, x, m, ref, sum);
  };
  if (full > 0) {
    row_u32x4 w[DEPTH][kRowVecs];
    int next = 0;
    auto load = [&](auto D) NVJSEL_INLINE {  // always a load: the last full chunk again at the end
      const char* p = base + ((size_t)e0 + (size_t)(next < full ? next : full - 1) * CHUNK + (size_t)lane * N) * es;
#pragma unroll
      for (int j = 0; j < kRowVecs; ++j) w[decltype(D)::value][j] = __builtin_nontemporal_load((const row_u32x4_any*)(p + j * 1024));
      ++next;
    };
    static_for<DEPTH - 1>([&](auto D) NVJSEL_INLINE { load(D); });
    int c = 0;
    for (; c + DEPTH <= full; c += DEPTH)
      static_for<DEPTH>([&](auto D) NVJSEL_INLINE {
        load(std::integral_constant<int, (decltype(D)::value + DEPTH - 1) % DEPTH>{});
        __builtin_amdgcn_sched_barrier(0);  // the loads first: else a round's are issued behind all its sums
        take(w[decltype(D)::value]);
        __builtin_amdgcn_sched_barrier(0);
      });
    static_for<DEPTH - 1>([&](auto D) NVJSEL_INLINE {
      if (c + decltype(D)::value < full) take(w[decltype(D)::value]);
    });
  }
  if (e0 + full * CHUNK < e1) {  // the share's last elements
    row_u32x4 w[kRowVecs];
#pragma unroll
    for (int j = 0; j < kRowVecs; ++j) w[j] = row_piece<DT>(base, e0 + full * CHUNK + (j * 64 + lane) * N, e1);
    take(w);
  }
  const float wm = wave_max_f32(m);
  const RowSum total = row_wave_total<DT, ENT>(base, e0, e1, wm, ref, sum, lane);
  if (lane == 0) parts[wave] = RowPart{total.sum, total.ent, wm, 0};
  __syncthreads();
  RowSum r{0.0, 0.0};
  float bm = -INFINITY;
  if (wave == 0) {
#pragma unroll
    for (int i = 0; i < kRowBlockWaves; ++i) bm = fmaxf(bm, parts[i].max);
#pragma unroll
    for (int i = 0; i < kRowBlockWaves; ++i) row_join(r, RowSum{parts[i].sum, parts[i].ent}, parts[i].max, bm);
  }
  if (a.blocks == 1) {
    if (tid == 0) row_answer_from<DT>(a.answers, a.logits, row * a.row_stride, a.vocab, row, bm, r);
    return;
  }
  if (tid == 0) {  // passed on at the device's coherence point, before the block's ticket is drawn
    RowPart* p = a.parts + (size_t)blockIdx.x;
    const uint64_t s = (uint64_t)__double_as_longlong(r.sum), t = (uint64_t)__double_as_longlong(r.ent);
    row_put<true>(&p->sum, (uint32_t)s, (uint32_t)(s >> 32));
    row_put<true>(&p->ent, (uint32_t)t, (uint32_t)(t >> 32));
    row_put<true>(&p->max, __float_as_uint(bm), 0u);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = ticket_add(a.tickets + row) == (unsigned int)a.blocks - 1;
  }
  __syncthreads();
  if (!last || wave != 0) return;
  if (tid == 0) __hip_atomic_store(a.tickets + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  RowSum own{0.0, 0.0};
  float om = -INFINITY;
  if (lane < a.blocks) {
    const RowPart* p = a.parts + (size_t)row * a.blocks + lane;
    const uint2 s = row_get<true>(&p->sum), t = row_get<true>(&p->ent), u = row_get<true>(&p->max);
    own = RowSum{two_words(s.x, s.y), two_words(t.x, t.y)};
    om = __uint_as_float(u.x);
  }
  const float rm = wave_max_f32(om);
  r = RowSum{0.0, 0.0};
  row_join(r, own, om, rm);
  r.sum = wave_sum_f64(r.sum);
  if constexpr (ENT) r.ent = wave_sum_f64(r.ent);
  if (lane == 0) row_answer_from<DT>(a.answers, a.logits, row * a.row_stride, a.vocab, row, rm, r);
}

// ---------------------------------------------------------------- the gradient

struct GradArgs {
  const void* logits;
  int vocab;
  int64_t row_stride;
  const void* tokens;
  int token64;
  const float* stats;           // [rows, 3] of the forward call
  const float* grad_logprobs;   // [rows] or null
  const float* grad_entropy;    // [rows] or null
  void* out;                    // [rows, out_stride] of the logits' type
  int64_t out_stride;
  int chunks;                   // blocks of a row
  int64_t row0;                 // of this launch
};

static constexpr int kGradPieces = 4;  // 16-byte pieces of a thread

// Elementwise: one exponential per logit, read once and written once.  p ln p is 0 where p
// is: ln p is held above -1e30 in that product; the hardware's exp2 gives 0 below 2^-126.  A row
// without a gradient (padding) is not read: zeros.  Bound: the reads and writes: 512 rows of 151,936 bf16
// logits (311 MB) 54-57 us, 5.5-5.8 TB/s, a large copy's 5.0; 2 pieces a thread 56.
template <int DT, bool ENT>
__global__ void __launch_bounds__(256) logprobs_grad_kernel(GradArgs a) {
  using E = RowElems<DT>;
  constexpr int N = E::N;
  const int64_t row = a.row0 + (int64_t)(blockIdx.x / (unsigned)a.chunks);
  const int c = (int)(blockIdx.x % (unsigned)a.chunks);
  const int64_t t = a.token64 ? ((const int64_t*)a.tokens)[row] : ((const int32_t*)a.tokens)[row];
  const bool asked = t >= 0 && t < a.vocab;
  const float g = asked && a.grad_logprobs ? a.grad_logprobs[row] : 0.0f;
  const float h = ENT ? a.grad_entropy[row] : 0.0f;
  const float m = a.stats[3 * row], ls = a.stats[3 * row + 1], entropy = a.stats[3 * row + 2];
  const bool zero = (g == 0.0f && h == 0.0f) || m == -INFINITY;
  const size_t es = DT == DT_F32 ? 4 : 2;
  const char* in = (const char*)a.logits + row * a.row_stride * (int64_t)es;
  char* out = (char*)a.out + row * a.out_stride * (int64_t)es;
#pragma unroll
  for (int j = 0; j < kGradPieces; ++j) {
    const int64_t o64 = ((int64_t)c * kGradPieces + j) * 256 * N + (int64_t)threadIdx.x * N;
    if (o64 >= a.vocab) return;
    const int o = (int)o64;
    float d[N];
#pragma unroll
    for (int e = 0; e < N; ++e) d[e] = 0.0f;
    if (!zero) {
      const row_u32x4 w = row_piece<DT>(in, o, a.vocab);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float lp = (E::get(w, e) - m) - ls, p = __builtin_amdgcn_exp2f(lp * kLog2e);
        d[e] = -g * p;
        if constexpr (ENT) d[e] -= h * (p * (fmaxf(lp, -1e30f) + entropy));
        if (o + e == t) d[e] += g;
      }
    }
    row_u32x4 r;
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(d[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint16_t lo, hi;
        if constexpr (DT == DT_BF16) {
          lo = __builtin_bit_cast(uint16_t, (__bf16)d[2 * e]);
          hi = __builtin_bit_cast(uint16_t, (__bf16)d[2 * e + 1]);
        } else {
          lo = __builtin_bit_cast(uint16_t, (_Float16)d[2 * e]);
          hi = __builtin_bit_cast(uint16_t, (_Float16)d[2 * e + 1]);
        }
        r[e] = (uint32_t)hi << 16 | lo;
      }
    }
    char* at = out + (size_t)o * es;
    if (o + N <= a.vocab) {
      *(row_u32x4_any*)at = r;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (o + e < a.vocab) {
          if constexpr (DT == DT_F32) ((uint32_t*)at)[e] = r[e];
          else ((uint16_t*)at)[e] = (uint16_t)(r[e >> 1] >> (16 * (e & 1)));
        }
    }
  }
}

template <int DT>
static int launch_grad(GradArgs a, int64_t rows, hipStream_t s) {
  const int per = 256 * kGradPieces * RowElems<DT>::N;
  a.chunks = (a.vocab - 1) / per + 1;
  const int64_t most = kLaunchBlocks / a.chunks;
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    const int64_t n = rows - r0 < most ? rows - r0 : most;
    a.row0 = r0;
    if (a.grad_entropy)
      hipLaunchKernelGGL((logprobs_grad_kernel<DT, true>), dim3((unsigned)(n * a.chunks)), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((logprobs_grad_kernel<DT, false>), dim3((unsigned)(n * a.chunks)), dim3(256), 0, s, a);
    NVJSEL_CHECK_LAUNCH("logprobs_grad_kernel");
  }
  return NVJSEL_OK;
}

// ---------------------------------------------------------------- host

// Waves' shares of a row without alternatives: enough waves to fill the device, whole chunks.
static void row_split(int64_t rows, int vocab, int dtype, int* share, int* blocks) {
  const int chunk = 64 * kRowVecs * (dtype == DT_F32 ? 4 : 8);
  const int chunks = (vocab - 1) / chunk + 1;
  int64_t b = rows > kRowTickets ? 1 : (int64_t)device_cu_count() * kRowWaves / kRowBlockWaves / rows;
  if (b > kRowBlocks) b = kRowBlocks;
  if (b < 1) b = 1;
  if (b > (chunks + kRowBlockWaves - 1) / kRowBlockWaves) b = (chunks + kRowBlockWaves - 1) / kRowBlockWaves;
  const int64_t waves = b * kRowBlockWaves;
  const int per = (int)((chunks + waves - 1) / waves);
  *share = per * chunk;
  *blocks = (int)((chunks + (int64_t)per * kRowBlockWaves - 1) / ((int64_t)per * kRowBlockWaves));
}

static size_t logprobs_bytes(int dtype, int64_t rows, int vocab, int num_top) {
  if (num_top == 0) {
    int share, blocks;
    row_split(rows, vocab, dtype, &share, &blocks);
    return kRowTickets * 4 + (blocks > 1 ? (size_t)rows * blocks * sizeof(RowPart) : 0);
  }
  const int n = (int)(rows < kTopRows ? rows : kTopRows);
  int shares, share, cap, group;
  beam_split(n, kBeamFew, vocab, num_top, dtype, &shares, &share, &cap, &group);
  return kRowTickets * 4 + (size_t)n * shares * (sizeof(BeamPart) + sizeof(double) + cap * sizeof(uint2));
}

template <int DT>
static int launch_row_sums(const RowArgs& a, int64_t rows, hipStream_t s) {
  if (a.answers.entropy)
    hipLaunchKernelGGL((row_sums_kernel<DT, true>), dim3((unsigned)(rows * a.blocks)), dim3(kRowThreads), 0, s, a);
  else
    hipLaunchKernelGGL((row_sums_kernel<DT, false>), dim3((unsigned)(rows * a.blocks)), dim3(kRowThreads), 0, s, a);
  NVJSEL_CHECK_LAUNCH("row_sums_kernel");
  return NVJSEL_OK;
}

template <int DT>
static int launch_top(const BeamArgs& a, hipStream_t s) {
  return a.answers.entropy ? launch_beam<DT, LP_ENTROPY>(a, s) : launch_beam<DT, LP_PLAIN>(a, s);
}

}  // namespace nvjsel

using namespace nvjsel;

static int logprobs_check(const char* who, int dtype, int64_t rows, int vocab, int num_top) {
  if (rows <= 0 || vocab <= 0) {
    set_error("%s requires non-empty dimensions (rows=%lld vocab=%d)", who, (long long)rows, vocab);
    return NVJSEL_EINVAL;
  }
  if (!valid_dtype(dtype)) { set_error("%s: unsupported logits dtype %d", who, dtype); return NVJSEL_EINVAL; }
  if (num_top < 0 || num_top > kBeamMax) {
    set_error("%s: num_top (%d) must be in 0..%d", who, num_top, kBeamMax);
    return NVJSEL_EINVAL;
  }
  if (vocab > (1 << kBeamVocabBits) || rows > kLaunchBlocks) {
    set_error("%s: vocab (%d) must be at most 2^26, rows (%lld) at most 2^23", who, vocab, (long long)rows);
    return NVJSEL_EINVAL;
  }
  return NVJSEL_OK;
}

static int logprobs_operands(const char* who, const void* logits, int dtype, int64_t row_stride, const void* tokens,
                             int token_bytes) {
  if (!logits || !tokens) { set_error("%s: null pointer", who); return NVJSEL_EINVAL; }
  if (((uintptr_t)logits) & (dtype_size(dtype) - 1)) { set_error("%s: unaligned logits", who); return NVJSEL_EINVAL; }
  if (row_stride < 0) { set_error("%s: negative stride", who); return NVJSEL_EINVAL; }
  if (token_bytes != 4 && token_bytes != 8) { set_error("%s: tokens must be int32 or int64", who); return NVJSEL_EINVAL; }
  if (((uintptr_t)tokens) & (token_bytes - 1)) { set_error("%s: unaligned tokens", who); return NVJSEL_EINVAL; }
  return NVJSEL_OK;
}

extern "C" size_t nvjsel_token_logprobs_workspace_size(int dtype, int64_t rows, int vocab, int num_top) {
  if (logprobs_check("token_logprobs", dtype, rows, vocab, num_top) != NVJSEL_OK) return 0;
  return logprobs_bytes(dtype, rows, vocab, num_top);
}

extern "C" int nvjsel_token_logprobs(const void* logits, int dtype, int64_t rows, int vocab, int64_t row_stride,
                                     const void* tokens, int token_bytes, int num_top, float* out_logprobs,
                                     float* out_entropy, float* out_top, int32_t* out_top_ids, float* out_stats,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = logprobs_check("token_logprobs", dtype, rows, vocab, num_top);
  if (rc == NVJSEL_OK) rc = logprobs_operands("token_logprobs", logits, dtype, row_stride, tokens, token_bytes);
  if (rc != NVJSEL_OK) return rc;
  if (!out_logprobs || (num_top > 0 && (!out_top || !out_top_ids)))
    return fail(NVJSEL_EINVAL, "token_logprobs: null output");
  const size_t need = logprobs_bytes(dtype, rows, vocab, num_top);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) {
    set_error("token_logprobs: workspace %zu bytes (16-byte aligned) < required %zu", workspace_bytes, need);
    return NVJSEL_EWORKSPACE;
  }
  hipStream_t s = (hipStream_t)stream;
  std::lock_guard<std::mutex> lock(launch_mutex());
  const RowAnswers answers{tokens, token_bytes == 8, out_logprobs, out_entropy, out_stats};
  if (num_top == 0) {
    RowArgs a{};
    a.logits = logits;
    a.vocab = vocab;
    a.row_stride = row_stride;
    row_split(rows, vocab, dtype, &a.share, &a.blocks);
    a.tickets = (unsigned int*)workspace;
    a.parts = (RowPart*)((char*)workspace + kRowTickets * 4);
    a.answers = answers;
    if (dtype == DT_F32) return launch_row_sums<DT_F32>(a, rows, s);
    if (dtype == DT_BF16) return launch_row_sums<DT_BF16>(a, rows, s);
    return launch_row_sums<DT_F16>(a, rows, s);
  }
  for (int64_t r0 = 0; r0 < rows; r0 += kTopRows) {
    const int n = (int)(rows - r0 < kTopRows ? rows - r0 : kTopRows);
    BeamArgs a{};
    a.logits = (const char*)logits + r0 * row_stride * (int64_t)dtype_size(dtype);
    a.batch = n;
    a.beams = 1;
    a.vocab = vocab;
    a.k = num_top;
    a.batch_stride = row_stride;
    beam_split(n, kBeamFew, vocab, num_top, dtype, &a.shares, &a.share, &a.cap, &a.group);
    a.tickets = (unsigned int*)workspace;
    a.blocks = (a.shares + kBeamBlockWaves - 1) / kBeamBlockWaves;
    a.parts = (BeamPart*)((char*)workspace + kRowTickets * 4);
    a.ents = (double*)(a.parts + (size_t)n * a.shares);
    a.cand = (uint2*)(a.ents + (size_t)n * a.shares);
    a.answers = answers;
    a.answers.tokens = (const char*)tokens + r0 * token_bytes;
    a.answers.logprobs += r0;
    if (out_entropy) a.answers.entropy += r0;
    if (out_stats) a.answers.stats += 3 * r0;
    a.out_scores = out_top + r0 * num_top;
    a.out_tokens = out_top_ids + r0 * num_top;
    rc = dtype == DT_F32 ? launch_top<DT_F32>(a, s) : dtype == DT_BF16 ? launch_top<DT_BF16>(a, s) : launch_top<DT_F16>(a, s);
    if (rc != NVJSEL_OK) return rc;
  }
  return NVJSEL_OK;
}

extern "C" int nvjsel_token_logprobs_grad(const void* logits, int dtype, int64_t rows, int vocab, int64_t row_stride,
                                          const void* tokens, int token_bytes, const float* stats,
                                          const float* grad_logprobs, const float* grad_entropy, void* out_grad,
                                          int64_t out_row_stride, void* stream) {
  clear_error();
  int rc = logprobs_check("token_logprobs_grad", dtype, rows, vocab, 0);
  if (rc == NVJSEL_OK) rc = logprobs_operands("token_logprobs_grad", logits, dtype, row_stride, tokens, token_bytes);
  if (rc != NVJSEL_OK) return rc;
  if (!stats || !out_grad || (!grad_logprobs && !grad_entropy))
    return fail(NVJSEL_EINVAL, "token_logprobs_grad: null pointer");
  if (((uintptr_t)out_grad) & (dtype_size(dtype) - 1)) return fail(NVJSEL_EINVAL, "token_logprobs_grad: unaligned gradient");
  if (out_row_stride < vocab && rows > 1) return fail(NVJSEL_EINVAL, "token_logprobs_grad: gradient row stride < vocab");
  GradArgs a{};
  a.logits = logits;
  a.vocab = vocab;
  a.row_stride = row_stride;
  a.tokens = tokens;
  a.token64 = token_bytes == 8;
  a.stats = stats;
  a.grad_logprobs = grad_logprobs;
  a.grad_entropy = grad_entropy;
  a.out = out_grad;
  a.out_stride = out_row_stride;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DT_F32) return launch_grad<DT_F32>(a, rows, s);
  if (dtype == DT_BF16) return launch_grad<DT_BF16>(a, rows, s);
  return launch_grad<DT_F16>(a, rows, s);
}
