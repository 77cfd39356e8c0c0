// Beam search's selection over beams and vocabulary, also taken by the log
// probabilities with top alternatives (one beam a row, no scores).
//
//   candidate (w, v) of request b:  S[b,w] + (l[b,w,v] - m) - log sum_v' exp(l[b,w,v'] - m),  m = max_v' l[b,w,v']
//
// the K best over all w and v, by value, then by w V + v.  Within a row the order
// is the logits' own, so one pass over them takes each part's maximum, sum of
// exponentials and the few logits that can be among the K best (beam_scan), and one
// block per request joins the parts, turns those logits into scores in fp64 and
// ranks them (beam_join).  With few parts a request's last block to finish them joins
// them in the same launch, with more a second kernel does (kBeamFew). fp64 there because two beams'
// candidates may lie closer than an fp32 score resolves; the sums of exponentials
// are fp32 within a lane's 16 or 32 logits of a chunk and fp64 across chunks, lanes and parts.
#pragma once
#include <float.h>

#include "row_sums.h"

namespace nvjsel {

static constexpr int kBeamMax = 64;        // beams and candidates per request: one lane each
static constexpr int kBeamRequests = 65536;  // of a call: a workspace's tickets are at the same place for every shape
static constexpr int kBeamVecs = 4;        // 16-byte pieces per lane and chunk
static constexpr int kBeamWaves = 16;      // per CU that a call is split into
static constexpr int kBeamSlots = 8;       // lanes' maxima kept of a share, each over as many chunks as it takes
// Pieces of a lane and chunk that a wave can set aside: 50 expected over 8 chunks at K = 16,
// 90 at 32 (256 rows of 248,320, K = 32: 42.8 us with 64, read again, 39.1 so); four blocks fit a CU.
static constexpr int kBeamHeld = 112;
static constexpr int kBeamThreads = 256, kBeamBlockWaves = kBeamThreads / 64;
// One launch scans and joins calls of up to kBeamOne parts, kBeamFew a request.  What
// passes between its blocks goes by the device's coherence point: calls of 64 / 400 / 512 /
// 625 / 1024 / 2048 parts take 9.9 / 11.6 / 11.0 / 12.2 / 12.7 / 18.5 us so and 12.4 / 12.1 /
// 12.3 / 11.6 / 11.5 / 12.7 in two kernels, one after the other from Python.  And the
// parts of a request at most.
static constexpr int kBeamOne = 512, kBeamFew = 256, kBeamLists = 2048;
static constexpr int kBeamJoinThreads = 512;             // of the second kernel
static constexpr int kBeamOneMax = 24;     // candidates that one maximum per lane bounds well enough, two above
static constexpr int kBeamClasses = 128;   // of parts or candidates, two per lane, for the join's bounds
static constexpr int kBeamFewShares = 4;   // of a row, whose sums a lane joins, not a wave (64 beams of one share: 14 us by waves, 1.2 so)
static constexpr int kBeamEarly = 1024;    // candidates that one launch's join loads with the parts
static constexpr int kBeamRefine = 128;    // candidates that are ranked without a second bound

struct BeamPart {  // of one wave's share of a row
  double sum;      // sum of exp(l - max)
  float max;
  int count;       // candidates
};

struct BeamArgs {
  const void* logits;
  int batch, beams, vocab, k;
  int64_t batch_stride, beam_stride;  // elements
  const float* scores;      // [batch, beams]
  const uint8_t* finished;  // [batch, beams] or null
  int end_token;
  int shares, share;  // parts of a row, and their length in elements (whole chunks)
  unsigned int* tickets;  // [batch], zero at rest: blocks that have finished their parts
  int blocks;             // of a request
  BeamPart* parts;        // [batch beams shares]
  uint2* cand;            // [batch beams shares][cap]: logit bits, token
  int cap;            // candidates of a share at most
  int group;          // chunks per kept maximum
  // log probabilities (LP): rows of one beam each, without scores
  RowAnswers answers;
  double* ents;  // of the parts: sum of exp(l - max) (l - max)
  float* out_scores;
  int32_t* out_parents;
  int32_t* out_tokens;
};

// LP: the rows are not beams, but ask for log probabilities.
enum { LP_NONE = 0, LP_PLAIN = 1, LP_ENTROPY = 2 };

// What a beam contributes: nothing, every token, one token, or NaN.
enum { BEAM_DEAD = 0, BEAM_LIVE = 1, BEAM_ENDED = 2, BEAM_NAN = 3, BEAM_ENDED_NAN = 4 };

__device__ __forceinline__ int beam_state(float score, bool ended) {
  if (score == -INFINITY) return BEAM_DEAD;
  if (!(score < INFINITY)) return ended ? BEAM_ENDED_NAN : BEAM_NAN;
  return ended ? BEAM_ENDED : BEAM_LIVE;
}

// The largest t with its last `skip` bits clear that at least k of the wave's 2 x 64
// numbers reach (0 if there are fewer than k): bit by bit, by counting lanes.
__device__ __forceinline__ uint32_t wave_kth(uint32_t x, uint32_t y, int k, int skip) {
  uint32_t t = 0;
  for (int i = 31; i >= skip; --i) {
    const uint32_t u = t | 1u << i;
    if (__builtin_popcountll(__ballot(x >= u)) + __builtin_popcountll(__ballot(y >= u)) >= k) t = u;
  }
  return t;
}
// The K best logits of a share exactly, one lane each in order, where too many
// logits reach the bound that the scan takes from its lanes' maxima: a row of equal
// or masked values.  A token enters by comparing all lanes at once; tokens are
// visited in order of index and enter only above the K-th value, so among equal
// logits the lowest indices stay, and a row of equal logits costs K entries.
template <int DT>
__device__ __forceinline__ void beam_best(const char* base, int e0, int e1, int k, int lane, float& val, uint32_t& idx) {
  using E = RowElems<DT>;
  val = -INFINITY;
  idx = 0xFFFFFFFFu;
  float thr = -INFINITY;
  for (int c0 = e0; c0 < e1; c0 += 64 * E::N) {
    const row_u32x4 w = row_piece<DT>(base, c0 + lane * E::N, e1);
    float gm = E::get(w, 0);
#pragma unroll
    for (int e = 1; e < E::N; ++e) gm = fmaxf(gm, E::get(w, e));
    uint64_t hit = __ballot(gm > thr);
    while (hit) {
      const int l = __builtin_ctzll(hit);
      row_u32x4 t;
#pragma unroll
      for (int q = 0; q < 4; ++q) t[q] = (uint32_t)__builtin_amdgcn_readlane((int)w[q], l);
      const uint32_t i0 = (uint32_t)(c0 + l * E::N);
#pragma unroll
      for (int e = 0; e < E::N; ++e) {
        const float x = E::get(t, e);
        if (x > thr) {
          const int pos = __builtin_popcountll(__ballot(val >= x));
          if (pos < k) {
            const float pv = __shfl_up(val, 1, 64);
            const uint32_t pi = (uint32_t)__shfl_up((int)idx, 1, 64);
            val = lane > pos ? pv : lane == pos ? x : val;
            idx = lane > pos ? pi : lane == pos ? i0 + (uint32_t)e : idx;
            thr = readlane_f(val, k - 1);  // -inf while fewer than K have entered
          }
        }
      }
      hit &= hit - 1;
      hit &= __ballot(gm > thr);
    }
  }
}

// One share of a row per wave, in chunks of 64 lanes x kBeamVecs pieces, the next one
// on its way in registers.  A lane keeps its own maximum and sum, so that the
// stream's sums cross no lanes.  The K-th largest of the 64 lanes' maxima so far (of
// 128, two per lane, for large K) is a bound that at least K logits reach and few
// more: 64 ln(64 / (64 - K)) expected, 18 at K = 16, 128 ln(128 / (128 - K)), 89 at 64.
// It is taken after 1, 2, 4, ... chunks, and a lane whose maximum of a chunk reaches it
// sets the chunk's pieces aside in LDS; at the end the logits among them that reach
// the last bound are the candidates.  Where more are set aside than there is room
// for, the pieces are read again instead, by the lanes' maxima of every chunk in LDS
// (V = 248,320, 256 rows, K = 16: 2 us more).
//
// Bound: the stream, and in part beside it an exponential and a maximum per logit and
// the pieces set aside: 256 rows of 248,320 bf16 logits (127 MB) take 26 us, 4.9 TB/s, 20 with sums of
// the logits themselves, 18 with nothing set aside either.  The bound by halving between the least and
// the greatest lane instead of bit by bit took 2 us more.
struct BeamScanLds {
  float lane_max[kBeamBlockWaves][kBeamSlots][64];
  row_u32x4 aside[kBeamBlockWaves][kBeamHeld][kBeamVecs];  // or, read again: the (slot, lane) pairs
  int aside_at[kBeamBlockWaves][kBeamHeld];               // their first element
};
static_assert(sizeof(row_u32x4) * kBeamHeld * kBeamVecs >= kBeamSlots * 64 * sizeof(uint16_t), "");

template <int DT, bool ONE, int LP>
__device__ __forceinline__ void beam_scan(const BeamArgs& a, BeamScanLds& lds, int row, int part, int wave, int lane) {
  using E = RowElems<DT>;
  constexpr int N = E::N, CHUNK = 64 * kBeamVecs * N, DEPTH = 2;
  const int wid = row * a.shares + part;
  const size_t es = DT == DT_F32 ? 4 : 2;
  const char* base = (const char*)a.logits +
                     ((int64_t)(row / a.beams) * a.batch_stride + (int64_t)(row % a.beams) * a.beam_stride) * (int64_t)es;
  const int e0 = part * a.share, e1 = min(a.vocab, e0 + a.share), k = a.k;
  const int full = (e1 - e0) / CHUNK;
  float (*lm)[64] = lds.lane_max[wave];
  auto& aside = lds.aside[wave];
  auto& aside_at = lds.aside_at[wave];

  float m = -INFINITY, ref = row_ref(-INFINITY), kept = -INFINITY;
  RowSum sum{0.0, 0.0};                    // relative to 2^ref
  float half[2] = {-INFINITY, -INFINITY};  // the maximum by pieces: the first and the last ones of every chunk
  float bound = -FLT_MAX;                  // of the candidates: -inf is none
  int taken = 0, held = 0;                 // chunks; pieces set aside
  auto find_bound = [&]() NVJSEL_INLINE {  // in 16 bits of the order: bf16's own, and as good a bound for the others
    const uint32_t t = k <= kBeamOneMax ? wave_kth(ord_f32(m), 0u, k, 16) : wave_kth(ord_f32(half[0]), ord_f32(half[1]), k, 16);
    bound = t <= ord_f32(-INFINITY) ? -FLT_MAX : unord_f32(t);
  };
  int slot = 0, more = a.group;
  auto take = [&](const row_u32x4 (&w)[kBeamVecs]) NVJSEL_INLINE {  // chunk `taken` of the share
    float x = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float y = -INFINITY;
#pragma unroll
      for (int j = h * kBeamVecs / 2; j < (h + 1) * kBeamVecs / 2; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) y = __builtin_elementwise_maximum(y, E::get(w[j], e));
      half[h] = __builtin_elementwise_maximum(half[h], y);
      x = __builtin_elementwise_maximum(x, y);
    }
    kept = __builtin_elementwise_maximum(kept, x);
    lm[slot][lane] = kept;
    if (--more == 0) {
      more = a.group;
      kept = -INFINITY;
      ++slot;
    }
    row_add<DT, LP == LP_ENTROPY>(w, x, m, ref, sum);
    if ((taken & (taken + 1)) == 0) find_bound();
    const uint64_t hit = __ballot(x >= bound);
    if (hit) {
      const int at = held + __builtin_popcountll(hit & ((1ull << lane) - 1));
      if (x >= bound && at < kBeamHeld) {
        aside_at[at] = e0 + taken * CHUNK + lane * N;
#pragma unroll
        for (int j = 0; j < kBeamVecs; ++j) aside[at][j] = w[j];
      }
      held += __builtin_popcountll(hit);
    }
    ++taken;
  };
  if (full > 0) {
    row_u32x4 w[DEPTH][kBeamVecs];
    int next = 0;
    auto load = [&](auto D) NVJSEL_INLINE {  // always a load: the last full chunk again at the end
      const char* p = base + ((size_t)e0 + (size_t)(next < full ? next : full - 1) * CHUNK + (size_t)lane * N) * es;
#pragma unroll
      for (int j = 0; j < kBeamVecs; ++j) w[decltype(D)::value][j] = __builtin_nontemporal_load((const row_u32x4_any*)(p + j * 1024));
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
  if (e0 + full * CHUNK < e1) {  // the row's last elements
    row_u32x4 w[kBeamVecs];
#pragma unroll
    for (int j = 0; j < kBeamVecs; ++j) w[j] = row_piece<DT>(base, e0 + full * CHUNK + (j * 64 + lane) * N, e1);
    take(w);
  }

  const float wm = wave_max_f32(m);
  const RowSum total = row_wave_total<DT, LP == LP_ENTROPY>(base, e0, e1, wm, ref, sum, lane);

  if (taken & (taken - 1)) find_bound();  // else it is of all chunks already
  uint2* cand = a.cand + (size_t)wid * a.cap;
  int count = 0;
  auto collect = [&](const row_u32x4& w, int o) NVJSEL_INLINE {  // the candidates of a piece per lane
    uint32_t hits = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) hits |= (uint32_t)(E::get(w, e) >= bound) << e;
    uint64_t some = __ballot(hits != 0);
    while (some) {  // a lane's first hit left, then its next
      const int e = __builtin_ctz(hits | 1u << 31), at = count + __builtin_popcountll(some & ((1ull << lane) - 1));
      if (hits && at < a.cap) {
        const uint32_t v = DT == DT_F32 ? (e & 2 ? (e & 1 ? w[3] : w[2]) : (e & 1 ? w[1] : w[0]))
                                        : (e & 4 ? (e & 2 ? w[3] : w[2]) : (e & 2 ? w[1] : w[0]));
        const float x = DT == DT_F32    ? __uint_as_float(v)
                        : DT == DT_BF16 ? bf16_to_f32((uint16_t)(e & 1 ? v >> 16 : v))
                                        : f16_to_f32((uint16_t)(e & 1 ? v >> 16 : v));
        row_put<ONE>(cand + at, __float_as_uint(x), (uint32_t)(o + e));
      }
      count += __builtin_popcountll(some);
      hits &= hits - 1;
      some = __ballot(hits != 0);
    }
  };
  __builtin_amdgcn_wave_barrier();  // LDS operations of a wave are performed in order
  if (held <= kBeamHeld) {
    for (int i0 = 0; i0 < held * kBeamVecs; i0 += 64) {
      const int i = i0 + lane;
      row_u32x4 w{E::none(), E::none(), E::none(), E::none()};
      int o = 0;
      if (i < held * kBeamVecs) {
        w = aside[i / kBeamVecs][i % kBeamVecs];
        o = aside_at[i / kBeamVecs] + (i % kBeamVecs) * 64 * N;
      }
      collect(w, o);
    }
  } else {
    uint16_t* pairs = (uint16_t*)&aside[0][0];
    const int slots = slot + (more < a.group);
    int np = 0;
    for (int c = 0; c < slots; ++c) {
      const bool hit = lm[c][lane] >= bound;
      const uint64_t b = __ballot(hit);
      if (hit) pairs[np + __builtin_popcountll(b & ((1ull << lane) - 1))] = (uint16_t)(c * 64 + lane);
      np += __builtin_popcountll(b);
    }
    __builtin_amdgcn_wave_barrier();
    for (int i0 = 0; i0 < np * kBeamVecs; i0 += 64) {  // a piece per lane
      const int i = i0 + lane, pair = i < np * kBeamVecs ? pairs[i / kBeamVecs] : 0;
      for (int g = 0; g < a.group; ++g) {
        int o = e0 + ((pair >> 6) * a.group + g) * CHUNK + ((i % kBeamVecs) * 64 + (pair & 63)) * N;
        o = i < np * kBeamVecs ? o : e1;
        collect(row_piece<DT>(base, o, e1), o);
      }
    }
  }
  if (count > a.cap) {
    float val;
    uint32_t idx;
    beam_best<DT>(base, e0, e1, k, lane, val, idx);
    const uint64_t b = __ballot(lane < k && val > -INFINITY);
    if (b >> lane & 1) row_put<ONE>(cand + lane, __float_as_uint(val), idx);
    count = __builtin_popcountll(b);
  }
  if (lane == 0) {
    const uint64_t u = (uint64_t)__double_as_longlong(total.sum);
    row_put<ONE>(&a.parts[wid].sum, (uint32_t)u, (uint32_t)(u >> 32));
    if constexpr (LP == LP_ENTROPY) {
      const uint64_t t = (uint64_t)__double_as_longlong(total.ent);
      row_put<ONE>(a.ents + wid, (uint32_t)t, (uint32_t)(t >> 32));
    }
    row_put<ONE>(&a.parts[wid].max, __float_as_uint(wm), (uint32_t)count);
  }
}

// A candidate: its score, then beam (6 bits), logit (32, the largest first) and
// token (26), the lowest first.  Equal scores go by beam and token; the logit
// between them keeps a beam's own order where its logits are closer than an fp64
// score resolves.
struct BeamKey {
  double s;
  uint64_t at;
};
static constexpr uint64_t kBeamNone = ~0ull;
static constexpr int kBeamVocabBits = 26;
__device__ __forceinline__ uint64_t beam_at(int w, float logit, uint32_t v) {
  return (uint64_t)w << 58 | (uint64_t)(~ord_f32(logit)) << kBeamVocabBits | v;
}
__device__ __forceinline__ bool beam_before(const BeamKey& x, const BeamKey& y) {
  return x.s > y.s || (x.s == y.s && x.at < y.at);
}
__device__ __forceinline__ BeamKey beam_xor(const BeamKey& x, int m) {
  return BeamKey{__shfl_xor(x.s, m, 64), shfl_xor_u64(x.at, m)};
}
__device__ __forceinline__ BeamKey beam_from(const BeamKey& x, int l) {
  const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)x.at, l, 64), hi = (uint32_t)__shfl((int)(uint32_t)(x.at >> 32), l, 64);
  return BeamKey{__shfl(x.s, l, 64), (uint64_t)hi << 32 | lo};
}
// One compare-exchange with the lane d away; first: the better one to the lower lane.
__device__ __forceinline__ void beam_step(BeamKey& x, int d, bool first, int lane) {
  const BeamKey o = beam_xor(x, d);
  const bool low = (lane & d) == 0, mine = beam_before(x, o);
  if ((first == low) != mine) x = o;
}
__device__ __forceinline__ void beam_sort(BeamKey& x, int lane) {
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d >= 1; d >>= 1) beam_step(x, d, (lane & size) == 0, lane);
}
// The best 64 of two sorted lists, sorted: x against y reversed, then a bitonic merge.
__device__ __forceinline__ void beam_merge(BeamKey& x, const BeamKey& y, int lane) {
  const BeamKey r = beam_from(y, 63 - lane);
  if (beam_before(r, x)) x = r;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) beam_step(x, d, true, lane);
}

// fp64 scores as unsigned numbers of the same order.
__device__ __forceinline__ uint64_t beam_ord(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return u >> 63 ? ~u : u | 1ull << 63;
}

// A request's parts joined by one block.  The rows' normalisers from their parts; then
// a bound: the parts fall into 128 classes, and the K-th best of the classes' best
// scores (by their first 32 bits) is one that at least K candidates reach.  The
// candidates that reach it, seldom more than twice K, are ranked by counting, each
// against all; where there are more than there is room for (many equal scores), every
// wave keeps the best 64 of its share of them sorted and the waves' lists are merged.
// Bound: a chain of memory round trips (parts, candidates), barriers and dependent
// instructions (an fp64 exponential a part and logarithm a beam, the bound's bits), 7 us
// whatever the size: with 256 rows its waves wait 70% of their time, and vector
// instructions fill 1% of it.
template <int LISTS>
struct BeamJoinLds {
  static constexpr int RANKED = LISTS == kBeamFew ? 512 : 1024;
  BeamKey keys[RANKED];
  BeamPart part[LISTS];
  double rlog[kBeamMax], rscore[kBeamMax];
  unsigned long long taken;        // parts that reach the bound, and above them their candidates
  int state[kBeamMax];
  float rmax[kBeamMax];
  uint32_t best_of[kBeamClasses];  // of the parts' classes: the scores' first 32 bits in order
  uint2 early[LISTS == kBeamFew ? kBeamEarly : 1];  // every part's first candidates
  double ent[LISTS == kBeamFew ? LISTS : 1];        // of the parts (LP_ENTROPY)
  int start[LISTS];                // of the parts that reach the bound: the number of their first candidate
  uint16_t list[LISTS];
  int found;
};

// A row's sums from its parts, by one wave.
template <int LISTS, bool ENT>
__device__ __forceinline__ RowSum beam_row_sum(const BeamJoinLds<LISTS>& lds, int parts, float& m, int lane) {
  m = -INFINITY;
  for (int i = lane; i < parts; i += 64) m = fmaxf(m, lds.part[i].max);
  m = wave_max_f32(m);
  RowSum r{0.0, 0.0};
  for (int i = lane; i < parts; i += 64) row_join(r, RowSum{lds.part[i].sum, ENT ? lds.ent[i] : 0.0}, lds.part[i].max, m);
  r.sum = wave_sum_f64(r.sum);
  if constexpr (ENT) r.ent = wave_sum_f64(r.ent);
  return r;
}

template <int DT, int LISTS, int THREADS, bool ONE, int LP>
__device__ __forceinline__ void beam_join(const BeamArgs& a, BeamJoinLds<LISTS>& lds, int req, int tid) {
  constexpr int RANKED = BeamJoinLds<LISTS>::RANKED;
  auto& state = lds.state;
  auto& rmax = lds.rmax;
  auto& rlog = lds.rlog;
  auto& rscore = lds.rscore;
  auto& best_of = lds.best_of;
  auto& taken = lds.taken;
  auto& found = lds.found;
  auto& part = lds.part;
  auto& list = lds.list;
  auto& start = lds.start;
  auto& keys = lds.keys;
  const int lane = tid & 63, wave = tid >> 6;
  const int W = a.beams, S = a.shares, k = a.k, lists = W * S;

  // LP: the last wave answers for the row, its token and the token's logit on their way beside the parts
  const bool answers = LP != LP_NONE && wave == THREADS / 64 - 1;
  int64_t token = -1;
  float own_logit = 0.0f, own_max = 0.0f;
  RowSum own_sum{0.0, 0.0};
  if (answers) token = row_token(a.answers, req);
  if (tid < kBeamClasses) best_of[tid] = 0;
  if (tid == 0) {
    found = 0;
    taken = 0;
  }
  // The parts' first candidates on their way with the parts, whatever of them
  // are there, so that the ones that reach the bound need no round trip of their own
  constexpr bool EARLY = ONE || LP != LP_NONE;
  int firsts = 0;
  uint2 e[EARLY ? kBeamEarly / THREADS : 1];
  if constexpr (EARLY) {
    firsts = min(kBeamEarly / lists, a.cap);
#pragma unroll
    for (int u = 0; u < kBeamEarly / THREADS; ++u) {
      const int i = min(tid + u * THREADS, lists * firsts - 1);
      e[u] = row_get<ONE>(a.cand + ((size_t)req * lists + i / firsts) * a.cap + i % firsts);
    }
  }
  for (int l = tid; l < lists; l += THREADS) {
    const BeamPart* p = a.parts + (size_t)req * lists + l;
    const uint2 u = row_get<ONE>(&p->sum), v = row_get<ONE>(&p->max);
    part[l].sum = two_words(u.x, u.y);
    part[l].max = __uint_as_float(v.x);
    part[l].count = (int)min(v.y, (uint32_t)a.cap);  // whatever is there, no candidate is read outside the workspace
    if constexpr (LP == LP_ENTROPY) {
      const uint2 t = row_get<ONE>(a.ents + (size_t)req * lists + l);
      lds.ent[l] = two_words(t.x, t.y);
    }
  }
  if (token >= 0 && token < a.vocab) own_logit = load_as_f32(a.logits, DT, (size_t)((int64_t)req * a.batch_stride + token));
  if constexpr (EARLY) {
#pragma unroll
    for (int u = 0; u < kBeamEarly / THREADS; ++u)
      if (tid + u * THREADS < lists * firsts) lds.early[tid + u * THREADS] = e[u];
  }
  if (tid < W) {
    const float sc = LP ? 0.0f : a.scores[(size_t)req * W + tid];
    state[tid] = LP ? BEAM_LIVE : beam_state(sc, a.finished && a.finished[(size_t)req * W + tid]);
    rscore[tid] = (double)sc;
  }
  __syncthreads();
  auto norm = [&](int w, float m, double t) NVJSEL_INLINE {  // a beam's maximum, and the sum relative to it
    const int st = !(t < INFINITY) ? BEAM_NAN : m == -INFINITY ? BEAM_DEAD : BEAM_LIVE;  // NaN: or an infinity; the mask leaves nothing
    state[w] = st;
    rmax[w] = m;
    rlog[w] = st != BEAM_LIVE ? 0.0 : LP ? row_log_sum(t) : log(t);
  };
  auto part_sum = [&](const BeamPart& p, float m) { return p.sum * exp((double)p.max - (m == -INFINITY ? 0.0 : (double)m)); };
  if constexpr (LP != LP_NONE) {  // one row
    if (wave == 0) {
      float m;
      const RowSum r = beam_row_sum<LISTS, false>(lds, S, m, lane);
      if (tid == 0) norm(0, m, r.sum);
    } else if (answers) {
      own_sum = beam_row_sum<LISTS, LP == LP_ENTROPY>(lds, S, own_max, lane);
    }
  } else if (S <= kBeamFewShares) {  // a lane each
    if (tid < W && state[tid] == BEAM_LIVE) {
      const BeamPart* p = part + tid * S;
      float m = -INFINITY;
      double t = 0.0;
      for (int i = 0; i < S; ++i) m = fmaxf(m, p[i].max);
      for (int i = 0; i < S; ++i) t += part_sum(p[i], m);
      norm(tid, m, t);
    }
  } else {  // a wave each
    for (int w = wave; w < W; w += (THREADS / 64)) {
      if (state[w] != BEAM_LIVE) continue;
      const BeamPart* p = part + w * S;
      float m = -INFINITY;
      double t = 0.0;
      for (int i = lane; i < S; i += 64) m = fmaxf(m, p[i].max);
      m = wave_max_f32(m);
      for (int i = lane; i < S; i += 64) t += part_sum(p[i], m);
      t = wave_sum_f64(t);
      if (lane == 0) norm(w, m, t);
    }
  }
  __syncthreads();
  if (answers && lane == 0) row_answer(a.answers, req, token >= 0 && token < a.vocab, own_logit, own_max, own_sum, rlog[0]);
  auto score = [&](int w, float x) { return rscore[w] + (((double)x - (double)rmax[w]) - rlog[w]); };

  // the parts' best scores by class; an ended beam's score counts with them
  auto put_best = [&](int l, double x) { atomicMax(&best_of[l % kBeamClasses], (uint32_t)(beam_ord(x) >> 32)); };
  for (int l = tid; l < lists; l += THREADS) {
    const int w = l / S;
    if (state[w] == BEAM_LIVE) {
      const float x = part[l].max;
      if (x > -INFINITY) put_best(l, score(w, x));
    } else if (state[w] == BEAM_ENDED && l % S == 0) {
      put_best(l, rscore[w]);
    }
  }
  __syncthreads();
  // to 12 bits of the score's mantissa
  uint64_t low = (uint64_t)wave_kth(best_of[lane], best_of[64 + lane], k, 8) << 32;

  auto scored = [&](int l, uint2 e) {  // a candidate of part l
    const int w = l / S;
    const float x = __uint_as_float(e.x);
    return BeamKey{score(w, x), beam_at(w, x, e.y)};
  };
  auto add = [&](const BeamKey& c) {
    if (beam_ord(c.s) < low) return;
    const int i = atomicAdd(&found, 1);
    if (i < RANKED) keys[i] = c;
  };
  for (int l = tid; l < lists; l += THREADS)
    if (state[l / S] == BEAM_LIVE && part[l].count > 0 && beam_ord(score(l / S, part[l].max)) >= low) {
      const unsigned long long at = atomicAdd(&taken, (unsigned long long)part[l].count << 32 | 1ull);
      list[(uint32_t)at] = (uint16_t)l;
      start[(uint32_t)at] = (int)(at >> 32);
    }
  __syncthreads();
  const int nl = (int)(uint32_t)taken, nc = (int)(taken >> 32);
  auto gather_by = [&](auto AHEAD, bool all) NVJSEL_INLINE {  // loads of a thread on their way together
    constexpr int N = decltype(AHEAD)::value;
    for (int i0 = tid; i0 < nc; i0 += N * THREADS) {
      if (!all && *(volatile int*)&found > RANKED) break;
      int of[N];
      uint2 c[N];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int i = min(i0 + u * THREADS, nc - 1);
        int lo = 0, hi = nl;  // the last list that starts at or before i
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (start[mid] <= i) lo = mid;
          else hi = mid;
        }
        of[u] = list[lo];
        const int j = i - start[lo];
        if (N == 1 && EARLY && j < firsts) c[u] = lds.early[of[u] * firsts + j];
        else c[u] = row_get<ONE>(a.cand + ((size_t)req * lists + of[u]) * a.cap + j);
      }
#pragma unroll
      for (int u = 0; u < N; ++u)
        if (i0 + u * THREADS < nc) add(scored(of[u], c[u]));
    }
  };
  auto gather = [&](bool all) NVJSEL_INLINE {  // or until there are too many to rank
    if (nc > 2 * THREADS) gather_by(std::integral_constant<int, 4>{}, all);
    else gather_by(std::integral_constant<int, 1>{}, all);
    if (tid < W && state[tid] == BEAM_ENDED) add(BeamKey{rscore[tid], beam_at(tid, 0.0f, (uint32_t)a.end_token)});
    __syncthreads();
  };
  gather(false);

  // Few parts bound badly, fewer than K not at all: the bound again, by the candidates' own
  // classes (18 requests, 8 beams, V = 2332, K = 16: 54 us with the 300 candidates ranked, 17 so)
  if (found > max(kBeamRefine, 3 * k)) {  // block-uniform
    static_assert(RANKED == 2 * THREADS, "");
    const int n = found;
    BeamKey mine[2] = {keys[tid], keys[tid + THREADS]};
    __syncthreads();
    if (tid < kBeamClasses) best_of[tid] = 0;
    if (tid == 0) found = 0;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (tid + h * THREADS < n) atomicMax(&best_of[tid % kBeamClasses], (uint32_t)(beam_ord(mine[h].s) >> 32));
    __syncthreads();
    const uint64_t t = (uint64_t)wave_kth(best_of[lane], best_of[64 + lane], k, 4) << 32;
    low = t > low ? t : low;
    if (n <= RANKED) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (tid + h * THREADS < n) add(mine[h]);
      __syncthreads();
    } else {
      gather(true);
    }
  }

  // NaN candidates come first, by place: every token of a NaN beam, the end token of an ended one
  int nan = 0;
  uint64_t nan_at = kBeamNone;
  const int own = lane < W ? state[lane] : BEAM_DEAD;
  for (uint64_t b = __ballot(own == BEAM_NAN || own == BEAM_ENDED_NAN); b && nan < k; b &= b - 1) {
    const int w = __builtin_ctzll(b), st = state[w];
    const int n = st == BEAM_NAN ? min(a.vocab, k - nan) : st == BEAM_ENDED_NAN ? 1 : 0;
    if (tid >= nan && tid < nan + n) nan_at = beam_at(w, 0.0f, (uint32_t)(st == BEAM_NAN ? tid - nan : a.end_token));
    nan += n;
  }
  auto put = [&](int j, const BeamKey& c) {
    const size_t o = (size_t)req * k + j;
    const bool none = c.at == kBeamNone;
    a.out_scores[o] = (float)c.s;
    if constexpr (!LP) a.out_parents[o] = none ? -1 : (int32_t)(c.at >> 58);
    a.out_tokens[o] = none ? -1 : (int32_t)(c.at & ((1ull << kBeamVocabBits) - 1));
  };
  if (tid < nan) put(tid, BeamKey{NAN, nan_at});

  const int n = found;
  if (n <= RANKED) {
    int each = 1;  // threads of a candidate
    while (each < 16 && 2 * each * n <= THREADS) each *= 2;
    for (int i0 = 0; i0 < n; i0 += THREADS / each) {
      const int i = i0 + tid / each;
      const BeamKey c = keys[i < n ? i : 0];
      int rank = 0;
      for (int j = tid & (each - 1); j < n; j += each) rank += beam_before(keys[j], c);
      for (int x = 1; x < each; x <<= 1) rank += __shfl_xor(rank, x, 64);
      if (i < n && (tid & (each - 1)) == 0 && nan + rank < k) put(nan + rank, c);
    }
    if (tid >= nan + n && tid < k) put(tid, BeamKey{-INFINITY, kBeamNone});
    return;
  }
  __syncthreads();
  BeamKey best{-INFINITY, kBeamNone};
  for (int l = wave; l < lists; l += (THREADS / 64)) {
    if (state[l / S] != BEAM_LIVE) continue;
    const int n = part[l].count;
    for (int j0 = 0; j0 < n; j0 += 64) {
      BeamKey c{-INFINITY, kBeamNone};
      if (j0 + lane < n) c = scored(l, row_get<ONE>(a.cand + ((size_t)req * lists + l) * a.cap + j0 + lane));
      if (!__any(beam_before(c, beam_from(best, k - 1)))) continue;
      beam_sort(c, lane);
      beam_merge(best, c, lane);
    }
  }
  if (wave == 0) {  // ended beams: one candidate each
    BeamKey c{-INFINITY, kBeamNone};
    if (lane < W && state[lane] == BEAM_ENDED) {
      c.s = rscore[lane];
      c.at = beam_at(lane, 0.0f, (uint32_t)a.end_token);
    }
    beam_sort(c, lane);
    beam_merge(best, c, lane);
  }
  keys[wave * 64 + lane] = best;
#pragma unroll
  for (int h = (THREADS / 64) / 2; h >= 1; h >>= 1) {
    __syncthreads();
    if (wave < h) {
      const BeamKey o = keys[(wave + h) * 64 + lane];
      beam_merge(best, o, lane);
      keys[wave * 64 + lane] = best;
    }
  }
  if (wave == 0 && nan + lane < k) put(nan + lane, best);
}

// One launch: the last block of a request to finish its parts joins them.
template <int DT, int LP>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_select_kernel(BeamArgs a) {
  using Join = BeamJoinLds<kBeamFew>;
  constexpr size_t room = sizeof(BeamScanLds) > sizeof(Join) ? sizeof(BeamScanLds) : sizeof(Join);
  __shared__ __attribute__((aligned(16))) char lds[room];
  __shared__ int last;
  const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int req = (int)blockIdx.x / a.blocks, l = (int)blockIdx.x % a.blocks * kBeamBlockWaves + wave;
  if (l < a.beams * a.shares) {
    const int row = req * a.beams + l / a.shares;
    if (LP || beam_state(a.scores[row], a.finished && a.finished[row]) == BEAM_LIVE)  // else its logits are not looked at
      beam_scan<DT, true, LP>(a, *(BeamScanLds*)lds, row, l % a.shares, wave, tid & 63);
  }
  // every wave's stores are performed before its block's ticket is drawn: the ticket is
  // behind the barrier, the barrier behind the wait
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) last = ticket_add(a.tickets + req) == (unsigned int)a.blocks - 1;
  __syncthreads();
  if (!last) return;
  if (tid == 0) __hip_atomic_store(a.tickets + req, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  beam_join<DT, kBeamFew, kBeamThreads, true, LP>(a, *(Join*)lds, req, tid);
}

template <int DT, int LP>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_scan_kernel(BeamArgs a) {
  __shared__ __attribute__((aligned(16))) BeamScanLds lds;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l = (int)blockIdx.x * kBeamBlockWaves + wave, row = l / a.shares;
  if (row >= a.batch * a.beams) return;
  if (!LP && beam_state(a.scores[row], a.finished && a.finished[row]) != BEAM_LIVE) return;  // its logits are not looked at
  beam_scan<DT, false, LP>(a, lds, row, l % a.shares, wave, (int)threadIdx.x & 63);
}

// LISTS: the parts of a request at most; rows that ask for log probabilities have up to kBeamFew.
// DT: for the token's own logit (LP).
template <int DT, int LISTS, int THREADS, int LP>
__global__ void __launch_bounds__(THREADS) beam_join_kernel(BeamArgs a) {
  __shared__ __attribute__((aligned(16))) BeamJoinLds<LISTS> lds;
  beam_join<DT, LISTS, THREADS, false, LP>(a, lds, (int)blockIdx.x, (int)threadIdx.x);
}

// Parts of a row: enough waves to fill the device, whole chunks each, and few
// enough lists (`most` of a request) for the join.
static void beam_split(int rows, int most, int vocab, int k, int dtype, int* shares, int* share, int* cap, int* group) {
  const int chunk = 64 * kBeamVecs * (dtype == DT_F32 ? 4 : 8);
  const int chunks = (vocab - 1) / chunk + 1;
  int64_t s = (int64_t)device_cu_count() * kBeamWaves / rows;
  if (s > most) s = most;
  if (s < 1) s = 1;
  if (s > chunks) s = chunks;
  const int per = (int)((chunks + s - 1) / s);
  *share = per * chunk;
  *group = (per + kBeamSlots - 1) / kBeamSlots;
  *shares = (chunks + per - 1) / per;
  *cap = k <= 32 ? 128 : 256;  // 30 expected at K = 24, 37 at 32, 89 at 64
}

// Scan and join, under the caller's lock.
template <int DT, int LP>
static int launch_beam(const BeamArgs& a, hipStream_t s) {
  constexpr int LISTS = LP ? kBeamFew : kBeamLists, THREADS = LP ? kBeamThreads : kBeamJoinThreads;
  const int64_t waves = (int64_t)a.batch * a.beams * a.shares;
  if (waves <= kBeamOne && a.beams * a.shares <= kBeamFew) {
    hipLaunchKernelGGL((beam_select_kernel<DT, LP>), dim3((unsigned)(a.batch * a.blocks)), dim3(kBeamThreads), 0, s, a);
    NVJSEL_CHECK_LAUNCH("beam_select_kernel");
    return NVJSEL_OK;
  }
  hipLaunchKernelGGL((beam_scan_kernel<DT, LP>), dim3((unsigned)((waves + kBeamBlockWaves - 1) / kBeamBlockWaves)),
                     dim3(kBeamThreads), 0, s, a);
  NVJSEL_CHECK_LAUNCH("beam_scan_kernel");
  hipLaunchKernelGGL((beam_join_kernel<LP ? DT : DT_F32, LISTS, THREADS, LP>), dim3((unsigned)a.batch), dim3(THREADS), 0, s, a);
  NVJSEL_CHECK_LAUNCH("beam_join_kernel");
  return NVJSEL_OK;
}

}  // namespace nvjsel
