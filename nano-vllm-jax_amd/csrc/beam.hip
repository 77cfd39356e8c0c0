// Beam search's selection over beams and vocabulary, and the reordering of the
// beams' states that follows it.
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
#include <float.h>

#include "nvjsel_device.h"
#include "nvjsel_host.h"

namespace nvjsel {

typedef uint32_t bm_u32x4 __attribute__((ext_vector_type(4)));
typedef bm_u32x4 bm_u32x4_any __attribute__((aligned(1)));  // 16 bytes from any address
typedef uint32_t bm_u32_any __attribute__((aligned(1)));

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
  float* out_scores;
  int32_t* out_parents;
  int32_t* out_tokens;
};

// Parts and candidates, 8 bytes at a time.  ONE: they pass between blocks of one launch,
// on any XCDs, written and read at the device's coherence point (agent scope).
template <bool ONE>
__device__ __forceinline__ void beam_put(void* p, uint32_t lo, uint32_t hi) {
  const unsigned long long v = (unsigned long long)hi << 32 | lo;
  if constexpr (ONE) __hip_atomic_store((unsigned long long*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else *(unsigned long long*)p = v;
}
template <bool ONE>
__device__ __forceinline__ uint2 beam_get(const void* p) {
  unsigned long long v;
  if constexpr (ONE) v = __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else v = *(const unsigned long long*)p;
  return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
}

// What a beam contributes: nothing, every token, one token, or NaN.
enum { BEAM_DEAD = 0, BEAM_LIVE = 1, BEAM_ENDED = 2, BEAM_NAN = 3, BEAM_ENDED_NAN = 4 };

__device__ __forceinline__ int beam_state(float score, bool ended) {
  if (score == -INFINITY) return BEAM_DEAD;
  if (!(score < INFINITY)) return ended ? BEAM_ENDED_NAN : BEAM_NAN;
  return ended ? BEAM_ENDED : BEAM_LIVE;
}

template <int DT>
struct BeamElems {
  static constexpr int N = DT == DT_F32 ? 4 : 8;  // elements of a 16-byte piece
  __device__ static __forceinline__ float get(const bm_u32x4& w, int e) {
    if constexpr (DT == DT_F32) return __uint_as_float(w[e]);
    else if constexpr (DT == DT_BF16) return __uint_as_float(e & 1 ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
    else return f16_to_f32((uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu));
  }
  __device__ static __forceinline__ uint32_t none() {  // -inf in every element of a word
    return DT == DT_F32 ? 0xFF800000u : DT == DT_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
  }
};

__device__ __forceinline__ float readlane_f(float v, int l) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l));
}
// Maximum and sum over a wave without LDS: rotations in rows of 16, then the rows' and
// halves' swaps.
template <int N>
__device__ __forceinline__ uint32_t row_ror(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xF, 0xF, false);
}
__device__ __forceinline__ float wave_max_f32(float v) {
  v = fmaxf(v, __uint_as_float(row_ror<8>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(row_ror<4>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(row_ror<2>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(row_ror<1>(__float_as_uint(v))));
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return xor32_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ double two_words(uint32_t lo, uint32_t hi) {
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
template <int N>
__device__ __forceinline__ double row_ror_add(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  return v + two_words(row_ror<N>((uint32_t)u), row_ror<N>((uint32_t)(u >> 32)));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  v = row_ror_add<1>(row_ror_add<2>(row_ror_add<4>(row_ror_add<8>(v))));
  uint64_t u = (uint64_t)__double_as_longlong(v);
  auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
  auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
  v = two_words(lo[0], hi[0]) + two_words(lo[1], hi[1]);
  u = (uint64_t)__double_as_longlong(v);
  lo = __builtin_amdgcn_permlane32_swap((uint32_t)u, (uint32_t)u, false, false);
  hi = __builtin_amdgcn_permlane32_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
  return two_words(lo[0], hi[0]) + two_words(lo[1], hi[1]);
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
// Exponentials are the hardware's exp2 (about 1 ulp) of fma(x, log2 e, -ref): one
// rounding of the difference.  ref is a whole number next to a lane's maximum times log2 e,
// so that a sum moves from one reference to another by its exponent alone, exactly, however
// often its maximum rises.  That holds for maxima up to this size; the reference stays
// within it, and a share whose own maximum does not is summed again (beam_sum_far).
static constexpr float kLog2e = 1.44269504088896341f, kBeamFar = 16384.0f;
__device__ __forceinline__ float beam_ref(float m) { return rintf(fminf(fmaxf(m, -kBeamFar), kBeamFar) * kLog2e); }
// sum, relative to 2^from, relative to 2^to.
__device__ __forceinline__ double beam_move(double sum, float from, float to) {
  return __builtin_amdgcn_ldexp(sum, (int)(from - to));
}
// The sum of N numbers, a power of two, in log2 N roundings.
template <int N>
__device__ __forceinline__ float sum_tree(const float (&t)[N]) {
  if constexpr (N == 1) {
    return t[0];
  } else {
    float u[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) u[i] = t[2 * i] + t[2 * i + 1];
    return sum_tree(u);
  }
}

// The piece at element o of a share that ends at e1; -inf past the end.
template <int DT>
__device__ __forceinline__ bm_u32x4 beam_piece(const char* base, int o, int e1) {
  using E = BeamElems<DT>;
  if (o + E::N <= e1) return *(const bm_u32x4_any*)(base + (size_t)o * (DT == DT_F32 ? 4 : 2));
  bm_u32x4 t;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t x = E::none();
    if constexpr (DT == DT_F32) {
      if (o + q < e1) x = ((const uint32_t*)base)[o + q];
    } else {
      if (o + 2 * q < e1) x = (x & 0xFFFF0000u) | ((const uint16_t*)base)[o + 2 * q];
      if (o + 2 * q + 1 < e1) x = (x & 0xFFFFu) | (uint32_t)((const uint16_t*)base)[o + 2 * q + 1] << 16;
    }
    t[q] = x;
  }
  return t;
}

// The sum of exp(l - m) of a share whose maximum m is known, a lane's part.
template <int DT>
__device__ __forceinline__ double beam_sum_far(const char* base, int e0, int e1, float m, int lane) {
  using E = BeamElems<DT>;
  double sum = 0.0;
  for (int o = e0 + lane * E::N; o < e1; o += 64 * E::N) {
    const bm_u32x4 w = beam_piece<DT>(base, o, e1);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E::N; ++e) s += __builtin_amdgcn_exp2f((E::get(w, e) - m) * kLog2e);
    sum += (double)s;
  }
  return sum;
}

// The K best logits of a share exactly, one lane each in order, where too many
// logits reach the bound that the scan takes from its lanes' maxima: a row of equal
// or masked values.  A token enters by comparing all lanes at once; tokens are
// visited in order of index and enter only above the K-th value, so among equal
// logits the lowest indices stay, and a row of equal logits costs K entries.
template <int DT>
__device__ __forceinline__ void beam_best(const char* base, int e0, int e1, int k, int lane, float& val, uint32_t& idx) {
  using E = BeamElems<DT>;
  val = -INFINITY;
  idx = 0xFFFFFFFFu;
  float thr = -INFINITY;
  for (int c0 = e0; c0 < e1; c0 += 64 * E::N) {
    const bm_u32x4 w = beam_piece<DT>(base, c0 + lane * E::N, e1);
    float gm = E::get(w, 0);
#pragma unroll
    for (int e = 1; e < E::N; ++e) gm = fmaxf(gm, E::get(w, e));
    uint64_t hit = __ballot(gm > thr);
    while (hit) {
      const int l = __builtin_ctzll(hit);
      bm_u32x4 t;
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
  bm_u32x4 aside[kBeamBlockWaves][kBeamHeld][kBeamVecs];  // or, read again: the (slot, lane) pairs
  int aside_at[kBeamBlockWaves][kBeamHeld];               // their first element
};
static_assert(sizeof(bm_u32x4) * kBeamHeld * kBeamVecs >= kBeamSlots * 64 * sizeof(uint16_t), "");

template <int DT, bool ONE>
__device__ __forceinline__ void beam_scan(const BeamArgs& a, BeamScanLds& lds, int row, int part, int wave, int lane) {
  using E = BeamElems<DT>;
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

  float m = -INFINITY, ref = beam_ref(-INFINITY), kept = -INFINITY;
  double sum = 0.0;                        // relative to 2^ref
  float half[2] = {-INFINITY, -INFINITY};  // the maximum by pieces: the first and the last ones of every chunk
  float bound = -FLT_MAX;                  // of the candidates: -inf is none
  int taken = 0, held = 0;                 // chunks; pieces set aside
  auto find_bound = [&]() NVJSEL_INLINE {  // in 16 bits of the order: bf16's own, and as good a bound for the others
    const uint32_t t = k <= kBeamOneMax ? wave_kth(ord_f32(m), 0u, k, 16) : wave_kth(ord_f32(half[0]), ord_f32(half[1]), k, 16);
    bound = t <= ord_f32(-INFINITY) ? -FLT_MAX : unord_f32(t);
  };
  int slot = 0, more = a.group;
  auto take = [&](const bm_u32x4 (&w)[kBeamVecs]) NVJSEL_INLINE {  // chunk `taken` of the share
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
    const float to = __builtin_elementwise_maximum(m, x), to_ref = beam_ref(to);
    // a chunk's terms in five roundings at most, from zero: added to the sum of the chunks
    // before, the small ones of a long share would be lost (one large logit and 122 chunks
    // of small ones: scores off by 9e-5 so)
    float s[kBeamVecs];
#pragma unroll
    for (int j = 0; j < kBeamVecs; ++j) {
      float t[N];
#pragma unroll
      for (int e = 0; e < N; ++e) t[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(E::get(w[j], e), kLog2e, -to_ref));
      s[j] = sum_tree(t);
    }
    sum = beam_move(sum, ref, to_ref) + (double)sum_tree(s);
    m = to;
    ref = to_ref;
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
    bm_u32x4 w[DEPTH][kBeamVecs];
    int next = 0;
    auto load = [&](auto D) NVJSEL_INLINE {  // always a load: the last full chunk again at the end
      const char* p = base + ((size_t)e0 + (size_t)(next < full ? next : full - 1) * CHUNK + (size_t)lane * N) * es;
#pragma unroll
      for (int j = 0; j < kBeamVecs; ++j) w[decltype(D)::value][j] = __builtin_nontemporal_load((const bm_u32x4_any*)(p + j * 1024));
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
    bm_u32x4 w[kBeamVecs];
#pragma unroll
    for (int j = 0; j < kBeamVecs; ++j) w[j] = beam_piece<DT>(base, e0 + full * CHUNK + (j * 64 + lane) * N, e1);
    take(w);
  }

  const float wm = wave_max_f32(m);
  double total;
  if (wm <= kBeamFar && (wm >= 100.0f - kBeamFar || wm == -INFINITY)) {
    const float wref = beam_ref(wm);
    total = wave_sum_f64(beam_move(sum, ref, wref));  // a NaN's sum is NaN
    // relative to exp(wm) now: exp(d), |d| < 0.35, by its series (to 2^-32)
    const double d = wm == -INFINITY ? 0.0 : ((double)wref - (double)wm * (double)kLog2e) * 0.6931471805599453;
    double f = 1.0;
#pragma unroll
    for (int i = 8; i >= 1; --i) f = __builtin_fma(f, d * (1.0 / i), 1.0);
    total *= f;
  } else {
    total = wave_sum_f64(beam_sum_far<DT>(base, e0, e1, wm, lane));
  }

  if (taken & (taken - 1)) find_bound();  // else it is of all chunks already
  uint2* cand = a.cand + (size_t)wid * a.cap;
  int count = 0;
  auto collect = [&](const bm_u32x4& w, int o) NVJSEL_INLINE {  // the candidates of a piece per lane
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
        beam_put<ONE>(cand + at, __float_as_uint(x), (uint32_t)(o + e));
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
      bm_u32x4 w{E::none(), E::none(), E::none(), E::none()};
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
        collect(beam_piece<DT>(base, o, e1), o);
      }
    }
  }
  if (count > a.cap) {
    float val;
    uint32_t idx;
    beam_best<DT>(base, e0, e1, k, lane, val, idx);
    const uint64_t b = __ballot(lane < k && val > -INFINITY);
    if (b >> lane & 1) beam_put<ONE>(cand + lane, __float_as_uint(val), idx);
    count = __builtin_popcountll(b);
  }
  if (lane == 0) {
    const uint64_t u = (uint64_t)__double_as_longlong(total);
    beam_put<ONE>(&a.parts[wid].sum, (uint32_t)u, (uint32_t)(u >> 32));
    beam_put<ONE>(&a.parts[wid].max, __float_as_uint(wm), (uint32_t)count);
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
  int start[LISTS];                // of the parts that reach the bound: the number of their first candidate
  uint16_t list[LISTS];
  int found;
};

template <int LISTS, int THREADS, bool ONE>
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

  if (tid < kBeamClasses) best_of[tid] = 0;
  if (tid == 0) {
    found = 0;
    taken = 0;
  }
  // One launch: the parts' first candidates on their way with the parts, whatever of them
  // are there, so that the ones that reach the bound need no round trip of their own
  int firsts = 0;
  uint2 e[ONE ? kBeamEarly / THREADS : 1];
  if constexpr (ONE) {
    firsts = min(kBeamEarly / lists, a.cap);
#pragma unroll
    for (int u = 0; u < kBeamEarly / THREADS; ++u) {
      const int i = min(tid + u * THREADS, lists * firsts - 1);
      e[u] = beam_get<ONE>(a.cand + ((size_t)req * lists + i / firsts) * a.cap + i % firsts);
    }
  }
  for (int l = tid; l < lists; l += THREADS) {
    const BeamPart* p = a.parts + (size_t)req * lists + l;
    const uint2 u = beam_get<ONE>(&p->sum), v = beam_get<ONE>(&p->max);
    part[l].sum = two_words(u.x, u.y);
    part[l].max = __uint_as_float(v.x);
    part[l].count = (int)min(v.y, (uint32_t)a.cap);  // whatever is there, no candidate is read outside the workspace
  }
  if constexpr (ONE) {
#pragma unroll
    for (int u = 0; u < kBeamEarly / THREADS; ++u)
      if (tid + u * THREADS < lists * firsts) lds.early[tid + u * THREADS] = e[u];
  }
  if (tid < W) {
    const float sc = a.scores[(size_t)req * W + tid];
    state[tid] = beam_state(sc, a.finished && a.finished[(size_t)req * W + tid]);
    rscore[tid] = (double)sc;
  }
  __syncthreads();
  auto norm = [&](int w, float m, double t) NVJSEL_INLINE {  // a beam's maximum, and the sum relative to it
    const int st = !(t < INFINITY) ? BEAM_NAN : m == -INFINITY ? BEAM_DEAD : BEAM_LIVE;  // NaN: or an infinity; the mask leaves nothing
    state[w] = st;
    rmax[w] = m;
    rlog[w] = st == BEAM_LIVE ? log(t) : 0.0;
  };
  auto part_sum = [&](const BeamPart& p, float m) { return p.sum * exp((double)p.max - (m == -INFINITY ? 0.0 : (double)m)); };
  if (S <= kBeamFewShares) {  // a lane each
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
        if (N == 1 && ONE && j < firsts) c[u] = lds.early[of[u] * firsts + j];
        else c[u] = beam_get<ONE>(a.cand + ((size_t)req * lists + of[u]) * a.cap + j);
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
    a.out_parents[o] = none ? -1 : (int32_t)(c.at >> 58);
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
      if (j0 + lane < n) c = scored(l, beam_get<ONE>(a.cand + ((size_t)req * lists + l) * a.cap + j0 + lane));
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
template <int DT>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_select_kernel(BeamArgs a) {
  using Join = BeamJoinLds<kBeamFew>;
  constexpr size_t room = sizeof(BeamScanLds) > sizeof(Join) ? sizeof(BeamScanLds) : sizeof(Join);
  __shared__ __attribute__((aligned(16))) char lds[room];
  __shared__ int last;
  const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int req = (int)blockIdx.x / a.blocks, l = (int)blockIdx.x % a.blocks * kBeamBlockWaves + wave;
  if (l < a.beams * a.shares) {
    const int row = req * a.beams + l / a.shares;
    if (beam_state(a.scores[row], a.finished && a.finished[row]) == BEAM_LIVE)  // else its logits are not looked at
      beam_scan<DT, true>(a, *(BeamScanLds*)lds, row, l % a.shares, wave, tid & 63);
  }
  // every wave's stores are performed before its block's ticket is drawn: the ticket is
  // behind the barrier, the barrier behind the wait
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) last = ticket_add(a.tickets + req) == (unsigned int)a.blocks - 1;
  __syncthreads();
  if (!last) return;
  if (tid == 0) __hip_atomic_store(a.tickets + req, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  beam_join<kBeamFew, kBeamThreads, true>(a, *(Join*)lds, req, tid);
}

template <int DT>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_scan_kernel(BeamArgs a) {
  __shared__ __attribute__((aligned(16))) BeamScanLds lds;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l = (int)blockIdx.x * kBeamBlockWaves + wave, row = l / a.shares;
  if (row >= a.batch * a.beams) return;
  if (beam_state(a.scores[row], a.finished && a.finished[row]) != BEAM_LIVE) return;  // its logits are not looked at
  beam_scan<DT, false>(a, lds, row, l % a.shares, wave, (int)threadIdx.x & 63);
}

__global__ void __launch_bounds__(kBeamJoinThreads) beam_join_kernel(BeamArgs a) {
  __shared__ __attribute__((aligned(16))) BeamJoinLds<kBeamLists> lds;
  beam_join<kBeamLists, kBeamJoinThreads, false>(a, lds, (int)blockIdx.x, (int)threadIdx.x);
}

// Parts of a row: enough waves to fill the device, whole chunks each, and few
// enough lists for the join.
static void beam_split(int rows, int beams, int vocab, int k, int dtype, int* shares, int* share, int* cap,
                       int* group) {
  const int chunk = 64 * kBeamVecs * (dtype == DT_F32 ? 4 : 8);
  const int chunks = (vocab - 1) / chunk + 1;
  int64_t s = (int64_t)device_cu_count() * kBeamWaves / rows;
  const int64_t most = kBeamLists / beams;
  if (s > most) s = most;
  if (s < 1) s = 1;
  if (s > chunks) s = chunks;
  const int per = (int)((chunks + s - 1) / s);
  *share = per * chunk;
  *group = (per + kBeamSlots - 1) / kBeamSlots;
  *shares = (chunks + per - 1) / per;
  *cap = k <= 32 ? 128 : 256;  // 30 expected at K = 24, 37 at 32, 89 at 64
}

static size_t beam_bytes(int batch, int beams, int shares, int cap) {
  return kBeamRequests * 4 + (size_t)batch * beams * shares * (sizeof(BeamPart) + cap * sizeof(uint2));
}

template <int DT>
static int launch_beam(const BeamArgs& a, hipStream_t s) {
  const int64_t waves = (int64_t)a.batch * a.beams * a.shares;
  std::lock_guard<std::mutex> lock(launch_mutex());
  if (waves <= kBeamOne && a.beams * a.shares <= kBeamFew) {
    hipLaunchKernelGGL(beam_select_kernel<DT>, dim3((unsigned)(a.batch * a.blocks)), dim3(kBeamThreads), 0, s, a);
    NVJSEL_CHECK_LAUNCH("beam_select_kernel");
    return NVJSEL_OK;
  }
  hipLaunchKernelGGL(beam_scan_kernel<DT>, dim3((unsigned)((waves + kBeamBlockWaves - 1) / kBeamBlockWaves)),
                     dim3(kBeamThreads), 0, s, a);
  NVJSEL_CHECK_LAUNCH("beam_scan_kernel");
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)a.batch), dim3(kBeamJoinThreads), 0, s, a);
  NVJSEL_CHECK_LAUNCH("beam_join_kernel");
  return NVJSEL_OK;
}

// ---------------------------------------------------------------- state reordering

static constexpr int kReorderTensors = 24;  // of one launch, in its arguments

struct ReorderTensor {
  char* data;
  int64_t row_bytes;   // from one row to the next
  int64_t span;        // contiguous bytes of a row, or of each outer index with lengths
  int64_t token;       // bytes of one position, 0 without lengths
  int outer;
  int rows;
  int chunks;          // blocks of each span
};

struct ReorderArgs {
  ReorderTensor t[kReorderTensors];
  const int32_t* parents;
  int64_t parent_stride;
  const int32_t* slots;    // [batch, beams] or null
  const int32_t* lengths;  // [batch] or null
  int beams;
};

// state[slot(b, w)] = old state[slot(b, parent(b, w))] in place.  A thread owns the
// same bytes of all beams of its request: it loads every moved beam's new value,
// then stores them, so no order of the moves matters and nothing waits for
// another thread.  Beams that keep their place are not touched.  Memory bound:
// each moved beam is written once; a source that several beams take comes from
// the cache after its first read.  The loads of W beams are in flight together, 16
// bytes a lane up to 16 beams and 4 above, so that they fit the registers.  Written and
// read, 12 f32 states of 64 rows x 1 MB, of the bytes that random parents move: 4 and 8
// beams 5.2 TB/s (1.12 GB 214 us; a large copy runs at 5.1), 16 beams 4.9, 17 to 64 beams, with
// 4 bytes a lane, 3.1 to 3.7.
template <int VEC, int WREG>
__global__ void __launch_bounds__(256) reorder_kernel(ReorderArgs a) {
  typedef typename std::conditional<VEC == 16, bm_u32x4, uint32_t>::type Vec;
  typedef typename std::conditional<VEC == 16, bm_u32x4_any, bm_u32_any>::type Any;
  const ReorderTensor& t = a.t[blockIdx.z];
  const int req = (int)blockIdx.y, W = a.beams;
  const int o = (int)blockIdx.x / t.chunks;
  if (o >= t.outer) return;
  int64_t valid = t.span;
  if (t.token) {
    const int64_t n = (int64_t)a.lengths[req] * t.token;
    valid = n < valid ? n : valid;
  }
  const int64_t at = ((int64_t)((int)blockIdx.x - o * t.chunks) * 256 + threadIdx.x) * VEC;
  if (at >= valid) return;
  char* base = t.data + (int64_t)o * t.span + at;

  const int32_t* __restrict__ parents = a.parents + (int64_t)req * a.parent_stride;
  const int32_t* __restrict__ slots = a.slots;
  auto slot = [&](int w) -> int { return slots ? slots[req * W + w] : req * W + w; };
  auto source = [&](int w) -> int {  // the row that beam w takes, -1: it stays as it is
    if (w >= W) return -1;
    const int p = parents[w];
    if (p < 0 || p >= W || p == w) return -1;
    const int to = slot(w), from = slot(p);
    return to < 0 || to >= t.rows || from < 0 || from >= t.rows ? -1 : from;
  };
  if (at + VEC <= valid) {
    Vec v[WREG];
    uint64_t moved = 0;
#pragma unroll
    for (int w = 0; w < WREG; ++w) {
      const int s = source(w);
      if (s >= 0) {
        v[w] = *(const Any*)(base + s * t.row_bytes);
        moved |= 1ull << w;
      }
    }
#pragma unroll
    for (int w = 0; w < WREG; ++w)
      if (moved >> w & 1) *(Any*)(base + slot(w) * t.row_bytes) = v[w];
  } else {  // the last bytes
    for (int64_t i = 0; i < valid - at; ++i) {
      uint8_t v[WREG];
      uint64_t moved = 0;
#pragma unroll
      for (int w = 0; w < WREG; ++w) {
        const int s = source(w);
        if (s >= 0) {
          v[w] = ((const uint8_t*)base)[s * t.row_bytes + i];
          moved |= 1ull << w;
        }
      }
#pragma unroll
      for (int w = 0; w < WREG; ++w)
        if (moved >> w & 1) ((uint8_t*)base)[slot(w) * t.row_bytes + i] = v[w];
    }
  }
}

template <int VEC, int WREG>
static int launch_reorder(const ReorderArgs& a, int count, int batch, int64_t blocks, hipStream_t s) {
  hipLaunchKernelGGL((reorder_kernel<VEC, WREG>), dim3((unsigned)blocks, (unsigned)batch, (unsigned)count), dim3(256), 0, s,
                     a);
  NVJSEL_CHECK_LAUNCH("reorder_kernel");
  return NVJSEL_OK;
}

}  // namespace nvjsel

using namespace nvjsel;

static int beam_check(const char* who, int dtype, int batch, int beams, int vocab, int k) {
  if (batch <= 0 || beams <= 0 || vocab <= 0) {
    set_error("%s requires non-empty dimensions (batch=%d beams=%d vocab=%d)", who, batch, beams, vocab);
    return NVJSEL_EINVAL;
  }
  if (!valid_dtype(dtype)) { set_error("%s: unsupported logits dtype %d", who, dtype); return NVJSEL_EINVAL; }
  if (beams > kBeamMax || k < 1 || k > kBeamMax) {
    set_error("%s: beams (%d) and candidates (%d) must be in 1..%d", who, beams, k, kBeamMax);
    return NVJSEL_EINVAL;
  }
  if (vocab > (1 << kBeamVocabBits) || batch > kBeamRequests) {
    set_error("%s: vocab (%d) must be at most 2^26, batch (%d) at most 65536", who, vocab, batch);
    return NVJSEL_EINVAL;
  }
  return NVJSEL_OK;
}

extern "C" size_t nvjsel_beam_select_workspace_size(int dtype, int batch, int beams, int vocab, int k) {
  if (beam_check("beam_select", dtype, batch, beams, vocab, k) != NVJSEL_OK) return 0;
  int shares, share, cap, group;
  beam_split(batch * beams, beams, vocab, k, dtype, &shares, &share, &cap, &group);
  return beam_bytes(batch, beams, shares, cap);
}

extern "C" int nvjsel_beam_select(const void* logits, int dtype, int batch, int beams, int vocab, int64_t batch_stride,
                                  int64_t beam_stride, const float* scores, const uint8_t* finished, int end_token, int k,
                                  float* out_scores, int32_t* out_parents, int32_t* out_tokens, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  clear_error();
  const int rc = beam_check("beam_select", dtype, batch, beams, vocab, k);
  if (rc != NVJSEL_OK) return rc;
  if (!logits || !scores || !out_scores || !out_parents || !out_tokens)
    return fail(NVJSEL_EINVAL, "beam_select: null pointer");
  if (((uintptr_t)logits) & (dtype_size(dtype) - 1)) return fail(NVJSEL_EINVAL, "beam_select: unaligned logits");
  if (beam_stride < 0 || batch_stride < 0) return fail(NVJSEL_EINVAL, "beam_select: negative stride");
  if (finished && (end_token < 0 || end_token >= vocab))
    return fail(NVJSEL_EINVAL, "beam_select: end token outside the vocabulary");
  BeamArgs a{};
  a.logits = logits;
  a.batch = batch;
  a.beams = beams;
  a.vocab = vocab;
  a.k = k;
  a.batch_stride = batch_stride;
  a.beam_stride = beam_stride;
  a.scores = scores;
  a.finished = finished;
  a.end_token = end_token;
  beam_split(batch * beams, beams, vocab, k, dtype, &a.shares, &a.share, &a.cap, &a.group);
  const size_t need = beam_bytes(batch, beams, a.shares, a.cap);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) {
    set_error("beam_select: workspace %zu bytes (16-byte aligned) < required %zu", workspace_bytes, need);
    return NVJSEL_EWORKSPACE;
  }
  a.tickets = (unsigned int*)workspace;
  a.blocks = (beams * a.shares + kBeamBlockWaves - 1) / kBeamBlockWaves;
  a.parts = (BeamPart*)((char*)workspace + kBeamRequests * 4);
  a.cand = (uint2*)(a.parts + (size_t)batch * beams * a.shares);
  a.out_scores = out_scores;
  a.out_parents = out_parents;
  a.out_tokens = out_tokens;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DT_F32) return launch_beam<DT_F32>(a, s);
  if (dtype == DT_BF16) return launch_beam<DT_BF16>(a, s);
  return launch_beam<DT_F16>(a, s);
}

extern "C" int nvjsel_reorder_states(const nvjsel_state* states, int count, const int32_t* parents, int64_t parent_stride,
                                     const int32_t* slots, const int32_t* lengths, int batch, int beams, void* stream) {
  clear_error();
  if (!states || !parents) return fail(NVJSEL_EINVAL, "reorder_states: null pointer");
  if (count <= 0 || batch <= 0 || beams <= 0) return fail(NVJSEL_EINVAL, "reorder_states requires non-empty dimensions");
  if (beams > kBeamMax || batch > 65535) {
    set_error("reorder_states: beams (%d) must be at most %d, batch (%d) at most 65535", beams, kBeamMax, batch);
    return NVJSEL_EINVAL;
  }
  if (parent_stride < 0) return fail(NVJSEL_EINVAL, "reorder_states: negative stride");
  for (int i = 0; i < count; ++i) {
    const nvjsel_state& t = states[i];
    if (!t.data || t.rows <= 0 || t.outer <= 0 || t.length <= 0 || t.token_bytes <= 0)
      return fail(NVJSEL_EINVAL, "reorder_states: empty state");
    if (t.length > (int64_t)1 << 40 || t.token_bytes > (int64_t)1 << 40 || t.length * (__int128)t.token_bytes * t.outer > t.row_bytes)
      return fail(NVJSEL_EINVAL, "reorder_states: rows overlap");
    if (!slots && t.rows < batch * (int64_t)beams)
      return fail(NVJSEL_EINVAL, "reorder_states: fewer rows than batch x beams");
  }
  const int vec = beams <= 16 ? 16 : 4;
  auto describe = [&](const nvjsel_state& t) {
    ReorderTensor r{};
    r.data = (char*)t.data;
    r.row_bytes = t.row_bytes;
    r.rows = t.rows;
    r.token = lengths ? t.token_bytes : 0;
    r.outer = lengths ? t.outer : 1;
    r.span = t.length * t.token_bytes * (lengths ? 1 : t.outer);
    const int64_t c = (r.span + 256 * vec - 1) / (256 * vec);
    r.chunks = c * (__int128)r.outer > 0xFFFFFF ? 0 : (int)c;  // 0: more than 2^32 threads
    return r;
  };
  for (int i = 0; i < count; ++i)  // of all of them, before any is moved
    if (describe(states[i]).chunks == 0) return fail(NVJSEL_EINVAL, "reorder_states: state too large");
  for (int i0 = 0; i0 < count; i0 += kReorderTensors) {
    const int n = count - i0 < kReorderTensors ? count - i0 : kReorderTensors;
    ReorderArgs a{};
    int64_t blocks = 1;
    for (int i = 0; i < n; ++i) {
      a.t[i] = describe(states[i0 + i]);
      const int64_t b = (int64_t)a.t[i].chunks * a.t[i].outer;
      if (b > blocks) blocks = b;
    }
    a.parents = parents;
    a.parent_stride = parent_stride;
    a.slots = slots;
    a.lengths = lengths;
    a.beams = beams;
    hipStream_t s = (hipStream_t)stream;
    const int rc = beams <= 4    ? launch_reorder<16, 4>(a, n, batch, blocks, s)
                   : beams <= 8  ? launch_reorder<16, 8>(a, n, batch, blocks, s)
                   : beams <= 16 ? launch_reorder<16, 16>(a, n, batch, blocks, s)
                                 : launch_reorder<4, 64>(a, n, batch, blocks, s);
    if (rc != NVJSEL_OK) return rc;
  }
  return NVJSEL_OK;
}
