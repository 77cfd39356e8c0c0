// Beam search's selection over beams and vocabulary, and the reordering of the
// beams' states that follows it.
//
//   candidate (w, v) of request b:  S[b,w] + (l[b,w,v] - m) - log sum_v' exp(l[b,w,v'] - m),  m = max_v' l[b,w,v']
//
// the K best over all w and v, by value, then by w V + v.  Within a row the order
// is the logits' own, so one pass over them keeps each part's K largest logits
// beside its maximum and its sum of exponentials (beam_scan_kernel), and a second
// kernel, one block per request, joins the parts, turns the survivors into
// scores in fp64 and ranks them (beam_select_kernel).  fp64 there because two
// beams' candidates may lie closer than an fp32 score resolves; the sums of
// exponentials are fp32 within a lane and fp64 across lanes and parts.
#include "nvjsel_device.h"
#include "nvjsel_host.h"

namespace nvjsel {

typedef uint32_t bm_u32x4 __attribute__((ext_vector_type(4)));
typedef bm_u32x4 bm_u32x4_any __attribute__((aligned(1)));  // 16 bytes from any address
typedef uint32_t bm_u32_any __attribute__((aligned(1)));

static constexpr int kBeamMax = 64;        // beams and candidates per request: one lane each
static constexpr int kBeamVecs = 8;        // 16-byte pieces per lane and chunk
static constexpr int kBeamScanThreads = 256;
static constexpr int kBeamSelectWaves = 16;

struct BeamPart {  // of one wave's share of a row
  double sum;      // sum of exp(l - max)
  float max;
  float pad;
};

struct BeamArgs {
  const void* logits;
  int batch, beams, vocab, k;
  int64_t batch_stride, beam_stride;  // elements
  const float* scores;      // [batch, beams]
  const uint8_t* finished;  // [batch, beams] or null
  int end_token;
  int shares, share;  // parts of a row, and their length in elements (whole chunks)
  BeamPart* parts;    // [batch beams shares]
  uint2* cand;        // [batch beams shares][k]: logit bits, token
  float* out_scores;
  int32_t* out_parents;
  int32_t* out_tokens;
};

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
__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}

// Sorts a wave's 64 values, the largest in lane 0 (bitonic).
__device__ __forceinline__ float wave_sort_desc(float v, int lane) {
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d >= 1; d >>= 1) {
      const float o = __shfl_xor(v, d, 64);
      const bool up = (lane & size) == 0, low = (lane & d) == 0;  // up: the larger value to the lower lane
      v = (up == low) ? fmaxf(v, o) : fminf(v, o);
    }
  return v;
}

// One share of a row per wave, in chunks of 64 lanes x kBeamVecs pieces that stay
// in registers: their maximum, their exponentials, and every logit above the
// K-th largest so far.  The K best so far lie in lanes 0 .. K - 1 in order; a
// token enters by comparing all lanes at once.  The first chunk starts from the
// K-th largest of the 64 lanes' maxima (at least K logits reach it), so that few
// tokens enter.  Tokens are visited in order of index and enter only above the
// K-th value, so among equal logits the lowest indices stay, and a row of equal
// logits costs no more than another.
template <int DT>
__global__ void __launch_bounds__(kBeamScanThreads) beam_scan_kernel(BeamArgs a) {
  using E = BeamElems<DT>;
  constexpr int N = E::N, CHUNK = 64 * kBeamVecs * N;
  const int lane = (int)threadIdx.x & 63;
  const int wid = (int)blockIdx.x * (kBeamScanThreads / 64) + ((int)threadIdx.x >> 6);
  const int row = wid / a.shares, part = wid % a.shares;
  if (row >= a.batch * a.beams) return;
  if (beam_state(a.scores[row], a.finished && a.finished[row]) != BEAM_LIVE) return;  // its logits are not looked at
  const size_t es = DT == DT_F32 ? 4 : 2;
  const char* base = (const char*)a.logits +
                     ((int64_t)(row / a.beams) * a.batch_stride + (int64_t)(row % a.beams) * a.beam_stride) * (int64_t)es;
  const int e0 = part * a.share, e1 = min(a.vocab, e0 + a.share);

  float val = -INFINITY;  // lane j: the j-th best so far
  uint32_t idx = 0xFFFFFFFFu;
  float thr = -INFINITY;  // logits above it enter
  float m = -INFINITY, sum = 0.0f;
  const int k = a.k;

  for (int c0 = e0; c0 < e1; c0 += CHUNK) {
    bm_u32x4 w[kBeamVecs];
    if (c0 + CHUNK <= e1) {
#pragma unroll
      for (int j = 0; j < kBeamVecs; ++j)
        w[j] = *(const bm_u32x4_any*)(base + ((size_t)c0 + (size_t)(j * 64 + lane) * N) * es);
    } else {
#pragma unroll
      for (int j = 0; j < kBeamVecs; ++j) {
        const int o = c0 + (j * 64 + lane) * N;
        if (o + N <= e1) w[j] = *(const bm_u32x4_any*)(base + (size_t)o * es);
        else {
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
          w[j] = t;
        }
      }
    }
    float gm[kBeamVecs], lm = -INFINITY;
#pragma unroll
    for (int j = 0; j < kBeamVecs; ++j) {
      gm[j] = E::get(w[j], 0);
#pragma unroll
      for (int e = 1; e < N; ++e) gm[j] = fmaxf(gm[j], E::get(w[j], e));
      lm = fmaxf(lm, gm[j]);
    }
    const float cm = wave_max_f32(lm);
    if (cm > m) {
      sum *= __expf(m - cm);  // 0 from -inf
      m = cm;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int j = 0; j < kBeamVecs; ++j)
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        s0 += __expf(E::get(w[j], e) - ref);
        s1 += __expf(E::get(w[j], e + 1) - ref);
      }
    sum += s0 + s1;

    if (c0 == e0) {
      const float f = readlane_f(wave_sort_desc(lm, lane), k - 1);
      // the largest float below f: a logit equal to f (or the other zero) is above it
      if (f > -INFINITY) thr = f == 0.0f ? -__uint_as_float(1u) : unord_f32(radix_key(f) - 1u);
    }
#pragma unroll
    for (int j = 0; j < kBeamVecs; ++j) {
      uint64_t hit = __ballot(gm[j] > thr);
      while (hit) {
        const int l = __builtin_ctzll(hit);
        bm_u32x4 t;
#pragma unroll
        for (int q = 0; q < 4; ++q) t[q] = (uint32_t)__builtin_amdgcn_readlane((int)w[j][q], l);
        const uint32_t i0 = (uint32_t)(c0 + (j * 64 + l) * N);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float x = E::get(t, e);
          if (x > thr) {
            const int pos = __builtin_popcountll(__ballot(val >= x));
            if (pos < k) {
              const float pv = __shfl_up(val, 1, 64);
              const uint32_t pi = (uint32_t)__shfl_up((int)idx, 1, 64);
              val = lane > pos ? pv : lane == pos ? x : val;
              idx = lane > pos ? pi : lane == pos ? i0 + (uint32_t)e : idx;
              const float last = readlane_f(val, k - 1);
              if (last > -INFINITY) thr = last;
            }
          }
        }
        hit &= hit - 1;
        hit &= __ballot(gm[j] > thr);
      }
    }
  }
  double total = (double)sum;
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) total += __shfl_xor(total, x, 64);
  if (lane == 0) {
    BeamPart p;
    p.sum = total;
    p.max = m;
    p.pad = 0.0f;
    a.parts[wid] = p;
  }
  if (lane < k) a.cand[(size_t)wid * k + lane] = make_uint2(__float_as_uint(val), idx);
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

__global__ void __launch_bounds__(64 * kBeamSelectWaves) beam_select_kernel(BeamArgs a) {
  __shared__ int state[kBeamMax];
  __shared__ float rmax[kBeamMax];
  __shared__ double rlog[kBeamMax], rscore[kBeamMax];
  __shared__ double ls[kBeamSelectWaves][64];
  __shared__ uint64_t lat[kBeamSelectWaves][64];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, req = (int)blockIdx.x;
  const int W = a.beams, S = a.shares, k = a.k;

  for (int w = wave; w < W; w += kBeamSelectWaves) {
    const float sc = a.scores[(size_t)req * W + w];
    int st = beam_state(sc, a.finished && a.finished[(size_t)req * W + w]);
    float m = -INFINITY;
    double t = 0.0;
    if (st == BEAM_LIVE) {
      const BeamPart* p = a.parts + ((size_t)req * W + w) * S;
      for (int i = lane; i < S; i += 64) m = fmaxf(m, p[i].max);
      m = wave_max_f32(m);
      const double ref = m == -INFINITY ? 0.0 : (double)m;
      for (int i = lane; i < S; i += 64) t += p[i].sum * exp((double)p[i].max - ref);
#pragma unroll
      for (int x = 32; x >= 1; x >>= 1) t += __shfl_xor(t, x, 64);
      if (!(t < INFINITY)) st = BEAM_NAN;      // a NaN or an infinity among the logits
      else if (m == -INFINITY) st = BEAM_DEAD;  // the mask leaves nothing
    }
    if (lane == 0) {
      state[w] = st;
      rmax[w] = m;
      rlog[w] = st == BEAM_LIVE ? log(t) : 0.0;
      rscore[w] = (double)sc;
    }
  }
  __syncthreads();

  BeamKey best{-INFINITY, kBeamNone};
  int k2 = 1;
  while (k2 < k) k2 *= 2;
  const int per = 64 / k2, lists = W * S, j = lane % k2;
  for (int l0 = wave * per; l0 < lists; l0 += kBeamSelectWaves * per) {
    const int l = l0 + lane / k2;
    BeamKey c{-INFINITY, kBeamNone};
    if (l < lists && j < k) {
      const int w = l / S;
      if (state[w] == BEAM_LIVE) {
        const uint2 e = a.cand[((size_t)req * lists + l) * k + j];
        const float x = __uint_as_float(e.x);
        if (x > -INFINITY) {
          c.s = rscore[w] + (((double)x - (double)rmax[w]) - rlog[w]);
          c.at = beam_at(w, x, e.y);
        }
      }
    }
    if (!__any(beam_before(c, beam_from(best, k - 1)))) continue;
    beam_sort(c, lane);
    beam_merge(best, c, lane);
  }
  if (wave == 0) {  // ended beams: one candidate each
    BeamKey c{-INFINITY, kBeamNone};
    if (lane < W && state[lane] == BEAM_ENDED) {
      c.s = rscore[lane];
      c.at = beam_at(lane, 0.0f, (uint32_t)a.end_token);
    }
    if (__any(c.at != kBeamNone)) {
      beam_sort(c, lane);
      beam_merge(best, c, lane);
    }
  }
  ls[wave][lane] = best.s;
  lat[wave][lane] = best.at;
#pragma unroll
  for (int h = kBeamSelectWaves / 2; h >= 1; h >>= 1) {
    __syncthreads();
    if (wave < h) {
      const BeamKey o{ls[wave + h][lane], lat[wave + h][lane]};
      beam_merge(best, o, lane);
      ls[wave][lane] = best.s;
      lat[wave][lane] = best.at;
    }
  }
  if (wave != 0) return;
  // NaN candidates come first, by place: every token of a NaN beam, the end token of an ended one
  int nan = 0;
  uint64_t at = kBeamNone;
  for (int w = 0; w < W && nan < k; ++w) {
    const int st = state[w];
    const int n = st == BEAM_NAN ? min(a.vocab, k - nan) : st == BEAM_ENDED_NAN ? 1 : 0;
    if (lane >= nan && lane < nan + n)
      at = beam_at(w, 0.0f, (uint32_t)(st == BEAM_NAN ? lane - nan : a.end_token));
    nan += n;
  }
  const int from = lane >= nan ? lane - nan : 0;
  BeamKey out = beam_from(best, from);
  if (lane < nan) out = BeamKey{NAN, at};
  if (lane < k) {
    const size_t o = (size_t)req * k + lane;
    const bool none = out.at == kBeamNone;
    a.out_scores[o] = (float)out.s;
    a.out_parents[o] = none ? -1 : (int32_t)(out.at >> 58);
    a.out_tokens[o] = none ? -1 : (int32_t)(out.at & ((1ull << kBeamVocabBits) - 1));
  }
}

// Parts of a row: enough waves to fill the device, whole chunks each, and few
// enough lists for the second kernel.
static void beam_split(int rows, int beams, int vocab, int k, int dtype, int* shares, int* share) {
  const int chunk = 64 * kBeamVecs * (dtype == DT_F32 ? 4 : 8);
  const int chunks = (vocab - 1) / chunk + 1;
  int64_t s = (int64_t)device_cu_count() * 16 / rows;
  const int64_t most = 16384 / ((int64_t)beams * k);
  if (s > most) s = most;
  if (s < 1) s = 1;
  if (s > chunks) s = chunks;
  const int per = (int)((chunks + s - 1) / s);
  *share = per * chunk;
  *shares = (chunks + per - 1) / per;
}

static size_t beam_bytes(int rows, int shares, int k) {
  return (size_t)rows * shares * sizeof(BeamPart) + (size_t)rows * shares * k * sizeof(uint2);
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
};

struct ReorderArgs {
  ReorderTensor t[kReorderTensors];
  const int32_t* parents;
  int64_t parent_stride;
  const int32_t* slots;    // [batch, beams] or null
  const int32_t* lengths;  // [batch] or null
  int beams;
  int chunks;  // per outer index, of the largest tensor
};

// state[slot(b, w)] = old state[slot(b, parent(b, w))] in place.  A thread owns the
// same bytes of all beams of its request: it loads every moved beam's new value,
// then stores them, so no order of the moves matters and nothing waits for
// another thread.  Beams that keep their place are not touched.  Memory bound:
// each moved beam is written once; a source that several beams take comes from
// the cache after its first read.
template <int VEC, int WREG>
__global__ void __launch_bounds__(256) reorder_kernel(ReorderArgs a) {
  typedef typename std::conditional<VEC == 16, bm_u32x4, uint32_t>::type Vec;
  typedef typename std::conditional<VEC == 16, bm_u32x4_any, bm_u32_any>::type Any;
  const ReorderTensor& t = a.t[blockIdx.z];
  const int req = (int)blockIdx.y, W = a.beams;
  const int o = (int)blockIdx.x / a.chunks;
  if (o >= t.outer) return;
  int64_t valid = t.span;
  if (t.token) {
    const int64_t n = (int64_t)a.lengths[req] * t.token;
    valid = n < valid ? n : valid;
  }
  const int64_t at = ((int64_t)((int)blockIdx.x % a.chunks) * 256 + threadIdx.x) * VEC;
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
  if (vocab > (1 << kBeamVocabBits) || (int64_t)batch * beams > (1 << 24)) {
    set_error("%s: vocab (%d) or batch x beams too large", who, vocab);
    return NVJSEL_EINVAL;
  }
  return NVJSEL_OK;
}

extern "C" size_t nvjsel_beam_select_workspace_size(int dtype, int batch, int beams, int vocab, int k) {
  if (beam_check("beam_select", dtype, batch, beams, vocab, k) != NVJSEL_OK) return 0;
  int shares, share;
  beam_split(batch * beams, beams, vocab, k, dtype, &shares, &share);
  return beam_bytes(batch * beams, shares, k);
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
  beam_split(batch * beams, beams, vocab, k, dtype, &a.shares, &a.share);
  const size_t need = beam_bytes(batch * beams, a.shares, k);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) {
    set_error("beam_select: workspace %zu bytes (16-byte aligned) < required %zu", workspace_bytes, need);
    return NVJSEL_EWORKSPACE;
  }
  a.parts = (BeamPart*)workspace;
  a.cand = (uint2*)(a.parts + (size_t)batch * beams * a.shares);
  a.out_scores = out_scores;
  a.out_parents = out_parents;
  a.out_tokens = out_tokens;
  hipStream_t s = (hipStream_t)stream;
  const int64_t waves = (int64_t)batch * beams * a.shares;
  const dim3 grid((unsigned)((waves + kBeamScanThreads / 64 - 1) / (kBeamScanThreads / 64)));
  if (dtype == DT_F32) hipLaunchKernelGGL(beam_scan_kernel<DT_F32>, grid, dim3(kBeamScanThreads), 0, s, a);
  else if (dtype == DT_BF16) hipLaunchKernelGGL(beam_scan_kernel<DT_BF16>, grid, dim3(kBeamScanThreads), 0, s, a);
  else hipLaunchKernelGGL(beam_scan_kernel<DT_F16>, grid, dim3(kBeamScanThreads), 0, s, a);
  NVJSEL_CHECK_LAUNCH("beam_scan_kernel");
  hipLaunchKernelGGL(beam_select_kernel, dim3((unsigned)batch), dim3(64 * kBeamSelectWaves), 0, s, a);
  NVJSEL_CHECK_LAUNCH("beam_select_kernel");
  return NVJSEL_OK;
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
  for (int i0 = 0; i0 < count; i0 += kReorderTensors) {
    const int n = count - i0 < kReorderTensors ? count - i0 : kReorderTensors;
    ReorderArgs a{};
    int64_t chunks = 1;
    int outer = 1;
    for (int i = 0; i < n; ++i) {
      const nvjsel_state& t = states[i0 + i];
      ReorderTensor& r = a.t[i];
      r.data = (char*)t.data;
      r.row_bytes = t.row_bytes;
      r.rows = t.rows;
      r.token = lengths ? t.token_bytes : 0;
      r.outer = lengths ? t.outer : 1;
      r.span = t.length * t.token_bytes * (lengths ? 1 : t.outer);
      const int64_t c = (r.span + 256 * vec - 1) / (256 * vec);
      if (c > chunks) chunks = c;
      if (r.outer > outer) outer = r.outer;
    }
    if (chunks * outer > 0x7FFFFFFF) return fail(NVJSEL_EINVAL, "reorder_states: state too large");
    a.parents = parents;
    a.parent_stride = parent_stride;
    a.slots = slots;
    a.lengths = lengths;
    a.beams = beams;
    a.chunks = (int)chunks;
    hipStream_t s = (hipStream_t)stream;
    const int rc = beams <= 4    ? launch_reorder<16, 4>(a, n, batch, chunks * outer, s)
                   : beams <= 8  ? launch_reorder<16, 8>(a, n, batch, chunks * outer, s)
                   : beams <= 16 ? launch_reorder<16, 16>(a, n, batch, chunks * outer, s)
                                 : launch_reorder<4, 64>(a, n, batch, chunks * outer, s);
    if (rc != NVJSEL_OK) return rc;
  }
  return NVJSEL_OK;
}
