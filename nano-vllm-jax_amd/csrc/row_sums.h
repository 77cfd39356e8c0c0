// Sums over a row of logits, shared by beam search's selection and the log
// probabilities of tokens: 16-byte pieces at any address, a wave's maximum and sums
// without LDS, and the sum of exponentials (with the entropy's) of one pass over a
// share of a row, whose reference moves as the maximum rises.
#pragma once
#include "nvjsel_device.h"
#include "nvjsel_host.h"

namespace nvjsel {

typedef uint32_t row_u32x4 __attribute__((ext_vector_type(4)));
typedef row_u32x4 row_u32x4_any __attribute__((aligned(1)));  // 16 bytes from any address
typedef uint32_t row_u32_any __attribute__((aligned(1)));

// Parts and candidates, 8 bytes at a time.  ONE: they pass between blocks of one launch,
// on any XCDs, written and read at the device's coherence point (agent scope).
template <bool ONE>
__device__ __forceinline__ void row_put(void* p, uint32_t lo, uint32_t hi) {
  const unsigned long long v = (unsigned long long)hi << 32 | lo;
  if constexpr (ONE) __hip_atomic_store((unsigned long long*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else *(unsigned long long*)p = v;
}
template <bool ONE>
__device__ __forceinline__ uint2 row_get(const void* p) {
  unsigned long long v;
  if constexpr (ONE) v = __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else v = *(const unsigned long long*)p;
  return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
}

template <int DT>
struct RowElems {
  static constexpr int N = DT == DT_F32 ? 4 : 8;  // elements of a 16-byte piece
  __device__ static __forceinline__ float get(const row_u32x4& w, int e) {
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
// Exponentials are the hardware's exp2 (about 1 ulp) of fma(x, log2 e, -ref): one
// rounding of the difference.  ref is a whole number next to a lane's maximum times log2 e,
// so that a sum moves from one reference to another by its exponent alone, exactly, however
// often its maximum rises.  That holds for maxima up to this size; the reference stays
// within it, and a share whose own maximum does not is summed again (row_sum_far).
static constexpr float kLog2e = 1.44269504088896341f, kRowFar = 16384.0f;
__device__ __forceinline__ float row_ref(float m) { return rintf(fminf(fmaxf(m, -kRowFar), kRowFar) * kLog2e); }
// sum, relative to 2^from, relative to 2^to.
__device__ __forceinline__ double row_move(double sum, float from, float to) {
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
__device__ __forceinline__ row_u32x4 row_piece(const char* base, int o, int e1) {
  using E = RowElems<DT>;
  if (o + E::N <= e1) return *(const row_u32x4_any*)(base + (size_t)o * (DT == DT_F32 ? 4 : 2));
  row_u32x4 t;
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

// A row's part: the sum of exp(l - max) and, where it is asked for, of exp(l - max) (l - max).
struct RowSum {
  double sum, ent;
};
struct RowPart {  // with its maximum, as parts of a row are passed on
  double sum, ent;
  float max;
  int pad;
};

// Adds V pieces per lane, whose maximum is x, to the lane's sums.  Relative to 2^ref,
// with y = l log2 e - ref: sum of 2^y, ent of 2^y y; both move to another reference by
//   sum' = 2^(ref - ref') sum,   ent' = 2^(ref - ref') (ent + (ref - ref') sum).
// 2^y is 0 below y = -150, and y is held above -200 in its product: -inf gives 0.
// The terms of a call in five roundings at most, from zero: added to the sum of those
// before, the small ones of a long share would be lost (one large logit and 122 chunks
// of small ones: scores off by 9e-5 so).
template <int DT, bool ENT, int V>
__device__ __forceinline__ void row_add(const row_u32x4 (&w)[V], float x, float& m, float& ref, RowSum& r) {
  using E = RowElems<DT>;
  const float to = __builtin_elementwise_maximum(m, x), to_ref = row_ref(to);
  float s[V], u[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float t[E::N], p[E::N];
#pragma unroll
    for (int e = 0; e < E::N; ++e) {
      const float y = __builtin_fmaf(E::get(w[j], e), kLog2e, -to_ref);
      t[e] = __builtin_amdgcn_exp2f(y);
      if constexpr (ENT) p[e] = t[e] * fmaxf(y, -200.0f);
    }
    s[j] = sum_tree(t);
    if constexpr (ENT) u[j] = sum_tree(p);
  }
  if constexpr (ENT) r.ent = row_move(r.ent + r.sum * (double)(ref - to_ref), ref, to_ref) + (double)sum_tree(u);
  r.sum = row_move(r.sum, ref, to_ref) + (double)sum_tree(s);
  m = to;
  ref = to_ref;
}

// The sums of a share whose maximum m is known, a lane's part; ent in units of log2 e.
template <int DT, bool ENT>
__device__ __forceinline__ RowSum row_sum_far(const char* base, int e0, int e1, float m, int lane) {
  using E = RowElems<DT>;
  RowSum r{0.0, 0.0};
  for (int o = e0 + lane * E::N; o < e1; o += 64 * E::N) {
    const row_u32x4 w = row_piece<DT>(base, o, e1);
    float s = 0.0f, u = 0.0f;
#pragma unroll
    for (int e = 0; e < E::N; ++e) {
      const float y = (E::get(w, e) - m) * kLog2e, t = __builtin_amdgcn_exp2f(y);
      s += t;
      if constexpr (ENT) u += t * fmaxf(y, -200.0f);
    }
    r.sum += (double)s;
    if constexpr (ENT) r.ent += (double)u;
  }
  return r;
}

// A wave's sums of its share from its lanes', relative to its maximum wm, ent in natural units.
template <int DT, bool ENT>
__device__ __forceinline__ RowSum row_wave_total(const char* base, int e0, int e1, float wm, float ref, const RowSum& own,
                                                 int lane) {
  RowSum r{0.0, 0.0};
  if (wm <= kRowFar && (wm >= 100.0f - kRowFar || wm == -INFINITY)) {
    const float wref = row_ref(wm);
    r.sum = wave_sum_f64(row_move(own.sum, ref, wref));  // a NaN's sum is NaN
    if constexpr (ENT) r.ent = wave_sum_f64(row_move(own.ent + own.sum * (double)(ref - wref), ref, wref));
    // relative to exp(wm) now: exp(d), |d| < 0.35, by its series (to 2^-32)
    const double b = wm == -INFINITY ? 0.0 : (double)wref - (double)wm * (double)kLog2e, d = b * 0.6931471805599453;
    double f = 1.0;
#pragma unroll
    for (int i = 8; i >= 1; --i) f = __builtin_fma(f, d * (1.0 / i), 1.0);
    if constexpr (ENT) r.ent = f * (r.ent + b * r.sum);
    r.sum *= f;
  } else {
    const RowSum far = row_sum_far<DT, ENT>(base, e0, e1, wm, lane);
    r.sum = wave_sum_f64(far.sum);
    if constexpr (ENT) r.ent = wave_sum_f64(far.ent);
  }
  if constexpr (ENT) r.ent *= 0.6931471805599453;
  return r;
}

// What the rows' answers are made of: the token asked of every row and where they go.
// stats: the row's maximum, the log of its sum and its entropy, for the gradient.
struct RowAnswers {
  const void* tokens;  // [rows] int32 or int64
  int token64;
  float* logprobs;     // [rows]
  float* entropy;      // [rows] or null
  float* stats;        // [rows, 3] or null
};

// Adds a part's sums, relative to its own maximum, to a row's, relative to m.
__device__ __forceinline__ void row_join(RowSum& r, const RowSum& part, float max, float m) {
  if (max == -INFINITY && part.sum == 0.0) return;  // nothing left in it
  const double d = (double)max - (double)m, f = exp(d);
  r.ent += f * (part.ent + part.sum * d);
  r.sum += f * part.sum;
}

// ln S: the row's maximum is one of its terms, 1 exactly, which the hardware's exp2 and a wave's series may leave an ulp
// or so below; no log probability is above 0.
__device__ __forceinline__ double row_log_sum(double sum) { return log(fmax(sum, 1.0)); }

// logprob = (x - m) - ln S for the token's logit x, entropy = ln S - T / S (r: S and T,
// relative to m).  Nothing left: -inf and 0; NaN or +inf among the logits: NaN; a row that
// asks for no token: 0.
// log_sum: ln S where it is a number.
__device__ __forceinline__ void row_answer(const RowAnswers& a, int64_t row, bool asked, float x, float m, const RowSum& r,
                                           double log_sum) {
  const bool nan = !(r.sum < INFINITY), none = !nan && r.sum == 0.0;
  const double ls = nan ? (double)NAN : none ? 0.0 : log_sum;
  a.logprobs[row] = !asked ? 0.0f : nan ? NAN : none ? -INFINITY : (float)(((double)x - (double)m) - ls);
  const double h = nan ? (double)NAN : none ? 0.0 : fmax(ls - r.ent / r.sum, 0.0);
  if (a.entropy) a.entropy[row] = (float)h;
  if (a.stats) {
    a.stats[3 * row] = nan ? NAN : m;
    a.stats[3 * row + 1] = (float)ls;
    a.stats[3 * row + 2] = (float)h;
  }
}
// The token asked of a row; one outside 0..vocab-1 asks for nothing.
__device__ __forceinline__ int64_t row_token(const RowAnswers& a, int64_t row) {
  return a.token64 ? ((const int64_t*)a.tokens)[row] : ((const int32_t*)a.tokens)[row];
}
// The same, the token's logit from the row at element `at`.
template <int DT>
__device__ __forceinline__ void row_answer_from(const RowAnswers& a, const void* logits, int64_t at, int vocab, int64_t row,
                                                float m, const RowSum& r) {
  const int64_t t = row_token(a, row);
  const bool asked = t >= 0 && t < vocab;
  row_answer(a, row, asked, asked ? load_as_f32(logits, DT, (size_t)(at + t)) : 0.0f, m, r, row_log_sum(r.sum));
}

}  // namespace nvjsel
