// Low-rank adapters of many requests at once beside a shared projection:
//
//   out[n] = base[n] + s_a sum_r y[n, r] B_a[:, r],   y[n, r] = sum_k x[n, k] A_a[r, k],   a = ids[n]
//
// (base[n] alone where ids[n] names no adapter).  Both products run on the matrix cores
// with fp32 sums, and out is rounded once.  s_a y lies in fp32 between them
// and enters the second as three bf16 terms (hi + mid + lo = y, 24 bits) beside bf16 tables, as two
// f16 terms of the row scaled to its largest value (22 bits; below 2^-39 of that value nothing)
// beside f16 ones.  x of another type than the tables is split into bf16 terms
// exactly (f16 two, f32 three), f16 tables beside them too.
//
// Rows name adapters in any order.  A matrix tile holds 16 rows whatever their adapters:
// each adapter among them is multiplied against all of them and a row keeps its own
// adapter's result, so that an infinity or NaN in one adapter's tables reaches no other row.
#include "lm_head_common.h"

namespace nvjsel {

static constexpr int kAdapterRank = 512;  // at most
static constexpr int kShrinkWaves = 8;    // of a block, which share the hidden size
// Steps of 32 hidden values, whose loads a wave has in flight, and blocks of a call (2000 prompt rows x 2560,
// rank 64, 2 / 4 / 5 steps: 11.6 / 12.3 / 14.5 us; 16 waves 14.8; blocks 256 to 1024 alike).
static constexpr int kShrinkSteps = 2;
static constexpr int kShrinkBlocks = 512;

// Terms that y is kept in.
__host__ __device__ constexpr int adapter_terms(int table_dtype) { return table_dtype == DT_BF16 ? 3 : 2; }

// f32 values as the next bf16 term, which leaves the remainders.  Cut off, not rounded: three terms hold all 24
// bits either way, and rounded the largest finite numbers would become infinite.
__device__ __forceinline__ u32x4_t bf16_term(float (&v)[8]) {
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = __float_as_uint(v[2 * j]), hi = __float_as_uint(v[2 * j + 1]) & 0xFFFF0000u;
    o[j] = hi | lo >> 16;
    v[2 * j] = v[2 * j] - __uint_as_float(lo & 0xFFFF0000u);
    v[2 * j + 1] = v[2 * j + 1] - __uint_as_float(hi);
  }
  return u32x4_t{o[0], o[1], o[2], o[3]};
}
__device__ __forceinline__ void f16_values(u32x4_t w, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = f16_to_f32((uint16_t)(w[j] & 0xFFFFu));
    v[2 * j + 1] = f16_to_f32((uint16_t)(w[j] >> 16));
  }
}
// x[k .. k + 7] of a row as it lies: loads without conditions, from the row's last eight where it
// ends before k + 8.  moved() puts those in place: the table is 0 behind the hidden size, so that
// any number may stand beside it (one that is not finite makes its row NaN all the same).
template <int XDT, int TDT>
struct AdapterX {
  static constexpr int NX = XDT == TDT ? 1 : XDT == DT_F32 ? 3 : XDT == DT_F16 ? 2 : 1;
  u32x4_t w[XDT == DT_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const char* row, int k, int hidden) {
    const int at = k < hidden - 8 ? k : hidden - 8;
    if constexpr (XDT == DT_F32) {
      typedef u32x4_t any __attribute__((aligned(4)));
      w[0] = *(const any*)((const float*)row + at);
      w[1] = *(const any*)((const float*)row + at + 4);
    } else {
      w[0] = *(const u32x4_any_t*)((const uint16_t*)row + at);
    }
  }
  __device__ __forceinline__ void move(int k, int hidden) {
    const int by = k + 8 - hidden < 0 ? 0 : k + 8 - hidden > 7 ? 7 : k + 8 - hidden;
    if constexpr (XDT == DT_F32) {
      uint32_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = w[e >> 2][e & 3];
#pragma unroll
      for (int d = 1; d < 8; d *= 2)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = by & d ? (e + d < 8 ? v[e + d] : 0u) : v[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e >> 2][e & 3] = v[e];
    } else {
      w[0] = shift_down8(w[0], by);
    }
  }
  // As matrix operands of 16 bits; none of them where !live.
  __device__ __forceinline__ void split(bool live, u32x4_t (&f)[NX]) const {
    const uint32_t mask = live ? ~0u : 0u;
    if constexpr (NX == 1) {
      f[0] = w[0] & mask;
    } else {
      float v[8];
      if constexpr (XDT == DT_F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(w[e >> 2][e & 3] & mask);
      } else {
        f16_values(w[0] & mask, v);
      }
#pragma unroll
      for (int t = 0; t < NX; ++t) f[t] = bf16_term(v);
    }
  }
};

struct AdapterArgs {
  const void* x;
  int64_t x_stride;
  const void* a;        // the tables in the order of a wave's loads (adapter_pack_kernel)
  const void* b;
  const float* scales;  // [count]
  const int32_t* ids;   // [rows]
  int rows, hidden, hidden_pad, rank, width, width_pad, count;
  uint16_t* terms;      // [rows, terms, rank]: y's
  float* row_scale;     // [rows]: what the terms are to be multiplied with (f16 tables)
  const void* base;
  int64_t base_stride;
  void* out;
  int64_t out_stride;
};

// The power of two that takes a row whose largest magnitude is m to 2^14 .. 2^15 (1 where it has none).
__device__ __forceinline__ int adapter_exponent(float m) {
  const int e = 15 - __builtin_amdgcn_frexp_expf(m);
  return !(m > 0.0f && m < INFINITY) ? 0 : e < -126 ? -126 : e > 126 ? 126 : e;
}
// The next term of v in the tables' type, which leaves the remainder (bf16 cut off, as x's).
template <int TDT>
__device__ __forceinline__ uint16_t adapter_term(float& v) {
  if constexpr (TDT == DT_F16) {
    const _Float16 h = (_Float16)v;
    v = v - (float)h;
    return __builtin_bit_cast(uint16_t, h);
  } else {
    const uint32_t h = __float_as_uint(v) & 0xFFFF0000u;
    v = v - __uint_as_float(h);
    return (uint16_t)(h >> 16);
  }
}

// y of 16 rows, 16 RG ranks a pass over the hidden size: block (tile, j) takes every J-th of the
// adapters among the rows, so that a decode step's many adapters run beside each other and a prompt's one
// leaves few blocks without work.  The waves split the hidden size, each with the loads of
// kShrinkSteps steps in flight; their sums meet in LDS, in order.
// Bound: latency of the loads, table and rows alike: 2000 f16 rows x 2560, rank 64, 11.5 us; without the
// table's loads 7.4, without the rows' 8.1, with neither 5.5; its ranks split over two or four blocks 12.5 and
// 16.9.  With tables as they come ([rank, hidden], a load of 16 rows) 17.
template <int XDT, int TDT, int RG>
__global__ void __launch_bounds__(64 * kShrinkWaves, 4) adapter_shrink_kernel(AdapterArgs a) {
  constexpr int NX = AdapterX<XDT, TDT>::NX, NT = adapter_terms(TDT), RANK = 16 * RG, S = kShrinkSteps;
  constexpr bool SPLIT = TDT == DT_F16 && XDT != DT_F16;  // the tables as two bf16 terms
  constexpr int MT = TDT == DT_F16 && !SPLIT ? DT_F16 : DT_BF16;
  __shared__ float part[kShrinkWaves][RANK][17];
  __shared__ float y[16][RG < 4 ? RANK : kAdapterRank];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15, row0 = (int)blockIdx.x * 16;
  const int row = row0 + c < a.rows ? row0 + c : a.rows - 1;
  int id = a.ids[row];
  if (row0 + c >= a.rows || id < 0 || id >= a.count) id = -1;
  const char* xrow = (const char*)a.x + (int64_t)row * a.x_stride * (XDT == DT_F32 ? 4 : 2);
  const int steps = a.hidden_pad / 32;
  const bool ragged = a.hidden % 8 != 0;
  uint32_t left = (uint32_t)__ballot(id >= 0) & 0xFFFFu;
  for (int nth = 0; left; ++nth) {
    const int own = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
    const uint32_t mine = (uint32_t)__ballot(id == own) & 0xFFFFu;
    left &= ~mine;
    if (nth % (int)gridDim.y != (int)blockIdx.y) continue;
    const float scale = a.scales[own];
    for (int r0 = 0; r0 < a.rank; r0 += RANK) {
      const u32x4_t* table = (const u32x4_t*)a.a + ((size_t)own * a.rank + r0) / 16 * steps * 64 + lane;
      const int tiles = (a.rank - r0) / 16;  // left, past which the last repeats: its sums are left out
      f32x4_t acc[RG];
#pragma unroll
      for (int t = 0; t < RG; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      for (int s0 = wave; s0 < steps; s0 += kShrinkWaves * S) {
        AdapterX<XDT, TDT> xs[S];
        u32x4_t w[S][RG];
#pragma unroll
        for (int u = 0; u < S; ++u) {  // past the end: the last step again, beside zeros
          const int s = s0 + u * kShrinkWaves < steps ? s0 + u * kShrinkWaves : steps - 1;
          xs[u].load(xrow, s * 32 + g * 8, a.hidden);
#pragma unroll
          for (int t = 0; t < RG; ++t) w[u][t] = table[((size_t)(t < tiles ? t : tiles - 1) * steps + s) * 64];
        }
        __builtin_amdgcn_sched_barrier(0);  // all of them before the first product
#pragma unroll
        for (int u = 0; u < S; ++u) {
          const int s = s0 + u * kShrinkWaves;
          u32x4_t xf[NX];
          if (ragged && s == steps - 1) xs[u].move(s * 32 + g * 8, a.hidden);
          xs[u].split(s < steps, xf);
#pragma unroll
          for (int t = 0; t < RG; ++t) {
            if constexpr (SPLIT) {
              float v[8];
              f16_values(w[u][t], v);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const u32x4_t term = bf16_term(v);
#pragma unroll
                for (int n = 0; n < NX; ++n) acc[t] = mfma16x16x32<MT>(term, xf[n], acc[t]);
              }
            } else {
#pragma unroll
              for (int n = 0; n < NX; ++n) acc[t] = mfma16x16x32<MT>(w[u][t], xf[n], acc[t]);
            }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < RG; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[wave][t * 16 + 4 * g + e][c] = acc[t][e];
      __syncthreads();
      for (int i = (int)threadIdx.x; i < RANK * 16; i += 64 * kShrinkWaves) {
        const int r = i >> 4, n = i & 15;
        float s = part[0][r][n];
#pragma unroll
        for (int w = 1; w < kShrinkWaves; ++w) s += part[w][r][n];
        if (r0 + r < a.rank) y[n][r0 + r] = s * scale;
      }
      __syncthreads();
    }
    for (int n = wave; n < 16; n += kShrinkWaves) {
      if (!(mine >> n & 1)) continue;
      float up = 1.0f;
      if constexpr (TDT == DT_F16) {
        float m = 0.0f;
        for (int r = lane; r < a.rank; r += 64) m = fmaxf(m, fabsf(y[n][r]));
        const int e = adapter_exponent(__uint_as_float(wave_max_u32(__float_as_uint(m))));
        up = __builtin_amdgcn_ldexpf(1.0f, e);
        if (lane == 0) a.row_scale[row0 + n] = __builtin_amdgcn_ldexpf(1.0f, -e);
      }
      uint16_t* out = a.terms + (size_t)(row0 + n) * NT * a.rank;
      for (int r = lane; r < a.rank; r += 64) {
        float v = y[n][r] * up;
#pragma unroll
        for (int t = 0; t < NT; ++t) out[t * a.rank + r] = adapter_term<TDT>(v);
      }
    }
    __syncthreads();  // y is free
  }
}

// 16 rows x 64 columns of base and out as they lie, 16 bytes a lane: the lanes of a row next to each
// other, so that an instruction takes whole cache lines.  (By the products' own layout, where
// neighbouring lanes hold other rows, copying 2000 x 4096 took 10.2 us, so 8.3.)
template <int ODT>
struct AdapterTile {
  static constexpr int E = ODT == DT_F32 ? 4 : 8, LANES = 64 / E, ROWS = 64 / LANES, Q = 16 / ROWS;
  u32x4_t w[Q];
  // row q * ROWS + lane / LANES of the tile, `left` elements of it at p; whole: of the wave's tile nothing is past the end
  __device__ __forceinline__ void load(int q, const char* p, int left, bool whole) {
    if (whole) {
      w[q] = *(const u32x4_any_t*)p;
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (ODT == DT_F32) w[q][e] = e < left ? ((const uint32_t*)p)[e] : 0u;
      else
        w[q][e] = (2 * e < left ? (uint32_t)((const uint16_t*)p)[2 * e] : 0u) |
                  (2 * e + 1 < left ? (uint32_t)((const uint16_t*)p)[2 * e + 1] << 16 : 0u);
    }
  }
  __device__ __forceinline__ void add(int q, const float* d) {
#pragma unroll
    for (int h = 0; h < E / 4; ++h) {
      const f32x4_t x = *(const f32x4_t*)(d + 4 * h);
      if constexpr (ODT == DT_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[q][e] = __float_as_uint(__uint_as_float(w[q][e]) + x[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t u = w[q][2 * h + e];
          if constexpr (ODT == DT_BF16)
            w[q][2 * h + e] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)(bf16_to_f32((uint16_t)(u >> 16)) + x[2 * e + 1])) << 16 |
                              __builtin_bit_cast(uint16_t, (__bf16)(bf16_to_f32((uint16_t)u) + x[2 * e]));
          else
            w[q][2 * h + e] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)(f16_to_f32((uint16_t)(u >> 16)) + x[2 * e + 1])) << 16 |
                              __builtin_bit_cast(uint16_t, (_Float16)(f16_to_f32((uint16_t)u) + x[2 * e]));
        }
      }
    }
  }
  __device__ __forceinline__ void store(int q, char* p, int left, bool whole) const {
    if (whole) {
      *(u32x4_any_t*)p = w[q];
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) {
        if constexpr (ODT == DT_F32) ((uint32_t*)p)[e] = w[q][e];
        else ((uint16_t*)p)[e] = (uint16_t)(w[q][e >> 1] >> (16 * (e & 1)));
      }
  }
};
static constexpr int kTilePitch = 68;  // floats of a row of a tile's sums in LDS

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
// v_mfma_f32_16x16x16: four k of a row per lane.
template <int WT>
__device__ __forceinline__ f32x4_t mfma16x16x16(u32x2_t a, u32x2_t b, f32x4_t c) {
  if constexpr (WT == DT_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a), __builtin_bit_cast(s16x4_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a), __builtin_bit_cast(f16x4_t, b), c, 0, 0, 0);
}

// ---- The tables' layout: pieces of 16 bytes (8 values) in the order of a wave's loads, 64 of them (1 KB)
// an instruction; piece of lane (c, g) = (lane & 15, lane >> 4), zeros behind the adapters' own sizes.
//   a: [count][rank / 16][hidden_pad / 32][lane]: A[16 i + c][32 s + 8 g ..]
//   b: [count][width_pad / 64][rank / 32][4][lane], ranks 32 and more:  B[column(t, c)][32 k + 8 g ..]
//      [count][width_pad / 64][2][lane], rank 16:                       B[column(2 l + (g >> 1), c)][8 (g & 1) ..]
//   column(t, c) = 64 group + 16 (c >> 2) + 4 t + (c & 3)
struct AdapterPack {
  const uint16_t* from;  // [count][major][minor], strides in elements, minor's 1
  int64_t count_stride, row_stride;
  int rank, hidden, width;              // of the adapters
  int rank_pad, hidden_pad, width_pad;  // of the table
  uint4* to;
  int64_t pieces;
};
template <bool B>
__global__ void __launch_bounds__(256) adapter_pack_kernel(AdapterPack p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.pieces) return;
  const int lane = (int)(i & 63), c = lane & 15, g = lane >> 4;
  int64_t j = i >> 6;
  int row, k;  // of the plain form
  if constexpr (!B) {
    const int steps = p.hidden_pad / 32;
    k = (int)(j % steps) * 32 + 8 * g;
    j /= steps;
    row = (int)(j % (p.rank_pad / 16)) * 16 + c;
    j /= p.rank_pad / 16;
  } else {
    int t;
    if (p.rank_pad == 16) {
      t = 2 * (int)(j & 1) + (g >> 1);
      k = 8 * (g & 1);
      j >>= 1;
    } else {
      t = (int)(j & 3);
      j >>= 2;
      k = (int)(j % (p.rank_pad / 32)) * 32 + 8 * g;
      j /= p.rank_pad / 32;
    }
    row = (int)(j % (p.width_pad / 64)) * 64 + 16 * (c >> 2) + 4 * t + (c & 3);
    j /= p.width_pad / 64;
  }
  const int rows = B ? p.width : p.rank, ks = B ? p.rank : p.hidden;
  const uint16_t* from = p.from + j * p.count_stride + (int64_t)row * p.row_stride + k;
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = row < rows && k + 2 * e < ks ? from[2 * e] : 0u;
    if (row < rows && k + 2 * e + 1 < ks) w[e] |= (uint32_t)from[2 * e + 1] << 16;
  }
  p.to[i] = make_uint4(w[0], w[1], w[2], w[3]);
}

// The adapter of row row0 + lane, -1: none.
template <int RT>
__device__ __forceinline__ int adapter_of(const AdapterArgs& a, int row0, int lane) {
  if (lane >= 16 * RT || row0 + lane >= a.rows) return -1;
  const int id = a.ids[row0 + lane];
  return id < 0 || id >= a.count ? -1 : id;
}
// A block's rows in order of adapter, in which the matrix tiles take them, those without one last: an
// adapter's rows lie in one tile or two, and the others need no product with it (64 rows of 16 adapters: 19 products of
// a tile with an adapter, in the order given 38 expected).  id becomes the place's, mine[]
// the row of column c of each tile, from the row (less row0) of place `lane`; returns the places that have an adapter.
template <int RT>
__device__ __forceinline__ uint64_t adapter_places(int& id, int row0, int (&mine)[RT], int& from) {
  const int lane = (int)threadIdx.x & 63, c = lane & 15;
  int place = 0, count = 0;
  for (uint64_t todo = __ballot(id >= 0), of; todo; todo &= ~of) {
    of = __ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctzll(todo)));
    if (of >> lane & 1) place = count + __builtin_popcountll(of & ((1ull << lane) - 1));
    count += __builtin_popcountll(of);
  }
  const uint64_t none = __ballot(id < 0);
  if (id < 0) place = count + __builtin_popcountll(none & ((1ull << lane) - 1));
  from = __builtin_amdgcn_ds_permute(place * 4, lane);
  id = __builtin_amdgcn_ds_bpermute(from * 4, id);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) mine[rt] = row0 + __builtin_amdgcn_ds_bpermute((rt * 16 + c) * 4, from);
  return count == 64 ? ~0ull : (1ull << count) - 1;
}

// A wave's 64 columns x 16 RT rows.  The matrix tiles' rows are columns of out, dealt so that
// a lane ends with 16 consecutive ones of one row: tile t's row i is column 16 (i >> 2) + 4 t + (i & 3).
// The table's rows of the next adapters (or steps of 32 of their ranks) are on their way in a ring of
// D slots, loads without conditions: the last adapter's again at the end.  base is
// requested before all of them.
// Rank 16 (WIDE false): a 16-byte load of a lane is half a row of the table, two tiles an
// instruction; swapping halves of the wave makes of it two operands of 16x16x16 products, lane
// (c, g) with ranks 8 (g & 1) + 4 (g >> 1) .. + 3, so that no byte is loaded twice for y's terms.
// Wider ranks: 16x16x32 products, 32 ranks a step, y's terms in LDS.
// Bound: memory.  64 bf16 rows of 16 adapters at 248,320 columns, rank 16 (191 MB): 42 us, 4.5 TB/s; 2 to 8
// slots, 32 columns a wave, non-temporal loads and stores and columns by XCD took 41 to 46, rows in blocks of 32 (the
// tables twice) 50.
template <int TDT, int ODT, bool WIDE, int RT>
__global__ void __launch_bounds__(256) adapter_expand_kernel(AdapterArgs a) {
  constexpr int CT = 4, NT = adapter_terms(TDT), D = WIDE ? 2 : 3, WL = WIDE ? CT : CT / 2;
  extern __shared__ __attribute__((aligned(16))) char staged[];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t v0 = ((int64_t)blockIdx.x * 4 + wave) * (16 * CT);
  const int row0 = (int)blockIdx.y * 16 * RT;
  int id = adapter_of<RT>(a, row0, lane);
  const bool in_place = a.out == a.base;
  if (in_place && __ballot(id >= 0) == 0) return;
  int mine[RT], from;
  const uint64_t named = adapter_places<RT>(id, row0, mine, from);
  constexpr int es = ODT == DT_F32 ? 4 : 2;
  using Tile = AdapterTile<ODT>;
  constexpr int Q = Tile::Q;
  __shared__ __attribute__((aligned(16))) float tile[4][16][kTilePitch];  // a wave's own
  const int first = lane % Tile::LANES * Tile::E;                          // this lane's first column
  const int64_t v = v0 + first;
  const int here = (int)(a.width - v < Tile::E ? a.width - v : Tile::E);  // its columns, none below 1
  const bool whole = v0 + 16 * CT <= a.width;
  auto place = [&](int rt, int q) NVJSEL_INLINE { return rt * 16 + q * Tile::ROWS + lane / Tile::LANES; };
  auto row_at = [&](int rt, int q) NVJSEL_INLINE { return row0 + __builtin_amdgcn_ds_bpermute(place(rt, q) * 4, from); };
  Tile out[RT];
  float up[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int row = row_at(rt, q);
      out[rt].load(q, (const char*)a.base + ((int64_t)(row < a.rows ? row : a.rows - 1) * a.base_stride + v) * es, here, whole);
    }
    up[rt] = TDT == DT_F16 && (named >> (rt * 16 + c) & 1) ? a.row_scale[mine[rt]] : 1.0f;
  }
  // a finished adapter's rows, through LDS into their tile's layout; others', and those without one, stay as
  // they are (0 added would turn -0 into 0)
  auto add = [&](int rt, uint64_t of, const f32x4_t (&d)[CT]) NVJSEL_INLINE {
    __builtin_amdgcn_wave_barrier();  // LDS operations of a wave are performed in order
#pragma unroll
    for (int t = 0; t < CT; ++t) *(f32x4_t*)&tile[wave][c][16 * g + 4 * t] = TDT == DT_F16 ? d[t] * up[rt] : d[t];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (of >> place(rt, q) & 1) out[rt].add(q, &tile[wave][q * Tile::ROWS + lane / Tile::LANES][first]);
  };
  if (named) {
    const int pitch = NT * a.rank * 2 + 16;  // bytes of a staged row
    u32x2_t y[RT][NT];
    if constexpr (!WIDE) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int row = mine[rt] < a.rows ? mine[rt] : a.rows - 1;
#pragma unroll
        for (int n = 0; n < NT; ++n)
          y[rt][n] = *(const u32x2_t*)(a.terms + ((size_t)row * NT + n) * 16 + 8 * (g & 1) + 4 * (g >> 1));
      }
    }
    // this lane's pieces of the first adapter; a wave's columns past the end are the last group's
    const int64_t group = v0 < a.width_pad ? v0 / 64 : a.width_pad / 64 - 1;
    const u32x4_t* table = (const u32x4_t*)a.b + (size_t)group * 64 * a.rank / 8 + lane;
    const size_t each = (size_t)a.width_pad * a.rank / 8;
    uint64_t ahead = named, same[D];
    int own = 0, kn = 0;
    int kk[D];
    u32x4_t raw[D][WL];
    auto fetch = [&](auto S) NVJSEL_INLINE {
      constexpr int s = decltype(S)::value;
      same[s] = 0;
      kk[s] = kn;
      if (ahead) {
        own = __builtin_amdgcn_readlane(id, __builtin_ctzll(ahead));
        same[s] = __ballot(id == own);
      }
      const u32x4_t* b = table + (size_t)own * each + (WIDE ? kn * 8 : 0);
#pragma unroll
      for (int l = 0; l < WL; ++l) raw[s][l] = b[l * 64];
      kn += 32;
      if (!WIDE || kn >= a.rank) {
        kn = 0;
        ahead &= ~same[s];
      }
    };
    f32x4_t sums[WIDE ? RT : 1][CT];
    auto body = [&](auto S) NVJSEL_INLINE {
      constexpr int s = decltype(S)::value;
      const uint64_t of = same[s];
      const int k = kk[s];
      u32x4_t w[WL];
#pragma unroll
      for (int l = 0; l < WL; ++l) w[l] = raw[s][l];
      if constexpr (!WIDE) {
#pragma unroll
        for (int l = 0; l < WL; ++l) {
          const auto x = __builtin_amdgcn_permlane32_swap(w[l][0], w[l][2], false, false);
          const auto z = __builtin_amdgcn_permlane32_swap(w[l][1], w[l][3], false, false);
          w[l] = u32x4_t{x[0], z[0], x[1], z[1]};
        }
      }
      fetch(S);
      const bool first = !WIDE || k == 0, last = !WIDE || k + 32 >= a.rank;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (!(of >> (rt * 16) & 0xFFFFu)) continue;
        f32x4_t (&d)[CT] = sums[WIDE ? rt : 0];
        if (first) {
#pragma unroll
          for (int t = 0; t < CT; ++t) d[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (WIDE) {
            const u32x4_t f = *(const u32x4_t*)(staged + (mine[rt] - row0) * pitch + (n * a.rank + k + 8 * g) * 2);
#pragma unroll
            for (int t = 0; t < CT; ++t) d[t] = mfma16x16x32<TDT>(w[t], f, d[t]);
          } else {
#pragma unroll
            for (int t = 0; t < CT; ++t)
              d[t] = mfma16x16x16<TDT>(u32x2_t{w[t / 2][2 * (t & 1)], w[t / 2][2 * (t & 1) + 1]}, y[rt][n], d[t]);
          }
        }
        if (last) add(rt, of, d);
      }
    };
    static_for<D>([&](auto S) NVJSEL_INLINE { fetch(S); });
    if constexpr (WIDE) {  // y's terms, rows as they lie, four loads of a thread on their way together
      const int pieces = NT * a.rank / 8, all = 16 * RT * pieces;
      for (int i0 = (int)threadIdx.x; i0 < all; i0 += 4 * 256) {
        u32x4_t terms[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * 256 < all ? i0 + u * 256 : all - 1, r = i / pieces;
          terms[u] = *(const u32x4_t*)(a.terms + ((size_t)(row0 + r < a.rows ? row0 + r : a.rows - 1) * pieces + i % pieces) * 8);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * 256;
          if (i < all) *(u32x4_t*)(staged + i / pieces * pitch + i % pieces * 16) = terms[u];
        }
      }
      __syncthreads();
    }
    bool more = true;
    while (more)
      static_for<D>([&](auto S) NVJSEL_INLINE {
        if (more) {
          if (same[decltype(S)::value]) body(S);
          else more = false;
        }
      });
  }
  if (v0 >= a.width) return;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int row = row_at(rt, q);
      if (row < a.rows && !(in_place && !(named >> place(rt, q) & 1)))
        out[rt].store(q, (char*)a.out + ((int64_t)row * a.out_stride + v) * es, here, whole);
    }
}

// Ranks 32 and 64 (KB steps of 32), 64 rows a block: a wave holds all of an adapter's table for its 64
// columns in registers, the next adapter's on its way, and takes the row tiles one after another, so that a
// prompt's table is read once for 64 rows and only one tile's sums are held.  Everything that a block
// reads is requested before its first product.  2000 f16 rows x 4096, rank 64: 12.5 us, in the ring above 14; the
// copy of base alone takes 8.3.
template <int TDT, int ODT, int KB>
__global__ void __launch_bounds__(256) adapter_expand64_kernel(AdapterArgs a) {
  constexpr int RT = 4, CT = 4, NT = adapter_terms(TDT), RANK = 32 * KB, PITCH = NT * RANK * 2 + 16;
  __shared__ __attribute__((aligned(16))) char staged[16 * RT * PITCH];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t v0 = ((int64_t)blockIdx.x * 4 + wave) * (16 * CT);
  const int row0 = (int)blockIdx.y * 16 * RT;
  int id = adapter_of<RT>(a, row0, lane);
  const bool in_place = a.out == a.base;
  if (in_place && __ballot(id >= 0) == 0) return;
  int mine[RT], from;
  const uint64_t named = adapter_places<RT>(id, row0, mine, from);
  constexpr int es = ODT == DT_F32 ? 4 : 2;
  using Tile = AdapterTile<ODT>;
  constexpr int Q = Tile::Q;
  __shared__ __attribute__((aligned(16))) float tile[4][16][kTilePitch];  // a wave's own
  const int first = lane % Tile::LANES * Tile::E;                          // this lane's first column
  const int64_t v = v0 + first;
  const int here = (int)(a.width - v < Tile::E ? a.width - v : Tile::E);  // its columns, none below 1
  const bool whole = v0 + 16 * CT <= a.width;
  auto place = [&](int rt, int q) NVJSEL_INLINE { return rt * 16 + q * Tile::ROWS + lane / Tile::LANES; };
  auto row_at = [&](int rt, int q) NVJSEL_INLINE { return row0 + __builtin_amdgcn_ds_bpermute(place(rt, q) * 4, from); };
  Tile out[RT];
  float up[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int row = row_at(rt, q);
      out[rt].load(q, (const char*)a.base + ((int64_t)(row < a.rows ? row : a.rows - 1) * a.base_stride + v) * es, here, whole);
    }
    up[rt] = TDT == DT_F16 && (named >> (rt * 16 + c) & 1) ? a.row_scale[mine[rt]] : 1.0f;
  }
  // a finished adapter's rows, through LDS into their tile's layout; others', and those without one, stay as
  // they are (0 added would turn -0 into 0)
  auto add = [&](int rt, uint64_t of, const f32x4_t (&d)[CT]) NVJSEL_INLINE {
    __builtin_amdgcn_wave_barrier();  // LDS operations of a wave are performed in order
#pragma unroll
    for (int t = 0; t < CT; ++t) *(f32x4_t*)&tile[wave][c][16 * g + 4 * t] = TDT == DT_F16 ? d[t] * up[rt] : d[t];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (of >> place(rt, q) & 1) out[rt].add(q, &tile[wave][q * Tile::ROWS + lane / Tile::LANES][first]);
  };
  if (named) {
    const int64_t group = v0 < a.width_pad ? v0 / 64 : a.width_pad / 64 - 1;
    const u32x4_t* table = (const u32x4_t*)a.b + (size_t)group * 64 * RANK / 8 + lane;
    const size_t each = (size_t)a.width_pad * RANK / 8;
    uint64_t ahead = named, same[2];
    int own = 0;
    u32x4_t w[2][KB][CT];
    auto fetch = [&](auto S) NVJSEL_INLINE {  // the next adapter's table; the last one's again at the end
      constexpr int s = decltype(S)::value;
      same[s] = 0;
      if (ahead) {
        own = __builtin_amdgcn_readlane(id, __builtin_ctzll(ahead));
        same[s] = __ballot(id == own);
        ahead &= ~same[s];
      }
      const u32x4_t* b = table + (size_t)own * each;
#pragma unroll
      for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int t = 0; t < CT; ++t) w[s][k][t] = b[(k * CT + t) * 64];
    };
    fetch(std::integral_constant<int, 0>{});
    constexpr int PIECES = NT * RANK / 8, LOADS = 16 * RT * PIECES / 256;
    static_assert(16 * RT * PIECES % 256 == 0, "");
    u32x4_t terms[LOADS];  // y's terms, rows as they lie
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int i = (int)threadIdx.x + u * 256, r = i / PIECES;
      terms[u] = *(const u32x4_t*)(a.terms + ((size_t)(row0 + r < a.rows ? row0 + r : a.rows - 1) * PIECES + i % PIECES) * 8);
    }
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int i = (int)threadIdx.x + u * 256;
      *(u32x4_t*)(staged + i / PIECES * PITCH + i % PIECES * 16) = terms[u];
    }
    __syncthreads();
    bool more = true;
    while (more)
      static_for<2>([&](auto S) NVJSEL_INLINE {
        constexpr int s = decltype(S)::value;
        if (more && same[s]) {
          const uint64_t of = same[s];
          fetch(std::integral_constant<int, 1 - s>{});
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            if (!(of >> (rt * 16) & 0xFFFFu)) continue;
            f32x4_t d[CT];
#pragma unroll
            for (int t = 0; t < CT; ++t) d[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KB; ++k)
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const u32x4_t f = *(const u32x4_t*)(staged + (mine[rt] - row0) * PITCH + (n * RANK + k * 32 + 8 * g) * 2);
#pragma unroll
                for (int t = 0; t < CT; ++t) d[t] = mfma16x16x32<TDT>(w[s][k][t], f, d[t]);
              }
            add(rt, of, d);
          }
        } else {
          more = false;
        }
      });
  }
  if (v0 >= a.width) return;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int row = row_at(rt, q);
      if (row < a.rows && !(in_place && !(named >> place(rt, q) & 1)))
        out[rt].store(q, (char*)a.out + ((int64_t)row * a.out_stride + v) * es, here, whole);
    }
}

template <int TDT, int ODT, bool WIDE, int RT>
static int launch_expand(const AdapterArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.width + 255) / 256), (unsigned)((a.rows + 16 * RT - 1) / (16 * RT)));
  const size_t lds = WIDE ? (size_t)16 * RT * (adapter_terms(TDT) * a.rank * 2 + 16) : 0;
  auto kern = adapter_expand_kernel<TDT, ODT, WIDE, RT>;
  if (lds > 40 * 1024)  // beside the tiles' own
    NVJSEL_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(kern, grid, dim3(256), lds, s, a);
  NVJSEL_CHECK_LAUNCH("adapter_expand_kernel");
  return NVJSEL_OK;
}

template <int TDT, int ODT>
static int launch_expand64(const AdapterArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.width + 255) / 256), (unsigned)((a.rows + 63) / 64));
  if (a.rank == 32) hipLaunchKernelGGL((adapter_expand64_kernel<TDT, ODT, 1>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((adapter_expand64_kernel<TDT, ODT, 2>), grid, dim3(256), 0, s, a);
  NVJSEL_CHECK_LAUNCH("adapter_expand64_kernel");
  return NVJSEL_OK;
}

template <int XDT, int TDT>
static int launch_shrink(const AdapterArgs& a, hipStream_t s) {
  const int tiles = (a.rows + 15) / 16;
  int each = 16;  // blocks of a tile
  while (each > 1 && tiles * each > kShrinkBlocks) each /= 2;
  const dim3 grid((unsigned)tiles, (unsigned)each), block(64 * kShrinkWaves);
  if (a.rank <= 16) hipLaunchKernelGGL((adapter_shrink_kernel<XDT, TDT, 1>), grid, block, 0, s, a);
  else if (a.rank <= 32) hipLaunchKernelGGL((adapter_shrink_kernel<XDT, TDT, 2>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((adapter_shrink_kernel<XDT, TDT, 4>), grid, block, 0, s, a);
  NVJSEL_CHECK_LAUNCH("adapter_shrink_kernel");
  return NVJSEL_OK;
}

template <int TDT>
static int launch_adapters(const AdapterArgs& a, int x_dtype, int out_dtype, hipStream_t s) {
  const int rc = x_dtype == DT_F32    ? launch_shrink<DT_F32, TDT>(a, s)
                 : x_dtype == DT_BF16 ? launch_shrink<DT_BF16, TDT>(a, s)
                                      : launch_shrink<DT_F16, TDT>(a, s);
  if (rc != NVJSEL_OK) return rc;
  auto expand = [&](auto O) -> int {
    constexpr int ODT = decltype(O)::value;
    if (a.rank == 16) {
      if (a.rows <= 16) return launch_expand<TDT, ODT, false, 1>(a, s);
      if (a.rows <= 32) return launch_expand<TDT, ODT, false, 2>(a, s);
      return launch_expand<TDT, ODT, false, 4>(a, s);
    }
    if (a.rows > 32 && a.rank <= 64) return launch_expand64<TDT, ODT>(a, s);
    if (a.rows <= 16 || a.rank > 256) return launch_expand<TDT, ODT, true, 1>(a, s);
    return launch_expand<TDT, ODT, true, 2>(a, s);
  };
  if (out_dtype == DT_F32) return expand(std::integral_constant<int, DT_F32>{});
  if (out_dtype == DT_BF16) return expand(std::integral_constant<int, DT_BF16>{});
  return expand(std::integral_constant<int, DT_F16>{});
}

}  // namespace nvjsel

using namespace nvjsel;

static bool adapter_sizes_ok(int table_dtype, int64_t rows, int rank) {
  return (table_dtype == NVJSEL_BF16 || table_dtype == NVJSEL_F16) && rows > 0 && rows <= (1 << 20) &&
         (rank == 16 || (rank > 0 && rank <= kAdapterRank && rank % 32 == 0));
}

extern "C" size_t nvjsel_adapters_workspace_size(int table_dtype, int64_t rows, int rank) {
  clear_error();
  if (!adapter_sizes_ok(table_dtype, rows, rank)) {
    set_error("apply_adapters: bad sizes (rows=%lld rank=%d table dtype=%d)", (long long)rows, rank, table_dtype);
    return 0;
  }
  return align_up((size_t)rows * adapter_terms(table_dtype) * rank * 2, 16) + (size_t)rows * 4;
}

extern "C" int nvjsel_adapters_pack(const void* plain, int which, int64_t count_stride, int64_t row_stride, int count, int rank,
                                    int hidden, int width, int rank_pad, void* packed, size_t packed_bytes, void* stream) {
  clear_error();
  if (which != 0 && which != 1) return fail(NVJSEL_EINVAL, "adapters_pack: which must be 0 (a) or 1 (b)");
  if (count <= 0 || rank <= 0 || hidden <= 0 || width <= 0) return fail(NVJSEL_EINVAL, "adapters_pack requires non-empty dimensions");
  if (!adapter_sizes_ok(NVJSEL_BF16, 1, rank_pad) || rank > rank_pad || hidden > (1 << 24) || width > (1 << 28))
    return fail(NVJSEL_EINVAL, "adapters_pack: bad sizes");
  if (!plain || !packed) return fail(NVJSEL_EINVAL, "adapters_pack: null pointer");
  if (((uintptr_t)plain & 1) || ((uintptr_t)packed & 15)) return fail(NVJSEL_EINVAL, "adapters_pack: unaligned pointer");
  if (count_stride < 0 || row_stride < 0) return fail(NVJSEL_EINVAL, "adapters_pack: negative stride");
  AdapterPack p{};
  p.from = (const uint16_t*)plain;
  p.count_stride = count_stride;
  p.row_stride = row_stride;
  p.rank = rank;
  p.hidden = hidden;
  p.width = width;
  p.rank_pad = rank_pad;
  p.hidden_pad = (hidden + 31) / 32 * 32;
  p.width_pad = (width + 63) / 64 * 64;
  p.to = (uint4*)packed;
  p.pieces = (int64_t)count * rank_pad * (which ? p.width_pad : p.hidden_pad) / 8;
  if (packed_bytes < (size_t)p.pieces * 16) return fail(NVJSEL_EINVAL, "adapters_pack: the table is too small");
  if (p.pieces / 256 >= 1 << 23) return fail(NVJSEL_EINVAL, "adapters_pack: too many values for a call");
  const dim3 grid((unsigned)((p.pieces + 255) / 256));
  if (which) hipLaunchKernelGGL((adapter_pack_kernel<true>), grid, dim3(256), 0, (hipStream_t)stream, p);
  else hipLaunchKernelGGL((adapter_pack_kernel<false>), grid, dim3(256), 0, (hipStream_t)stream, p);
  NVJSEL_CHECK_LAUNCH("adapter_pack_kernel");
  return NVJSEL_OK;
}

extern "C" int nvjsel_apply_adapters(const void* x, int x_dtype, int64_t x_stride, const void* base, int out_dtype,
                                     int64_t base_stride, const void* a_table, const void* b_table, int table_dtype,
                                     const float* scales, int count, int rank, int hidden, int width, const int32_t* ids,
                                     int64_t rows, void* out, int64_t out_stride, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  clear_error();
  if (rows <= 0 || hidden <= 0 || width <= 0 || count <= 0) {
    set_error("apply_adapters requires non-empty dimensions (rows=%lld hidden=%d width=%d adapters=%d)", (long long)rows,
              hidden, width, count);
    return NVJSEL_EINVAL;
  }
  if (!valid_dtype(x_dtype) || !valid_dtype(out_dtype) || (table_dtype != NVJSEL_BF16 && table_dtype != NVJSEL_F16)) {
    set_error("apply_adapters: unsupported dtype (x=%d out=%d tables=%d)", x_dtype, out_dtype, table_dtype);
    return NVJSEL_EINVAL;
  }
  if (!adapter_sizes_ok(table_dtype, rows, rank)) {
    set_error("apply_adapters: rank (%d) must be 16 or a multiple of 32 up to %d, rows (%lld) at most 2^20", rank,
              kAdapterRank, (long long)rows);
    return NVJSEL_EINVAL;
  }
  if (hidden < 8) return fail(NVJSEL_EUNSUPPORTED, "apply_adapters: hidden below 8 (pad x with zeros)");
  if (hidden > (1 << 24) || width > (1 << 28)) return fail(NVJSEL_EINVAL, "apply_adapters: hidden or width too large");
  if (!x || !base || !a_table || !b_table || !scales || !ids || !out) return fail(NVJSEL_EINVAL, "apply_adapters: null pointer");
  if ((((uintptr_t)a_table) | ((uintptr_t)b_table)) & 15) return fail(NVJSEL_EINVAL, "apply_adapters: unaligned tables");
  if ((((uintptr_t)x) & (dtype_size(x_dtype) - 1)) || ((((uintptr_t)base) | ((uintptr_t)out)) & (dtype_size(out_dtype) - 1)))
    return fail(NVJSEL_EINVAL, "apply_adapters: unaligned rows");
  if (x_stride < 0 || base_stride < 0) return fail(NVJSEL_EINVAL, "apply_adapters: negative stride");
  if (rows > 1 && out_stride < width) return fail(NVJSEL_EINVAL, "apply_adapters: output row stride < width");
  if (out == base && rows > 1 && out_stride != base_stride)
    return fail(NVJSEL_EINVAL, "apply_adapters: in place, with another stride");
  const size_t need = nvjsel_adapters_workspace_size(table_dtype, rows, rank);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) {
    set_error("apply_adapters: workspace %zu bytes (16-byte aligned) < required %zu", workspace_bytes, need);
    return NVJSEL_EWORKSPACE;
  }
  AdapterArgs g{};
  g.x = x;
  g.x_stride = x_stride;
  g.a = a_table;
  g.b = b_table;
  g.scales = scales;
  g.ids = ids;
  g.rows = (int)rows;
  g.hidden = hidden;
  g.hidden_pad = (hidden + 31) / 32 * 32;
  g.rank = rank;
  g.width = width;
  g.count = count;
  g.width_pad = (width + 63) / 64 * 64;
  g.terms = (uint16_t*)workspace;
  g.row_scale = (float*)((char*)workspace + align_up((size_t)rows * adapter_terms(table_dtype) * rank * 2, 16));
  g.base = base;
  g.base_stride = base_stride;
  g.out = out;
  g.out_stride = out_stride;
  std::lock_guard<std::mutex> lock(launch_mutex());
  if (table_dtype == NVJSEL_BF16) return launch_adapters<DT_BF16>(g, x_dtype, out_dtype, (hipStream_t)stream);
  return launch_adapters<DT_F16>(g, x_dtype, out_dtype, (hipStream_t)stream);
}
