// Low-rank adapters of many requests at once beside a shared projection:
//
//   out[n] = base[n] + s_a sum_r y[n, r] B_a[:, r],   y[n, r] = sum_k x[n, k] A_a[r, k],   a = ids[n]
//
// (base[n] alone where ids[n] names no adapter).  Both products run on the matrix cores
// with fp32 sums, and out is rounded once.  y is kept in more than 16 bits between them:
// s_a y as three bf16 terms (hi + mid + lo = y, 24 bits) beside bf16 tables, as two f16
// terms of the row scaled to its largest value (22 bits; below 2^-39 of that value
// nothing) beside f16 ones.  x of another type than the tables is split into bf16 terms
// exactly (f16 two, f32 three), f16 tables beside them too.
//
// Rows name adapters in any order.  A matrix tile holds 16 rows whatever their adapters:
// each adapter among them is multiplied against all of them and a row keeps its own
// adapter's result, so that an infinity or NaN in one adapter's tables reaches no other row.
#include "lm_head_common.h"

namespace nvjsel {

static constexpr int kAdapterRank = 512;  // at most
static constexpr int kShrinkWaves = 8;    // of a block, which share the hidden size
static constexpr int kShrinkRank = 64;    // rank of a pass over the hidden rows

// Terms that y is kept in.
__host__ __device__ constexpr int adapter_terms(int table_dtype) { return table_dtype == DT_BF16 ? 3 : 2; }

// Eight elements at p, the first `left` of them (the rest 0), as NX matrix operands of 16 bits.
template <int XDT, int TDT>
struct AdapterX {
  static constexpr int NX = XDT == TDT ? 1 : XDT == DT_F32 ? 3 : XDT == DT_F16 ? 2 : 1;
};
// f32 values as the next bf16 term, which leaves the remainders.
__device__ __forceinline__ u32x4_t bf16_term(float (&v)[8]) {
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = __builtin_bit_cast(uint16_t, (__bf16)v[2 * j]), hi = __builtin_bit_cast(uint16_t, (__bf16)v[2 * j + 1]);
    o[j] = hi << 16 | lo;
    v[2 * j] = v[2 * j] - __uint_as_float(o[j] << 16);
    v[2 * j + 1] = v[2 * j + 1] - __uint_as_float(o[j] & 0xFFFF0000u);
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
template <int XDT, int TDT>
__device__ __forceinline__ void adapter_x(const char* row, int k, int left, u32x4_t (&f)[AdapterX<XDT, TDT>::NX]) {
  constexpr int NX = AdapterX<XDT, TDT>::NX;
  float v[8];
  if constexpr (XDT == DT_F32) {
    const float* p = (const float*)row + k;
    if (left >= 8) {
      typedef u32x4_t any __attribute__((aligned(4)));
      const u32x4_t a = *(const any*)p, b = *(const any*)(p + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = __uint_as_float(a[j]);
        v[4 + j] = __uint_as_float(b[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < NX; ++t) f[t] = bf16_term(v);
  } else {
    const uint16_t* p = (const uint16_t*)row + k;
    u32x4_t w{0u, 0u, 0u, 0u};
    if (left >= 8) {
      w = *(const u32x4_any_t*)p;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) w[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
    }
    if constexpr (NX == 1) {
      f[0] = w;
    } else {
      f16_values(w, v);
#pragma unroll
      for (int t = 0; t < NX; ++t) f[t] = bf16_term(v);
    }
  }
}

struct AdapterArgs {
  const void* x;
  int64_t x_stride;
  const void* a;        // [count, rank, hidden_pad], zeros behind the adapters' own sizes
  const void* b;        // [count, width, rank]
  const float* scales;  // [count]
  const int32_t* ids;   // [rows]
  int rows, hidden, hidden_pad, rank, width, count;
  uint16_t* terms;      // [rows, terms, rank]
  float* row_scale;     // [rows]: what the terms are to be multiplied with (f16 tables)
  const void* base;
  int64_t base_stride;
  void* out;
  int64_t out_stride;
};

// y of 16 rows and one of their adapters: block (tile, j) takes row j's adapter where no row
// before it has the same one.  The waves split the hidden size; their sums meet in LDS, in
// order.
template <int XDT, int TDT>
__global__ void __launch_bounds__(64 * kShrinkWaves) adapter_shrink_kernel(AdapterArgs a) {
  constexpr int NX = AdapterX<XDT, TDT>::NX, NT = adapter_terms(TDT);
  constexpr bool SPLIT = TDT == DT_F16 && XDT != DT_F16;  // the tables as two bf16 terms
  constexpr int MT = TDT == DT_F16 && !SPLIT ? DT_F16 : DT_BF16;
  __shared__ float part[kShrinkWaves][kShrinkRank][17];
  __shared__ float y[16][kAdapterRank];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15, row0 = (int)blockIdx.x * 16, j = (int)blockIdx.y;
  const int row = row0 + c < a.rows ? row0 + c : a.rows - 1;
  int id = a.ids[row];
  if (row0 + c >= a.rows || id < 0 || id >= a.count) id = -1;
  const int own = __builtin_amdgcn_readlane(id, j);
  const uint32_t mine = (uint32_t)__ballot(id == own) & 0xFFFFu;
  if (own < 0 || __builtin_ctz(mine) != j) return;

  const char* xrow = (const char*)a.x + (int64_t)row * a.x_stride * (XDT == DT_F32 ? 4 : 2);
  const uint16_t* table = (const uint16_t*)a.a + (size_t)own * a.rank * a.hidden_pad;
  const int steps = a.hidden_pad / 32;
  const float scale = a.scales[own];
  for (int r0 = 0; r0 < a.rank; r0 += kShrinkRank) {
    f32x4_t acc[kShrinkRank / 16];
#pragma unroll
    for (int t = 0; t < kShrinkRank / 16; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = wave; s < steps; s += kShrinkWaves) {
      const int k = s * 32 + g * 8;
      u32x4_t xf[NX];
      adapter_x<XDT, TDT>(xrow, k, a.hidden - k, xf);
#pragma unroll
      for (int t = 0; t < kShrinkRank / 16; ++t) {
        if (r0 + t * 16 >= a.rank) break;
        const int r = r0 + t * 16 + c;
        u32x4_t w{0u, 0u, 0u, 0u};
        if (r < a.rank) w = *(const u32x4_t*)(table + (size_t)r * a.hidden_pad + k);
        if constexpr (SPLIT) {
          float v[8];
          f16_values(w, v);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const u32x4_t term = bf16_term(v);
#pragma unroll
            for (int n = 0; n < NX; ++n) acc[t] = mfma16x16x32<MT>(term, xf[n], acc[t]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < NX; ++n) acc[t] = mfma16x16x32<MT>(w, xf[n], acc[t]);
        }
      }
    }
    if (r0) __syncthreads();
#pragma unroll
    for (int t = 0; t < kShrinkRank / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave][t * 16 + 4 * g + e][c] = acc[t][e];
    __syncthreads();
    for (int i = (int)threadIdx.x; i < kShrinkRank * 16; i += 64 * kShrinkWaves) {
      const int r = i >> 4, n = i & 15;
      float s = part[0][r][n];
#pragma unroll
      for (int w = 1; w < kShrinkWaves; ++w) s += part[w][r][n];
      if (r0 + r < a.rank) y[n][r0 + r] = s * scale;
    }
  }
  __syncthreads();
  for (int n = wave; n < 16; n += kShrinkWaves) {
    if (!(mine >> n & 1)) continue;
    float up = 1.0f;
    if constexpr (TDT == DT_F16) {  // the row's largest value to 2^14 .. 2^15
      float m = 0.0f;
      for (int r = lane; r < a.rank; r += 64) m = fmaxf(m, fabsf(y[n][r]));
      m = __uint_as_float(wave_max_u32(__float_as_uint(m)));
      int e = 15 - __builtin_amdgcn_frexp_expf(m);
      if (!(m > 0.0f && m < INFINITY)) e = 0;
      e = e < -126 ? -126 : e > 126 ? 126 : e;
      up = __builtin_amdgcn_ldexpf(1.0f, e);
      if (lane == 0) a.row_scale[row0 + n] = __builtin_amdgcn_ldexpf(1.0f, -e);
    }
    uint16_t* out = a.terms + (size_t)(row0 + n) * NT * a.rank;
    for (int r = lane; r < a.rank; r += 64) {
      float v = y[n][r] * up;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (TDT == DT_F16) {
          const _Float16 h = (_Float16)v;
          out[t * a.rank + r] = __builtin_bit_cast(uint16_t, h);
          v = v - (float)h;
        } else {
          const __bf16 h = (__bf16)v;
          out[t * a.rank + r] = __builtin_bit_cast(uint16_t, h);
          v = v - (float)h;
        }
      }
    }
  }
}

// 16 consecutive elements of a row as f32 and back; `left` of them exist.
template <int ODT>
__device__ __forceinline__ void load16(const char* row, int64_t v, int left, float (&x)[16]) {
  if constexpr (ODT == DT_F32) {
    typedef u32x4_t any __attribute__((aligned(4)));
    const float* p = (const float*)row + v;
    if (left >= 16) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const u32x4_t w = *(const any*)(p + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * q + e] = __uint_as_float(w[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = e < left ? p[e] : 0.0f;
    }
  } else {
    const uint16_t* p = (const uint16_t*)row + v;
    uint32_t w[8];
    if (left >= 16) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const u32x4_t u = *(const u32x4_any_t*)(p + 8 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * q + e] = u[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[e] = (2 * e < left ? (uint32_t)p[2 * e] : 0u) | (2 * e + 1 < left ? (uint32_t)p[2 * e + 1] << 16 : 0u);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
      x[e] = ODT == DT_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
    }
  }
}
template <int ODT>
__device__ __forceinline__ void store16(char* row, int64_t v, int left, const float (&x)[16]) {
  if constexpr (ODT == DT_F32) {
    typedef u32x4_t any __attribute__((aligned(4)));
    float* p = (float*)row + v;
    if (left >= 16) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(any*)(p + 4 * q) = u32x4_t{__float_as_uint(x[4 * q]), __float_as_uint(x[4 * q + 1]), __float_as_uint(x[4 * q + 2]),
                                     __float_as_uint(x[4 * q + 3])};
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e < left) p[e] = x[e];
    }
  } else {
    uint16_t* p = (uint16_t*)row + v;
    uint16_t h[16];
#pragma unroll
    for (int e = 0; e < 16; ++e)
      h[e] = ODT == DT_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)x[e]) : __builtin_bit_cast(uint16_t, (_Float16)x[e]);
    if (left >= 16) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        u32x4_t w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (uint32_t)h[8 * q + 2 * e + 1] << 16 | h[8 * q + 2 * e];
        *(u32x4_any_t*)(p + 8 * q) = w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e < left) p[e] = h[e];
    }
  }
}

// A wave's 64 columns x 16 RT rows.  The matrix tiles' rows are columns of out, dealt so that
// a lane ends with 16 consecutive ones of one row: tile t's row i is column 16 (i >> 2) + 4 t +
// (i & 3).  OCT: eights of a rank below 32, whose terms lie side by side along a matrix
// instruction's k (4: a multiple of 32, a term after another).
template <int TDT, int ODT, int OCT, int RT>
__global__ void __launch_bounds__(256) adapter_expand_kernel(AdapterArgs a) {
  constexpr int NT = adapter_terms(TDT);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t v0 = ((int64_t)blockIdx.x * 4 + wave) * 64;
  const int row0 = (int)blockIdx.y * 16 * RT;
  if (v0 >= a.width) return;
  int id = -1;  // of row row0 + lane
  if (lane < 16 * RT && row0 + lane < a.rows) {
    id = a.ids[row0 + lane];
    if (id >= a.count) id = -1;
  }
  const uint64_t named = __ballot(id >= 0);
  const bool in_place = a.out == a.base;
  if (in_place && named == 0) return;
  const uint16_t* terms[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = row0 + rt * 16 + c < a.rows ? row0 + rt * 16 + c : a.rows - 1;
    terms[rt] = a.terms + (size_t)row * NT * a.rank;
  }
  size_t brow[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int64_t v = v0 + 16 * (c >> 2) + 4 * t + (c & 3);
    brow[t] = (size_t)(v < a.width ? v : a.width - 1) * a.rank;
  }
  f32x4_t acc[RT][4];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[rt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto keep = [&](int rt, uint64_t same, const f32x4_t (&d)[4]) NVJSEL_INLINE {
    const bool mine = same >> (rt * 16 + c) & 1;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[rt][t][e] = mine ? d[t][e] : acc[rt][t][e];
  };
  if constexpr (OCT < 4) {
    constexpr int STEPS = (NT * OCT + 3) / 4;
    u32x4_t y[RT][STEPS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int q = 4 * s + g;
        y[rt][s] = q < NT * OCT && named ? *(const u32x4_t*)(terms[rt] + q * 8) : u32x4_t{0u, 0u, 0u, 0u};
      }
    for (uint64_t left = named; left;) {
      const int own = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
      const uint64_t same = __ballot(id == own);
      left &= ~same;
      const uint16_t* b = (const uint16_t*)a.b + (size_t)own * a.width * a.rank;
      u32x4_t w[4][STEPS];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) w[t][s] = *(const u32x4_t*)(b + brow[t] + (4 * s + g) % OCT * 8);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (!(same >> (rt * 16) & 0xFFFFu)) continue;
        f32x4_t d[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          d[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < STEPS; ++s) d[t] = mfma16x16x32<TDT>(w[t][s], y[rt][s], d[t]);
        }
        keep(rt, same, d);
      }
    }
  } else {
    for (uint64_t left = named; left;) {
      const int own = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
      const uint64_t same = __ballot(id == own);
      left &= ~same;
      const uint16_t* b = (const uint16_t*)a.b + (size_t)own * a.width * a.rank;
      f32x4_t d[RT][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int t = 0; t < 4; ++t) d[rt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      for (int k = g * 8; k < a.rank; k += 32) {
        u32x4_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t] = *(const u32x4_t*)(b + brow[t] + k);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          if (!(same >> (rt * 16) & 0xFFFFu)) continue;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const u32x4_t y = *(const u32x4_t*)(terms[rt] + n * a.rank + k);
#pragma unroll
            for (int t = 0; t < 4; ++t) d[rt][t] = mfma16x16x32<TDT>(w[t], y, d[rt][t]);
          }
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) keep(rt, same, d[rt]);
    }
  }
  const int64_t v = v0 + 16 * g;
  const int left = (int)(a.width - v < 16 ? a.width - v : 16);
  if (left <= 0) return;
  constexpr int es = ODT == DT_F32 ? 4 : 2;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = row0 + rt * 16 + c;
    const bool has = named >> (rt * 16 + c) & 1;
    if (row >= a.rows || (in_place && !has)) continue;
    float x[16];
    load16<ODT>((const char*)a.base + (int64_t)row * a.base_stride * es, v, left, x);
    if (has) {  // (a row without an adapter is copied as it is: 0 added would turn -0 into 0)
      const float up = TDT == DT_F16 ? a.row_scale[row] : 1.0f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * t + e] += TDT == DT_F16 ? acc[rt][t][e] * up : acc[rt][t][e];
    }
    store16<ODT>((char*)a.out + (int64_t)row * a.out_stride * es, v, left, x);
  }
}

template <int TDT, int ODT, int RT>
static int launch_expand_rows(const AdapterArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.width + 255) / 256), (unsigned)((a.rows + 16 * RT - 1) / (16 * RT)));
  if (a.rank == 8) hipLaunchKernelGGL((adapter_expand_kernel<TDT, ODT, 1, RT>), grid, dim3(256), 0, s, a);
  else if (a.rank == 16) hipLaunchKernelGGL((adapter_expand_kernel<TDT, ODT, 2, RT>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((adapter_expand_kernel<TDT, ODT, 4, RT>), grid, dim3(256), 0, s, a);
  NVJSEL_CHECK_LAUNCH("adapter_expand_kernel");
  return NVJSEL_OK;
}

template <int TDT>
static int launch_adapters(const AdapterArgs& a, int x_dtype, int out_dtype, hipStream_t s) {
  const dim3 grid((unsigned)((a.rows + 15) / 16), 16), block(64 * kShrinkWaves);
  if (x_dtype == DT_F32) hipLaunchKernelGGL((adapter_shrink_kernel<DT_F32, TDT>), grid, block, 0, s, a);
  else if (x_dtype == DT_BF16) hipLaunchKernelGGL((adapter_shrink_kernel<DT_BF16, TDT>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((adapter_shrink_kernel<DT_F16, TDT>), grid, block, 0, s, a);
  NVJSEL_CHECK_LAUNCH("adapter_shrink_kernel");
  auto expand = [&](auto O) -> int {
    constexpr int ODT = decltype(O)::value;
    if (a.rows <= 16) return launch_expand_rows<TDT, ODT, 1>(a, s);
    return launch_expand_rows<TDT, ODT, 2>(a, s);
  };
  if (out_dtype == DT_F32) return expand(std::integral_constant<int, DT_F32>{});
  if (out_dtype == DT_BF16) return expand(std::integral_constant<int, DT_BF16>{});
  return expand(std::integral_constant<int, DT_F16>{});
}

}  // namespace nvjsel

using namespace nvjsel;

static bool adapter_sizes_ok(int table_dtype, int64_t rows, int rank) {
  return (table_dtype == NVJSEL_BF16 || table_dtype == NVJSEL_F16) && rows > 0 && rows <= (1 << 20) &&
         (rank == 8 || rank == 16 || (rank > 0 && rank <= kAdapterRank && rank % 32 == 0));
}

extern "C" size_t nvjsel_adapters_workspace_size(int table_dtype, int64_t rows, int rank) {
  clear_error();
  if (!adapter_sizes_ok(table_dtype, rows, rank)) {
    set_error("apply_adapters: bad sizes (rows=%lld rank=%d table dtype=%d)", (long long)rows, rank, table_dtype);
    return 0;
  }
  return align_up((size_t)rows * adapter_terms(table_dtype) * rank * 2, 16) + (size_t)rows * 4;
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
    set_error("apply_adapters: rank (%d) must be 8, 16 or a multiple of 32 up to %d, rows (%lld) at most 2^20", rank,
              kAdapterRank, (long long)rows);
    return NVJSEL_EINVAL;
  }
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
