// LM head with 4-bit weights and group scales: dense logits, and greedy top-1
// without logits.
//
//   w[v,k] = s[v,G] (q[v,k] - z[v,G]),  G = k / group,  q in 0..15 (z = 8 without zero points)
//   logit[b,v] = sum_G s[v,G] (sum_{k in G} x[b,k] q[v,k] - z[v,G] sum_{k in G} x[b,k])
//
// The inner sums run on the matrix cores.  A nibble becomes a 16-bit float
// without a conversion: placed in the top mantissa bits of 16.0 it reads 16 + q
// exactly, so one shift and one and-or make two operands.  The accumulator of
// a group starts at -(16 + z) times the group's sum of activations, so that
// the offset is gone when the group ends; then it is scaled into the row's
// total.  Sums are fp32 throughout (the activations' group sums fp64, rounded
// once).  The offset is the smallest one that an exponent's mantissa holds: with
// 128 + q (no shift for a quarter of the nibbles) the partial sums are six
// times larger than the result's terms, and so is their rounding.
//
// Packed layout (w4_pack_kernel): blocks of 16 vocabulary rows x 128 k, 1 KB
// each, in the order in which a wave's 16-byte loads feed the matrix
// instructions: lane l holds row l & 15, word j the eight k at 32 j + 8 (l >> 4),
// the nibble of k = 2 p at bits 4 p, of 2 p + 1 at 16 + 4 p.  All k blocks of 16 rows lie
// together, then the next 16 rows.  The scales follow, 16 rows x 128 / group
// per block, and the zero points in the same order.  Rows past V and k past H
// are zero with scale zero.
#pragma once
#include "lm_head_common.h"

namespace nvjsel {

static constexpr int kW4Waves = 8, kW4Threads = 64 * kW4Waves;

struct W4Layout {
  int tiles, kblocks, ng;  // 16-row tiles, 128-wide k blocks, groups per k block
  size_t scales, zeros, total;  // byte offsets of the parts, and the size
};

__host__ __device__ inline W4Layout w4_layout(int V, int H, int group, bool zeros) {
  W4Layout w;
  w.tiles = (V + 15) / 16;
  w.kblocks = (H + 127) / 128;
  w.ng = 128 / group;
  const size_t blocks = (size_t)w.tiles * w.kblocks;
  w.scales = blocks * 1024;
  w.zeros = w.scales + (blocks * 16 * w.ng * 2 + 255) / 256 * 256;
  w.total = w.zeros + (zeros ? (blocks * 16 * w.ng + 255) / 256 * 256 : 0);
  return w;
}

struct W4Args {
  const void* hidden;
  int hidden_dtype;
  const uint8_t* packed;
  int scale_dtype;
  int zeros;   // zero points are there
  int V, H;
  int B, rows;  // batch rows of this pass; their slots in LDS (a power of two up to 16, or 16 MB)
  int kc;      // k blocks of the hidden in LDS at a time
  int reduce_cast;
  unsigned long long* row_keys;
  unsigned int* counter;
  int32_t* out_ids;
  float* out_best;
  void* out_logits;
  int out_dtype;
  long long out_stride;
};

// 16 + q of the eight nibbles of a packed word, as bf16 or f16 pairs.
template <int FMT>
__device__ __forceinline__ u32x4_t w4_unpack(uint32_t w) {
  u32x4_t r;
  if constexpr (FMT == DT_BF16) {  // mantissa bits 3..6
    r.x = ((w << 3) & 0x00780078u) | 0x41804180u;
    r.y = ((w >> 1) & 0x00780078u) | 0x41804180u;
    r.z = ((w >> 5) & 0x00780078u) | 0x41804180u;
    r.w = ((w >> 9) & 0x00780078u) | 0x41804180u;
  } else {  // mantissa bits 6..9
    r.x = ((w << 6) & 0x03C003C0u) | 0x4C004C00u;
    r.y = ((w << 2) & 0x03C003C0u) | 0x4C004C00u;
    r.z = ((w >> 2) & 0x03C003C0u) | 0x4C004C00u;
    r.w = ((w >> 6) & 0x03C003C0u) | 0x4C004C00u;
  }
  return r;
}

// k blocks kb0 .. of the hidden into LDS, as the matrix instructions' operands:
// 16-byte slots [(4 kb + j) MB TERMS + mb TERMS + t][k eighth][row].  Three terms: x =
// the bf16 values that its leading, next and last eight bits make (exact); a
// value that is not finite keeps its first term only.  Then the sums of each
// group's activations, [group][16 MB].
template <int FMT, int TERMS, int MB, int NG>
__device__ __forceinline__ void w4_stage_hidden(const W4Args& a, int kb0, int nkb, u32x4_t* frag, float* xsum) {
  const int lane = (int)threadIdx.x & 63, u = lane & 15, j = u >> 2, qd = u & 3;
  const int items = a.rows * nkb;  // 16 lanes each
  const int rt = a.rows < 16 ? a.rows : 16;
  for (int it = (int)threadIdx.x >> 4; it < items; it += kW4Threads / 16) {
    const int row = it % a.rows, kb = it / a.rows, k = (kb0 + kb) * 128 + 8 * u;
    float x[8];
    if (row < a.B && k < a.H) {
      load8_as_f32(a.hidden, a.hidden_dtype, (size_t)row * a.H + k, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    }
    const int mb = row >> 4, slot = row & 15;
    u32x4_t* dst = frag + ((size_t)((kb * 4 + j) * MB + mb) * TERMS * 4 + qd) * rt + slot;
    uint32_t h[TERMS][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (TERMS == 1) {
        h[0][e] = FMT == DT_BF16 ? bf16_bits_rne(x[e]) : f16_bits(x[e]);
      } else {
        const uint32_t b = __float_as_uint(x[e]);
        const bool fin = (b & 0x7F800000u) != 0x7F800000u;
        h[0][e] = fin ? b >> 16 : bf16_bits_rne(x[e]);
        const float r1 = x[e] - __uint_as_float(b & 0xFFFF0000u);
        h[1][e] = fin ? __float_as_uint(r1) >> 16 : 0u;
        const float r2 = r1 - __uint_as_float(__float_as_uint(r1) & 0xFFFF0000u);
        h[2][e] = fin ? __float_as_uint(r2) >> 16 : 0u;
      }
    }
#pragma unroll
    for (int t = 0; t < TERMS; ++t)
      dst[t * 4 * rt] = u32x4_t{h[t][0] | h[t][1] << 16, h[t][2] | h[t][3] << 16, h[t][4] | h[t][5] << 16,
                                h[t][6] | h[t][7] << 16};
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += (double)x[e];
#pragma unroll
    for (int m = 1; m < 16 / NG; m <<= 1) sum += __shfl_xor(sum, m, 64);
    if (u % (16 / NG) == 0) xsum[(kb * NG + u / (16 / NG)) * 16 * MB + row] = (float)sum;
  }
}

// One block per CU, eight waves.  A wave takes NT adjacent tiles of 16
// vocabulary rows at a time and runs over all of H, its next k blocks' 1 KB pieces
// on the way in registers (DEPTH); the waves share the hidden in LDS, all of it
// where it fits and kc k blocks at a time where not.  Matrix tile: M = batch
// rows, N = vocabulary rows, so that a lane's four results share their scale.
template <int FMT, int TERMS, int MB, int NT, int NG, int MODE>
__global__ void __launch_bounds__(kW4Threads, 2) lm_head_w4_kernel(W4Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int DEPTH = 3;
  const W4Layout lay = w4_layout(a.V, a.H, 128 / NG, a.zeros != 0);
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int KB = lay.kblocks, kc = a.kc, rt = a.rows < 16 ? a.rows : 16;
  u32x4_t* frag = (u32x4_t*)lds;
  float* xsum = (float*)(lds + (size_t)kc * 4 * MB * TERMS * 4 * rt * 16);
  const int supers = (lay.tiles + NT - 1) / NT;
  const int step = (int)gridDim.x * kW4Waves;
  const int first = (int)blockIdx.x * kW4Waves + wave;
  const int rounds = (supers - (int)blockIdx.x * kW4Waves + step - 1) / step;  // of the block: some waves repeat the last tile
  const int n = rounds * KB;

  const u32x4_t* wq = (const u32x4_t*)a.packed;
  const uint8_t* sc = a.packed + lay.scales;
  const uint8_t* zp = a.packed + lay.zeros;

  struct Item {
    u32x4_t w[NT];
    uint32_t s[NT][(NG + 1) / 2];
    uint32_t z[NT];
  };
  Item ring[DEPTH];

  // the item to be requested next
  int lkb = 0, lsuper = first;
  auto load = [&](auto D, int) NVJSEL_INLINE {
    Item& it = ring[decltype(D)::value];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      int tile = lsuper * NT + t;
      tile = tile < lay.tiles ? tile : lay.tiles - 1;
      const size_t blk = (size_t)tile * KB + lkb;
      it.w[t] = __builtin_nontemporal_load(wq + blk * 64 + lane);
      const size_t m = blk * 16 + (lane & 15);
      if constexpr (NG == 1) it.s[t][0] = ((const uint16_t*)sc)[m];
      else if constexpr (NG == 2) it.s[t][0] = ((const uint32_t*)sc)[m];
      else {
        const uint64_t v = ((const uint64_t*)sc)[m];
        it.s[t][0] = (uint32_t)v;
        it.s[t][1] = (uint32_t)(v >> 32);
      }
      if (a.zeros) {
        if constexpr (NG == 1) it.z[t] = zp[m];
        else if constexpr (NG == 2) it.z[t] = ((const uint16_t*)zp)[m];
        else it.z[t] = ((const uint32_t*)zp)[m];
      } else it.z[t] = 0x08080808u;
    }
    if (++lkb == KB) { lkb = 0; lsuper += step; }
  };

  f32x4_t total[NT][MB];
  unsigned long long best[MB][4];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
#pragma unroll
    for (int i = 0; i < 4; ++i) best[m][i] = 0ull;
#pragma unroll
    for (int t = 0; t < NT; ++t) total[t][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  const int arow = (lane & 15) < rt ? (lane & 15) : rt - 1;
  int kb = 0, kl = 0, super = first;  // the item in work; kl: its k block in LDS
  auto body = [&](auto D, int) NVJSEL_INLINE {
    if (kc < KB && kl == 0) {
      __syncthreads();
      w4_stage_hidden<FMT, TERMS, MB, NG>(a, kb, KB - kb < kc ? KB - kb : kc, frag, xsum);
      __syncthreads();
    }
    const Item& it = ring[decltype(D)::value];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4_t acc[NT][MB];
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        const f32x4_t xs = *(const f32x4_t*)(xsum + (kl * NG + g) * 16 * MB + 16 * m + 4 * (lane >> 4));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float z = -16.0f - (float)((it.z[t] >> (8 * g)) & 0xFFu);
          acc[t][m] = f32x4_t{xs.x * z, xs.y * z, xs.z * z, xs.w * z};
        }
      }
#pragma unroll
      for (int j = g * 4 / NG; j < (g + 1) * 4 / NG; ++j) {
        u32x4_t wf[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) wf[t] = w4_unpack<FMT>(it.w[t][j]);
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int c = 0; c < TERMS; ++c) {
            const u32x4_t xf = frag[((size_t)((kl * 4 + j) * MB + m) * TERMS * 4 + c * 4 + (lane >> 4)) * rt + arow];
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t][m] = mfma16x16x32<FMT>(xf, wf[t], acc[t][m]);
          }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t sb = (it.s[t][g / 2] >> (16 * (g & 1))) & 0xFFFFu;
        const float s = a.scale_dtype == DT_BF16 ? bf16_to_f32((uint16_t)sb) : f16_to_f32((uint16_t)sb);
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) total[t][m][i] = __builtin_fmaf(s, acc[t][m][i], total[t][m][i]);
      }
    }
    if (++kl == kc) kl = 0;
    if (++kb < KB) return;
    kb = kl = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int tile = super * NT + t, v = tile * 16 + (lane & 15);
      const bool in = tile < lay.tiles && v < a.V;
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int b = 16 * m + 4 * (lane >> 4) + i;
          const float val = apply_cast(total[t][m][i], a.reduce_cast);
          if constexpr (MODE == MODE_GREEDY) {
            if (in && b < a.B) best[m][i] = max_u64(best[m][i], argmax_key(val, (uint32_t)v));
          } else if (in && b < a.B) {
            const size_t o = (size_t)b * (size_t)a.out_stride + (size_t)v;
            if (a.out_dtype == DT_F32) ((float*)a.out_logits)[o] = val;
            else if (a.out_dtype == DT_BF16) ((__bf16*)a.out_logits)[o] = (__bf16)val;
            else ((_Float16*)a.out_logits)[o] = (_Float16)val;
          }
          total[t][m][i] = 0.0f;
        }
    }
    super += step;
  };

  ring_pipeline<DEPTH>(n, load, body, [&]() NVJSEL_INLINE {
    if (kc >= KB) {
      w4_stage_hidden<FMT, TERMS, MB, NG>(a, 0, KB, frag, xsum);
      __syncthreads();
    }
  });

  if constexpr (MODE == MODE_GREEDY) {
    __syncthreads();  // the hidden in LDS has been read
    unsigned long long* red = (unsigned long long*)lds;
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned long long k = best[m][i];
#pragma unroll
        for (int x = 8; x >= 1; x >>= 1) k = max_u64(k, shfl_xor_u64(k, x));
        if ((lane & 15) == 0) red[wave * 16 * MB + 16 * m + 4 * (lane >> 4) + i] = k;
      }
    block_commit<kW4Waves, 16 * MB>(red, a.B, a.row_keys);
    finish_rows(a.row_keys, a.counter, a.B, a.out_ids, a.out_best);
  }
}

template <int FMT, int TERMS, int MB, int NG, int MODE>
static int launch_w4(W4Args a, hipStream_t stream) {
  constexpr int NT = 2;
  auto kern = lm_head_w4_kernel<FMT, TERMS, MB, NT, NG, MODE>;
  const W4Layout lay = w4_layout(a.V, a.H, 128 / NG, a.zeros != 0);
  a.rows = 16 * MB;
  if (MB == 1) {
    a.rows = 1;
    while (a.rows < a.B) a.rows *= 2;
  }
  const size_t per_kb = (size_t)a.rows * 256 * TERMS + (size_t)NG * 16 * MB * 4;
  const size_t most = 150 * 1024, red = (size_t)kW4Waves * 16 * MB * 8;
  int chunks = 1;
  while ((size_t)((lay.kblocks + chunks - 1) / chunks) * per_kb > most) ++chunks;
  a.kc = (lay.kblocks + chunks - 1) / chunks;
  size_t lds = a.kc * per_kb;
  if (lds < red) lds = red;
  if (lds > 48 * 1024)
    NVJSEL_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  const int supers = (lay.tiles + NT - 1) / NT, cus = device_cu_count();
  const int need = (supers + kW4Waves - 1) / kW4Waves;
  hipLaunchKernelGGL(kern, dim3(need < cus ? need : cus), dim3(kW4Threads), lds, stream, a);
  NVJSEL_CHECK_LAUNCH("lm_head_w4_kernel");
  return NVJSEL_OK;
}

template <int FMT, int TERMS, int MB, int MODE>
static int launch_w4_group(const W4Args& a, int group, hipStream_t s) {
  if (group == 128) return launch_w4<FMT, TERMS, MB, 1, MODE>(a, s);
  if (group == 64) return launch_w4<FMT, TERMS, MB, 2, MODE>(a, s);
  return launch_w4<FMT, TERMS, MB, 4, MODE>(a, s);
}

// The passes by mode and activation type, each in a translation unit of its own
// (lm_head_w4_bf16.hip, _f16.hip, _f32.hip): batch rows up to kW4Rows, kW4RowsF32 for f32.
static constexpr int kW4Rows = 64, kW4RowsF32 = 32;
int w4_pass_bf16(int mode, const W4Args& a, int group, hipStream_t s);
int w4_pass_f16(int mode, const W4Args& a, int group, hipStream_t s);
int w4_pass_f32(int mode, const W4Args& a, int group, hipStream_t s);

}  // namespace nvjsel
