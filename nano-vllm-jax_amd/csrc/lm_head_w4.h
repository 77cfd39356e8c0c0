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
// total.  Sums are fp32 throughout: a group's, up to 2 x 31 x 128 |x| with the offset, stay
// within it for |x| up to 2^115.  The offset is the smallest one that an
// exponent's mantissa holds: with 128 + q (no shift for a quarter of the nibbles)
// the partial sums are six times larger than the result's terms, and so is their
// rounding.
//
// Packed layout (w4_pack_kernel): blocks of 32 vocabulary rows x 128 k, 2 KB
// each, in the order in which a wave's 16-byte loads feed the 16x16x32 matrix
// instructions: piece t (1 KB), lane l, word j hold row 16 t + (l & 15) and the
// eight k at 32 j + 8 (l >> 4), the nibble of the even k = 2 p at bits 4 p, of 2 p + 1
// at 16 + 4 p.  All k blocks of 32 rows lie together, then the next 32 rows.  The
// scales follow, per block [row of 16][t][128 / group], and the zero points, 16 added,
// in the same order.  Rows past V and k past H are zero with scale zero.
//
// What bounds it: up to 16 rows the weights' stream, V = 248,320, H = 1024, groups of
// 128: one row 26.8 us (131 MB, 4.9 TB/s), 16 rows 25.7; V = 151,936, H = 2560, groups of 64
// with zero points, 8 f16 rows 40.4 us (5.3 TB/s).  With more rows no unit is full: 64 rows,
// V = 128,256, H = 2048, 50 us (670 TFLOP/s), the matrix pipe busy for 26% of it, other vector
// instructions 37%, LDS 25% (more than half of that bank conflicts), and the two waves of a SIMD
// wait for 31% of their time.  Vector and matrix instructions overlap little: of 32 additions
// between four products less than half is hidden.  A shift or an or takes 2.5 to 2.8 clocks
// of a SIMD, v_and_or_b32 or an fma 4 to 4.7, the 16x16x32 product 17 and the 32x32x16 one 33,
// so the smaller tile costs half where up to 16 batch rows are there and nothing where there
// are more.
#pragma once
#include "lm_head_common.h"

namespace nvjsel {

static constexpr int kW4Waves = 8, kW4Threads = 64 * kW4Waves;
static constexpr size_t kW4Lds = 150 * 1024;  // for the hidden and its groups' sums
static constexpr int kW4Turn = 8;             // k blocks between barriers at most, where not all of it fits

struct W4Layout {
  int tiles, kblocks, ng;  // 32-row tiles, 128-wide k blocks, groups per k block
  size_t scales, zeros, total;  // byte offsets of the parts, and the size
};

__host__ __device__ inline W4Layout w4_layout(int V, int H, int group, bool zeros) {
  W4Layout w;
  w.tiles = (V + 31) / 32;
  w.kblocks = (H + 127) / 128;
  w.ng = 128 / group;
  const size_t blocks = (size_t)w.tiles * w.kblocks;
  w.scales = blocks * 2048;
  w.zeros = w.scales + (blocks * 32 * w.ng * 2 + 255) / 256 * 256;
  w.total = w.zeros + (zeros ? (blocks * 32 * w.ng + 255) / 256 * 256 : 0);
  return w;
}

struct W4Args {
  const void* hidden;
  int hidden_dtype;
  const uint8_t* packed;
  int scale_dtype;
  int zeros;   // zero points are there
  int V, H;
  int B;       // batch rows of this pass
  int blocks;  // of each group of rows that a block holds; the groups follow each other in the grid
  int kc;      // k blocks of the hidden that LDS holds
  int reduce_cast;
  unsigned long long* row_keys;
  unsigned int* counter;
  int32_t* out_ids;
  float* out_best;
  void* out_logits;
  int out_dtype;
  long long out_stride;
};

// 16 + q of the eight nibbles of a packed word, as bf16 or f16 pairs.  The mask and
// the exponents are held in registers: as literals they take two instructions a
// pair where v_and_or_b32 takes one (V = 248,320, H = 1024, one row 29.1 against 28.0 us).
struct W4Consts {
  uint32_t mask, base;
};
template <int FMT>
__device__ __forceinline__ W4Consts w4_consts() {
  W4Consts c;
  if constexpr (FMT == DT_BF16) {  // mantissa bits 3..6
    asm("s_mov_b32 %0, 0x00780078" : "=s"(c.mask));
    asm("v_mov_b32 %0, 0x41804180" : "=v"(c.base));
  } else {  // mantissa bits 6..9
    asm("s_mov_b32 %0, 0x03c003c0" : "=s"(c.mask));
    asm("v_mov_b32 %0, 0x4c004c00" : "=v"(c.base));
  }
  return c;
}
template <int FMT>
__device__ __forceinline__ u32x4_t w4_unpack(uint32_t w, const W4Consts& c) {
  u32x4_t r;
  if constexpr (FMT == DT_BF16) {
    r.x = ((w << 3) & c.mask) | c.base;
    r.y = ((w >> 1) & c.mask) | c.base;
    r.z = ((w >> 5) & c.mask) | c.base;
    r.w = ((w >> 9) & c.mask) | c.base;
  } else {
    r.x = ((w << 6) & c.mask) | c.base;
    r.y = ((w << 2) & c.mask) | c.base;
    r.z = ((w >> 2) & c.mask) | c.base;
    r.w = ((w >> 6) & c.mask) | c.base;
  }
  return r;
}

template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}

// k blocks kb0 .. of the hidden into LDS, as the matrix instructions' operands:
// 16-byte slots [((4 kb + j) MB + mb) TERMS + t][k quarter][row of RT].  Three terms: x =
// the bf16 values that its leading, next and last eight bits make (exact); a value
// that is not finite keeps its first term only.  No terms (0): f32 too, the three of
// up to four batch rows as rows 4 t + b of one matrix tile, a third of the products; the
// last four rows stay as LDS was and are left out of the results.  Then, by the matrix cores, the
// groups' sums of activations times -1 (zero points) or -(16 + 8): xsum [group][MB][16],
// with three terms the leading one's sums, then the other two's.  Each has accumulators of
// its own: at the leading term's offset the others would lose half of their bits (16
// rows, H = 1024: relative error 1.5e-6 with one sum, 2e-7 with two).
// first(): the loads that may be on their way while the weights' first ones are
// requested; rest(): everything else.
template <int FMT, int TERMS, int MB, int RT, int NG, bool ZEROS>
struct W4Stage {
  static constexpr int U = TERMS == 1 ? 8 : 4, EACH = kW4Threads / 16, LD = TERMS == 1 ? 1 : 2;
  static constexpr int TM = TERMS ? TERMS : 1, ROWS = TERMS ? RT * MB : 4;  // terms of a slot, rows to load
  static constexpr int XS = TERMS == 3 ? 2 : 1;                              // sums of a group
  u32x4_t v[U][LD];

  template <int N = U>
  __device__ __forceinline__ void load(const W4Args& a, int kb0, int items, int it0) {
    const int u = (int)threadIdx.x & 15;  // eight k of a k block
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int it = it0 + i * EACH, row = it % (ROWS), k = (kb0 + it / (ROWS)) * 128 + 8 * u;
      const bool in = it < items && row < a.B && k < a.H;
      const size_t at = in ? (size_t)row * a.H + k : 0;  // always a load, of the first values where none is wanted
#pragma unroll
      for (int h = 0; h < LD; ++h) {
        if constexpr (TERMS == 1) v[i][h] = *(const u32x4_any_t*)((const uint16_t*)a.hidden + at);
        else v[i][h] = *(const u32x4_any_t*)((const float*)a.hidden + at + 4 * h);
      }
    }
  }
  // Item i's eight values in their slots, kb the k block's place in LDS; put: its terms as
  // they go there, zero where the item lies outside.
  static constexpr int PUT = TERMS == 1 ? 1 : 3;
  __device__ __forceinline__ void put(int i, bool in, int kb, int row, u32x4_t* frag, u32x4_t (&out)[PUT]) {
    const int u = (int)threadIdx.x & 15;
    u32x4_t* dst = frag + (((kb * 4 + (u >> 2)) * MB + row / RT) * TM * 4 + (u & 3)) * RT + row % RT;
    if constexpr (TERMS == 1) {
      out[0] = in ? v[i][0] : u32x4_t{0u, 0u, 0u, 0u};
      *dst = out[0];
    } else {
      uint32_t h[3][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t b = in ? v[i][e >> 2][e & 3] : 0u;
        const float x = __uint_as_float(b);
        const bool fin = (b & 0x7F800000u) != 0x7F800000u;
        h[0][e] = fin ? b >> 16 : bf16_bits_rne(x);
        const float r1 = x - __uint_as_float(b & 0xFFFF0000u);
        h[1][e] = fin ? __float_as_uint(r1) >> 16 : 0u;
        const float r2 = r1 - __uint_as_float(__float_as_uint(r1) & 0xFFFF0000u);
        h[2][e] = fin ? __float_as_uint(r2) >> 16 : 0u;
      }
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        out[t] = u32x4_t{h[t][0] | h[t][1] << 16, h[t][2] | h[t][3] << 16, h[t][4] | h[t][5] << 16, h[t][6] | h[t][7] << 16};
        dst[TERMS ? t * 4 * RT : 4 * t] = out[t];
      }
    }
  }
  __device__ __forceinline__ void store(const W4Args& a, int kb0, int items, int it0, u32x4_t* frag) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int it = it0 + i * EACH, row = it % (ROWS), kb = it / (ROWS), k = (kb0 + kb) * 128 + 8 * ((int)threadIdx.x & 15);
      if (it >= items) break;
      u32x4_t out[PUT];
      put(i, row < a.B && k < a.H, kb, row, frag, out);
    }
  }
  // One k block at a time, on its way while others are in work (STAGED): load() with
  // one k block's items, then this, its groups' sums by the lanes that hold them.
  static_assert(ROWS <= EACH * U, "");
  __device__ __forceinline__ void store_one(const W4Args& a, int kb0, int at, u32x4_t* frag, float* xsum) {
    const int u = (int)threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < (ROWS + EACH - 1) / EACH; ++i) {
      const int row = ((int)threadIdx.x >> 4) + i * EACH;
      if (ROWS % EACH && row >= ROWS) break;
      u32x4_t out[PUT];
      put(i, row < a.B && kb0 * 128 + 8 * u < a.H, at, row, frag, out);
      float sum[PUT];
#pragma unroll
      for (int t = 0; t < PUT; ++t) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = out[t][e >> 1];
          s += FMT == DT_BF16 ? __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16) : f16_to_f32((uint16_t)(e & 1 ? w >> 16 : w));
        }
        sum[t] = s;
      }
      if constexpr (TERMS == 3) sum[1] += sum[2];
      const float f = ZEROS ? -1.0f : -24.0f;
#pragma unroll
      for (int t = 0; t < (TERMS == 0 ? 3 : XS); ++t) {
        float s = sum[t];  // over the 16 / NG lanes of a group
        s += dpp_f32<0xB1>(s);
        s += dpp_f32<0x4E>(s);
        if (NG <= 2) s += dpp_f32<0x141>(s);
        if (NG == 1) s += dpp_f32<0x140>(s);
        if (u % (16 / NG) == 0)
          xsum[((at * NG + u / (16 / NG)) * MB + row / 16) * XS * 16 + (TERMS == 0 ? 4 * t + row : 16 * t + row % 16)] = s * f;
      }
    }
  }
  __device__ __forceinline__ void load_one(const W4Args& a, int kb) {
    load<(ROWS + EACH - 1) / EACH>(a, kb, ROWS, (int)threadIdx.x >> 4);
  }
  __device__ __forceinline__ void first(const W4Args& a, int kb0, int nkb) {
    load(a, kb0, ROWS * nkb, (int)threadIdx.x >> 4);
  }
  __device__ __forceinline__ void rest(const W4Args& a, int kb0, int nkb, u32x4_t* frag, float* xsum) {
    const int items = ROWS * nkb;
    store(a, kb0, items, (int)threadIdx.x >> 4, frag);
    for (int it0 = ((int)threadIdx.x >> 4) + U * EACH; it0 < items; it0 += U * EACH) {
      load(a, kb0, items, it0);
      store(a, kb0, items, it0, frag);
    }
    __syncthreads();
    const int lane = (int)threadIdx.x & 63;
    const uint32_t one =
        ZEROS ? (FMT == DT_BF16 ? 0xBF80BF80u : 0xBC00BC00u) : (FMT == DT_BF16 ? 0xC1C0C1C0u : 0xCE00CE00u);
    const u32x4_t ones{one, one, one, one};
    const u32x4_t* mine = frag + (lane >> 4) * RT + (lane & (RT - 1));
    for (int g = (int)threadIdx.x >> 6; g < nkb * NG; g += kW4Waves) {
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        f32x4_t d[XS];
#pragma unroll
        for (int h = 0; h < XS; ++h) d[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4 / NG; ++j)
#pragma unroll
          for (int c = TM - 1; c >= 0; --c)
            d[c ? XS - 1 : 0] =
                mfma16x16x32<FMT>(mine[(((g * (4 / NG) + j) * MB + m) * TM + c) * 4 * RT], ones, d[c ? XS - 1 : 0]);
#pragma unroll
        for (int h = 0; h < XS; ++h)
          if ((lane & 15) == 0) *(f32x4_t*)(xsum + ((g * MB + m) * XS + h) * 16 + 4 * (lane >> 4)) = d[h];
      }
    }
    __syncthreads();
  }
};

// One block per CU, eight waves.  A wave takes a block of 32 vocabulary rows at a
// time and runs over all of H, its next k blocks' pieces on the way in registers
// (DEPTH); the waves share the hidden in LDS, all of it where it fits, kc k blocks in
// a ring where not (STAGED).  Matrix tile: M = batch rows (MB tiles of 16), N =
// vocabulary rows, so that a lane's results share their scale.  RT: batch rows that
// have slots in LDS (8: the others repeat them).
//
// Rows go round all waves of the device while every wave gets some; what is left is
// dealt to the blocks, and a block splits its rest by k blocks over its waves, which
// join their parts through LDS at the end (V = 151,936, H = 2560, 8 rows: 46 us with
// whole tiles only, 2.3 rounds of them, 42 split).  STAGED waves walk the k blocks
// together, two tiles at a time (NB: half as many reads of the hidden), and repeat the
// last tile instead; with every k block the block stores one of the hidden, requested
// with the last one, for half a ring later, and a barrier every half ring keeps both
// ends apart (64 rows, V = 128,256, H = 2048: 58 us where all waves stopped to fill the
// LDS, 50 so).
template <int FMT, int TERMS, int MB, int RT, int NG, bool ZEROS, bool STAGED, int MODE>
__global__ void __launch_bounds__(kW4Threads, 2) lm_head_w4_kernel(W4Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int TM = TERMS ? TERMS : 1, XS = TERMS == 3 ? 2 : 1, ROWS = TERMS ? RT * MB : 4;
  constexpr int NB = STAGED ? 2 : 1, DEPTH = STAGED ? 2 : 4, NT = 2 * NB;
  const W4Layout lay = w4_layout(a.V, a.H, 128 / NG, ZEROS);
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  // the block's group of batch rows
  const int batch = a.B, blocks = a.blocks, row0 = (int)((unsigned)blockIdx.x / (unsigned)blocks) * ROWS;
  const int block = (int)blockIdx.x - row0 / ROWS * blocks;
  a.B = batch - row0 < ROWS ? batch - row0 : ROWS;
  a.hidden = (const char*)a.hidden + (size_t)row0 * a.H * (TERMS == 1 ? 2 : 4);
  const int KB = lay.kblocks, kc = a.kc, col = lane & 15;
  u32x4_t* frag = (u32x4_t*)lds;
  float* xsum = (float*)(lds + (size_t)kc * 256 * TM * RT * MB);
  const u32x4_t* mine = frag + (lane >> 4) * RT + (lane & (RT - 1));
  const float* xmine = xsum + 4 * (lane >> 4);

  const int step = blocks * kW4Waves, first = block * kW4Waves + wave;
  const int supers = (lay.tiles + NB - 1) / NB;
  const int full = STAGED ? (supers - block * kW4Waves + step - 1) / step : lay.tiles / step;  // whole rounds
  // the block's rest: tiles from rest0, its k blocks dealt to the waves
  int rest0 = 0, nrest = 0;
  if (!STAGED) {
    const int rest = lay.tiles - full * step;
    const int each = (int)((unsigned)rest / (unsigned)blocks), more = rest - each * blocks;
    const int r0 = each * block + (block < more ? block : more), r1 = r0 + each + (block < more);
    rest0 = full * step + r0;
    nrest = (r1 - r0) * KB;
  }
  auto from = [&](int w) { return (int)((unsigned)(nrest * w) / kW4Waves); };  // first k block of wave w's part
  const int p0 = from(wave), p1 = from(wave + 1);
  const int n = full * KB + p1 - p0;
  const int tail_tile = rest0 + p0 / KB, tail_kb = p0 % KB;

  const W4Consts consts = w4_consts<FMT>();
  const uint32_t bf16_mask = a.scale_dtype == DT_BF16 ? 0xFFFFFFFFu : 0u;
  const uint32_t zoff = (uint32_t)(col * 2 * NG) & ~3u, zshift = NG == 1 ? (col & 1) * 16 : 0;

  // Scales and zero points are loaded as the aligned words that hold them: a 16-bit
  // load's extension would be waited for a round of the ring early.
  struct Item {
    u32x4_t w[NT];
    uint32_t s[NB][NG];  // two 16-bit scales each: [t][g]
    uint32_t z[NB][(NG + 1) / 2];
  };
  Item ring[DEPTH];

  int lkb = full ? 0 : tail_kb, ltile = full ? first : tail_tile, lfull = full;  // the item to be requested next
  auto load = [&](auto D) NVJSEL_INLINE {
    Item& it = ring[decltype(D)::value];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int at = ltile * NB + n, tile = at < lay.tiles ? at : lay.tiles - 1;
      const size_t blk = (size_t)tile * KB + lkb;
      const u32x4_t* wb = (const u32x4_t*)(a.packed + blk * 2048) + lane;
      it.w[2 * n] = __builtin_nontemporal_load(wb);
      it.w[2 * n + 1] = __builtin_nontemporal_load(wb + 64);
      const uint32_t* sb = (const uint32_t*)(a.packed + lay.scales + blk * (64 * NG)) + col * NG;
      if constexpr (NG == 4) {
        const u32x4_t v = *(const u32x4_t*)sb;
#pragma unroll
        for (int g = 0; g < 4; ++g) it.s[n][g] = v[g];
      } else if constexpr (NG == 2) {
        const uint64_t v = *(const uint64_t*)sb;
        it.s[n][0] = (uint32_t)v;
        it.s[n][1] = (uint32_t)(v >> 32);
      } else it.s[n][0] = *sb;
      if constexpr (ZEROS) {
        const uint8_t* zb = a.packed + lay.zeros + blk * (32 * NG) + zoff;
        if constexpr (NG == 4) {
          const uint64_t v = *(const uint64_t*)zb;
          it.z[n][0] = (uint32_t)v;
          it.z[n][1] = (uint32_t)(v >> 32);
        } else it.z[n][0] = *(const uint32_t*)zb;
      }
    }
    if (++lkb == KB) {
      --lfull;
      lkb = lfull == 0 ? tail_kb : 0;
      ltile = lfull == 0 ? tail_tile : lfull > 0 ? ltile + step : ltile + 1;
    }
  };

  // greedy: the best so far of each row among this lane's columns; no index yet: ~0, beside a NaN
  float total[NT][MB][4], bval[MB][4], foreign[NT][MB][4];  // foreign: not STAGED
  uint32_t bidx[MB][4];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bval[m][i] = NAN;
      bidx[m][i] = 0xFFFFFFFFu;
#pragma unroll
      for (int t = 0; t < NT; ++t) total[t][m][i] = foreign[t][m][i] = 0.0f;
    }

  char* orow[MB];  // logits: the rows that this lane stores (f32: the first of four)
  if constexpr (MODE == MODE_LOGITS) {
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const bool f32 = a.out_dtype == DT_F32;
      orow[m] = (char*)a.out_logits +
                (size_t)(row0 + 16 * m + 4 * (lane >> 4) + (f32 ? 0 : lane & 3)) * (size_t)a.out_stride * (f32 ? 4 : 2);
    }
  }

  // A tile's totals are whole: rounded, and scored or stored.
  auto finish_tile = [&](int tile) NVJSEL_INLINE {
    if constexpr (TERMS == 0) {  // the terms of a row meet: lane quarters 0, 1 and 2
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = xpose_add16(lane < 48 ? total[t][0][i] : 0.0f, lane < 48 ? total[t][0][i] : 0.0f);
          total[t][0][i] = xpose_add32(x, x);
        }
    }
    if (a.reduce_cast == 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) total[t][m][i] = round_bf16(total[t][m][i]);
    } else if (a.reduce_cast == 2) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) total[t][m][i] = round_f16(total[t][m][i]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int v = (tile * NB + (t >> 1)) * 32 + 16 * (t & 1) + col;
      const bool in = v < a.V;
      if constexpr (MODE == MODE_GREEDY) {
        bool up = false;  // seldom: a lane's best of so many tiles
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) up |= !(total[t][m][i] <= bval[m][i]);
        if (__any(up && in)) {
#pragma unroll
          for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = total[t][m][i], y = bval[m][i];  // in order of index: equal ones stay, the first NaN too
              if (in && (bidx[m][i] == 0xFFFFFFFFu || x > y || (x != x && y == y))) {
                bval[m][i] = x;
                bidx[m][i] = (uint32_t)v;
              }
            }
        }
      } else {
        // 16-bit logits are transposed in quads of lanes (four rows x four columns) and
        // stored 8 bytes per lane, at any element address; the vocabulary's last quad
        // may be partial
        const int v4 = v & ~3, left = a.V - v4;
#pragma unroll
        for (int m = 0; m < MB; ++m) {
          const int b = 16 * m + 4 * (lane >> 4);
          if (a.out_dtype != DT_F32) {
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = total[t][m][i];
            const uint2 q = quad_transpose16(x, a.out_dtype, lane);
            if (left > 0 && b + (lane & 3) < a.B) {
              uint16_t* out = (uint16_t*)orow[m] + v4;
              if (left >= 4) {
                *(u32x2_any_t*)out = u32x2_t{q.x, q.y};
              } else {
                out[0] = (uint16_t)q.x;
                if (left > 1) out[1] = (uint16_t)(q.x >> 16);
                if (left > 2) out[2] = (uint16_t)q.y;
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (in && b + i < a.B) ((float*)orow[m])[(size_t)i * (size_t)a.out_stride + v] = total[t][m][i];
          }
        }
      }
    }
  };

  int kb = full ? 0 : tail_kb, tile = full ? first : tail_tile, left = full;  // the item in work
  // STAGED: the item's place in LDS, the items to the next barrier; the k block on its way and its place
  int at = 0, turn = 0, skb = kc / 2 % KB, sat = kc / 2;
  W4Stage<FMT, TERMS, MB, RT, NG, ZEROS> st;
  auto body = [&](auto D) NVJSEL_INLINE {
    if constexpr (STAGED) {
      if (turn == 0) {
        __syncthreads();
        turn = kc / 2;
      }
      --turn;
      st.store_one(a, skb, sat, frag, xsum);
      if (++skb == KB) skb = 0;
      if (++sat == kc) sat = 0;
      st.load_one(a, skb);
    }
    const Item& it = ring[decltype(D)::value];
    const int kx = STAGED ? at : kb;
    const u32x4_t* fk = mine + kx * (4 * MB * TM * 4 * RT);
    const float* xk = xmine + kx * (NG * MB * XS * 16);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4_t acc[XS][NT][MB];
#pragma unroll
      for (int h = 0; h < XS; ++h)
#pragma unroll
        for (int m = 0; m < MB; ++m) {
          const f32x4_t xs = *(const f32x4_t*)(xk + ((g * MB + m) * XS + h) * 16);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if constexpr (ZEROS) {
              const int zi = (t & 1) * NG + g;  // byte of the block's zero points of this row
              const float z = (float)(((it.z[t >> 1][zi >> 2] >> zshift) >> (8 * (zi & 3))) & 0xFFu);  // packed as 16 + z
              acc[h][t][m] = f32x4_t{xs.x * z, xs.y * z, xs.z * z, xs.w * z};
            } else acc[h][t][m] = xs;
          }
        }
#pragma unroll
      for (int j = g * 4 / NG; j < (g + 1) * 4 / NG; ++j) {
        u32x4_t wf[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) wf[t] = w4_unpack<FMT>(it.w[t][j], consts);
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int c = TM - 1; c >= 0; --c) {
            const u32x4_t xf = fk[((j * MB + m) * TM + c) * 4 * RT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
              acc[c ? XS - 1 : 0][t][m] = mfma16x16x32<FMT>(xf, wf[t], acc[c ? XS - 1 : 0][t][m]);
          }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int si = (t & 1) * NG + g;  // 16-bit scale of the block's scales of this row
        const uint32_t sb = it.s[t >> 1][si >> 1] >> (16 * (si & 1));
        const uint32_t fh = __float_as_uint(f16_to_f32((uint16_t)sb));
        const float s = __uint_as_float((sb << 16 & bf16_mask) | (fh & ~bf16_mask));
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float sum = XS == 2 ? acc[XS - 1][t][m][i] + acc[0][t][m][i] : acc[0][t][m][i];
            total[t][m][i] = __builtin_fmaf(s, sum, total[t][m][i]);
          }
      }
    }
    if (STAGED && ++at == kc) at = 0;
    if (++kb < KB) return;
    if (!STAGED && left == 0 && tile == tail_tile && tail_kb != 0) {  // the end of another wave's tile
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) foreign[t][m][i] = total[t][m][i];
    } else {
      finish_tile(tile);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) total[t][m][i] = 0.0f;
    if (left > 0) --left;  // as the loads go
    const bool to_tail = left == 0 && (tile < rest0 || STAGED);
    kb = to_tail ? tail_kb : 0;
    tile = to_tail ? tail_tile : left > 0 ? tile + step : tile + 1;
  };

  // Every load is unconditional (tiles past the end repeat the last one), so that the
  // waits count the same requests on every path to a body: with bounds tests before
  // the first loads each round of the ring waited for all of it.
  if constexpr (STAGED) {
    static_for<DEPTH - 1>([&](auto D) NVJSEL_INLINE { load(D); });
    for (int i = 0; i < kc / 2; ++i) {
      st.load_one(a, i % KB);
      st.store_one(a, i % KB, i, frag, xsum);
    }
    st.load_one(a, skb);
  } else {
    st.first(a, 0, KB);
    static_for<DEPTH - 1>([&](auto D) NVJSEL_INLINE { load(D); });
    st.rest(a, 0, KB, frag, xsum);
  }
  int i = 0;
  for (; i + DEPTH <= n; i += DEPTH)
    static_for<DEPTH>([&](auto D) NVJSEL_INLINE {
      load(std::integral_constant<int, (decltype(D)::value + DEPTH - 1) % DEPTH>{});
      body(D);
    });
  static_for<DEPTH - 1>([&](auto D) NVJSEL_INLINE {
    if (i + decltype(D)::value < n) body(D);
  });

  if (nrest) {  // block-uniform: the parts of tiles meet
    __syncthreads();  // the hidden in LDS has been read
    float* part = (float*)lds;  // [wave][t][m][i][lane]
    const int pend = p1 % KB != 0 && p1 > p0 ? p1 / KB : -1;  // this wave's last tile is not whole
    const bool owns = pend >= 0 && pend * KB >= p0;           // and begins here
    if (p1 > p0 && tail_kb != 0) {
      const bool ended = (p0 / KB + 1) * KB <= p1;  // its part reaches the tile's end: set aside; else still in total
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            part[(((wave * NT + t) * MB + m) * 4 + i) * 64 + lane] = ended ? foreign[t][m][i] : total[t][m][i];
    }
    __syncthreads();
    if (owns) {
      for (int w = wave + 1; w < kW4Waves && from(w) < (pend + 1) * KB; ++w) {
        if (from(w + 1) == from(w)) continue;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) total[t][m][i] += part[(((w * NT + t) * MB + m) * 4 + i) * 64 + lane];
      }
      finish_tile(rest0 + pend);
    }
  }

  if constexpr (MODE == MODE_GREEDY) {
    __syncthreads();  // LDS has been read
    unsigned long long* red = (unsigned long long*)lds;
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned long long k = bidx[m][i] == 0xFFFFFFFFu ? 0ull : argmax_key(bval[m][i], bidx[m][i]);
#pragma unroll
        for (int x = 8; x >= 1; x >>= 1) k = max_u64(k, shfl_xor_u64(k, x));
        if (col == 0) red[wave * 16 * MB + 16 * m + 4 * (lane >> 4) + i] = k;
      }
    block_commit<kW4Waves, 16 * MB>(red, a.B, a.row_keys + row0);
    finish_rows(a.row_keys, a.counter, batch, a.out_ids, a.out_best);
  }
}

// How a pass is laid over the device by one shape of tiles.
struct W4Plan {
  int groups, blocks;  // of batch rows; blocks of each
  int kc;              // k blocks of the hidden in LDS at a time
  bool staged;
  size_t lds;
  float us;  // estimated
};

// Rows beyond a tile's go to groups of blocks of their own, which read the same weights;
// blocks with the same tiles share an XCD's L2 (blocks are dealt to the 8 XCDs in turn).
static inline W4Plan w4_plan(const W4Args& a, int group, int terms, int mb, int rt) {
  const W4Layout lay = w4_layout(a.V, a.H, group, a.zeros);
  const size_t per_kb = (size_t)rt * mb * 256 * (terms ? terms : 1) + (size_t)lay.ng * 16 * mb * (terms == 3 ? 8 : 4);
  const int rows = terms ? rt * mb : 4, cus = device_cu_count();
  W4Plan p;
  p.groups = (a.B + rows - 1) / rows;
  const int fit = (int)(kW4Lds / per_kb);
  p.staged = lay.kblocks > fit;
  p.kc = p.staged ? 2 * (fit / 2 < kW4Turn ? fit / 2 : kW4Turn) : lay.kblocks;
  p.lds = p.kc * per_kb;
  const size_t parts = (size_t)kW4Waves * mb * 2048;  // of the tiles that waves split; the rows' keys need less
  if (p.lds < parts) p.lds = parts;
  const int waves = p.staged ? (lay.tiles + 1) / 2 : lay.tiles, need = p.staged ? (waves + kW4Waves - 1) / kW4Waves : waves;
  int most = cus / p.groups;
  if (p.groups > 1 && most > 8) most &= ~7;
  if (most < 1) most = 1;
  p.blocks = need < most ? need : most;

  // us: a call (between logits' and greedy's, so that both add up in the same order), and
  // per k block the hidden's staging and a round of all waves: a fit to timings of every
  // shape.  Over 175 greedy calls (1..256 rows, V 8,000..248,320, H 1024..8192) the shape that
  // it picks took 0.5% longer than the fastest on average and 12% at most, the widest one 32%.
  struct Fit {
    float call, stage, round, staged;
  };
  static constexpr Fit fits[6] = {
      {6.4f, 0.06f, 0.48f, 1.00f},   // eight rows
      {6.4f, 0.10f, 0.53f, 0.98f},   // one tile of 16
      {7.4f, 0.22f, 0.70f, 1.42f},   // two
      {9.6f, 0.55f, 1.21f, 2.20f},   // four
      {6.6f, 0.09f, 0.50f, 1.20f},   // four rows of three terms
      {6.5f, 0.34f, 0.85f, 1.90f}};  // one tile, three terms apart
  const Fit& f = fits[terms == 3 ? 5 : terms == 0 ? 4 : rt == 8 ? 0 : mb == 4 ? 3 : mb];
  const int slots = p.blocks * kW4Waves;
  const float each = p.staged ? f.staged * ((waves + slots - 1) / slots)
                              : f.stage + f.round * fmaxf((float)waves / slots, 1.0f / kW4Waves);
  p.us = f.call + lay.kblocks * each;
  return p;
}

template <int FMT, int TERMS, int MB, int RT, int NG, bool ZEROS, int MODE>
static int launch_w4(W4Args a, const W4Plan& p, hipStream_t stream) {
  a.kc = p.kc;
  a.blocks = p.blocks;
  auto kern = p.staged ? lm_head_w4_kernel<FMT, TERMS, MB, RT, NG, ZEROS, true, MODE>
                       : lm_head_w4_kernel<FMT, TERMS, MB, RT, NG, ZEROS, false, MODE>;
  if (p.lds > 48 * 1024)
    NVJSEL_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds));
  hipLaunchKernelGGL(kern, dim3(p.blocks * p.groups), dim3(kW4Threads), p.lds, stream, a);
  NVJSEL_CHECK_LAUNCH("lm_head_w4_kernel");
  return NVJSEL_OK;
}

template <int FMT, int TERMS, int MB, int RT, int MODE>
static int launch_w4_group(const W4Args& a, int group, const W4Plan& p, hipStream_t s) {
  if (a.zeros) {
    if (group == 128) return launch_w4<FMT, TERMS, MB, RT, 1, true, MODE>(a, p, s);
    if (group == 64) return launch_w4<FMT, TERMS, MB, RT, 2, true, MODE>(a, p, s);
    return launch_w4<FMT, TERMS, MB, RT, 4, true, MODE>(a, p, s);
  }
  if (group == 128) return launch_w4<FMT, TERMS, MB, RT, 1, false, MODE>(a, p, s);
  if (group == 64) return launch_w4<FMT, TERMS, MB, RT, 2, false, MODE>(a, p, s);
  return launch_w4<FMT, TERMS, MB, RT, 4, false, MODE>(a, p, s);
}

// The widest tile reads and unpacks the weights the fewest times; narrower ones leave more
// of the hidden in LDS, and stage it sooner (us a call, its host time of some 9 among
// them: 8 rows, V = 50,000, H = 8192: 46 with 8 rows' slots, 68 with 16; 64 rows, V = 32,000, H =
// 4096: 41 with 16 rows a tile, 74 with 64, staged) and give a small vocabulary's tiles to more
// blocks (48 rows, V = 8000, H = 1024: 11 with 16 rows, 22 with 64), but a large one costs more with
// them (64 rows, V = 248,320, H = 1024: 70 with 16, 55 with 64).  f32: the terms apart where the
// hidden stays in LDS so (16 rows, V = 248,320, H = 1024: 39, 75 in fours; 64 rows 107, 249 in
// fours), rows in fours where not (16 rows, V = 8000, H = 4096: 21, 65 staged).  Every group of 16
// f32 rows unpacks the weights again (V = 128,256, H = 2048: 16 / 32 / 64 / 128 rows 45 / 71 / 127 /
// 236 us); two tiles of three terms were no faster than two groups of one.
template <int FMT, int TERMS, int MODE>
static int w4_pass(const W4Args& a, int group, hipStream_t s) {
  if constexpr (TERMS == 3) {
    const W4Plan fours = w4_plan(a, group, 0, 1, 16), one = w4_plan(a, group, 3, 1, 16);
    if (a.B <= 4 || fours.us < one.us) return launch_w4_group<FMT, 0, 1, 16, MODE>(a, group, fours, s);
    return launch_w4_group<FMT, 3, 1, 16, MODE>(a, group, one, s);
  } else {
    W4Plan best = w4_plan(a, group, TERMS, 1, 8);
    int mb = 0;
    for (int m = 1; a.B > 8 * m && m <= 4; m *= 2) {
      const W4Plan p = w4_plan(a, group, TERMS, m, 16);
      if (p.us < best.us) {
        best = p;
        mb = m;
      }
    }
    if (mb == 4) return launch_w4_group<FMT, TERMS, 4, 16, MODE>(a, group, best, s);
    if (mb == 2) return launch_w4_group<FMT, TERMS, 2, 16, MODE>(a, group, best, s);
    if (mb == 1) return launch_w4_group<FMT, TERMS, 1, 16, MODE>(a, group, best, s);
    return launch_w4_group<FMT, TERMS, 1, 8, MODE>(a, group, best, s);
  }
}

// The passes by mode and activation type, each in a translation unit of its
// own; up to kW4Rows batch rows, whose groups read the weights together (256 rows, V =
// 151,936, H = 1024: 150 us in launches of 64 rows, 108 of 128, 98 of 256).
static constexpr int kW4Rows = 256;
int w4_greedy_bf16(const W4Args& a, int group, hipStream_t s);
int w4_greedy_f16(const W4Args& a, int group, hipStream_t s);
int w4_greedy_f32(const W4Args& a, int group, hipStream_t s);
int w4_logits_bf16(const W4Args& a, int group, hipStream_t s);
int w4_logits_f16(const W4Args& a, int group, hipStream_t s);
int w4_logits_f32(const W4Args& a, int group, hipStream_t s);

}  // namespace nvjsel
