// LM head with 4-bit weights (lm_head_w4.h): packing, rounding weights to 4
// bits, and the C entry points.
#include "lm_head_w4.h"

namespace nvjsel {

// One thread per two packed 32-bit words of a block; the first ones also write
// its scales and zero points.
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* __restrict__ q, const uint16_t* __restrict__ scales,
                                                      const uint8_t* __restrict__ zeros, int V, int H, int group,
                                                      uint8_t* __restrict__ packed) {
  const W4Layout lay = w4_layout(V, H, group, zeros != nullptr);
  const size_t blocks = (size_t)lay.tiles * lay.kblocks;
  const int G = H / group;
  for (size_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int tile = (int)(blk / lay.kblocks), kb = (int)(blk % lay.kblocks);
    const int t = (int)threadIdx.x, lane = t >> 2, j = t & 3, k0 = kb * 128 + 32 * j + 8 * (lane >> 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int v = tile * 32 + 16 * h + (lane & 15);
      uint32_t w = 0;
      if (v < V && k0 < H) {  // H is a multiple of 32: the eight k are all there
        const uint8_t* src = q + ((size_t)v * H + k0) / 2;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const uint32_t b = src[p];
          w |= (b & 15u) << (4 * p) | (b >> 4) << (16 + 4 * p);
        }
      }
      ((uint32_t*)packed)[blk * 512 + h * 256 + t] = w;
    }
    if (t < 32 * lay.ng) {
      const int r = t / lay.ng, g = kb * lay.ng + t % lay.ng, vs = tile * 32 + 16 * (r & 1) + (r >> 1);
      const bool in = vs < V && g < G;
      ((uint16_t*)(packed + lay.scales))[blk * 32 * lay.ng + t] = in ? scales[(size_t)vs * G + g] : (uint16_t)0;
      if (zeros) (packed + lay.zeros)[blk * 32 * lay.ng + t] = in ? (uint8_t)(16 + (zeros[(size_t)vs * G + g] & 15)) : (uint8_t)16;
    }
  }
}

// Rounds weights to 4 bits by groups of one row: one wave per (row, group),
// element strides sv and sk.  Without zero points s = max|w| / 7 and q - 8 =
// rint(w / s) in -8..7; with them s = (max - min) / 15 over the values and 0,
// z = rint(-min / s).  The codes are taken against the scale as it is stored.  A group
// that holds a NaN or an infinity gets a NaN scale, which makes its row's logits NaN; a
// finite one whose scale is beyond its type the type's largest, and its codes end at 0 and 15.
__global__ void __launch_bounds__(256) w4_quantize_kernel(const void* __restrict__ weight, int wdt, int64_t sv, int64_t sk,
                                                          int V, int H, int group, int sdt, uint8_t* __restrict__ q,
                                                          uint16_t* __restrict__ scales, uint8_t* __restrict__ zeros) {
  const int G = H / group, lane = (int)threadIdx.x & 63;
  const size_t items = (size_t)V * G, step = (size_t)gridDim.x * 4;
  for (size_t i = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < items; i += step) {
    const int v = (int)(i / G), g = (int)(i % G);
    const bool two = 2 * lane < group;  // a lane holds elements 2 lane and 2 lane + 1
    const int64_t e = (int64_t)v * sv + (int64_t)(g * group + 2 * lane) * sk;
    const float a = two ? load_as_f32(weight, wdt, (size_t)e) : 0.0f;
    const float b = two ? load_as_f32(weight, wdt, (size_t)(e + sk)) : 0.0f;
    float lo = fminf(fminf(a, b), 0.0f), hi = fmaxf(fmaxf(a, b), 0.0f);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      lo = fminf(lo, __shfl_xor(lo, m, 64));
      hi = fmaxf(hi, __shfl_xor(hi, m, 64));
    }
    float raw = zeros ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f;
    if (!__builtin_isfinite(raw)) raw = hi / 15.0f - lo / 15.0f;  // hi - lo is beyond f32
    const bool finite = !__any(!__builtin_isfinite(a) || !__builtin_isfinite(b));  // of the wave's group
    const float most = sdt == DT_BF16 ? 0x1.FEp127f : 65504.0f;
    const float s = finite ? fminf(round_to_dtype(raw, sdt), most) : NAN;
    float z = 8.0f;
    if (zeros) z = s > 0.0f ? fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f) : 0.0f;
    const float ca = s > 0.0f ? fminf(fmaxf(rintf(a / s) + z, 0.0f), 15.0f) : z;
    const float cb = s > 0.0f ? fminf(fmaxf(rintf(b / s) + z, 0.0f), 15.0f) : z;
    if (two) q[((size_t)v * H + g * group) / 2 + lane] = (uint8_t)((uint32_t)ca | (uint32_t)cb << 4);
    if (lane == 0) {
      scales[i] = (uint16_t)(sdt == DT_BF16 ? bf16_bits_rne(s) : f16_bits(s));
      if (zeros) zeros[i] = (uint8_t)z;
    }
  }
}

static int w4_check_shape(const char* who, int V, int H, int group) {
  if (V <= 0 || H <= 0) {
    set_error("%s requires non-empty dimensions (hidden=%d vocab=%d)", who, H, V);
    return NVJSEL_EINVAL;
  }
  if (group != 32 && group != 64 && group != 128) {
    set_error("%s: group must be 32, 64 or 128 (got %d)", who, group);
    return NVJSEL_EINVAL;
  }
  if (H % group) {
    set_error("%s: hidden %d is not a multiple of the group %d", who, H, group);
    return NVJSEL_EINVAL;
  }
  if (V > 0x7FFFFFFF - 4096 || H > (1 << 20)) {
    set_error("%s: vocab or hidden too large", who);
    return NVJSEL_EINVAL;
  }
  return NVJSEL_OK;
}

static int w4_entry(int mode, const void* hidden, int hidden_dtype, const void* packed, size_t packed_bytes,
                    int scale_dtype, int has_zeros, int group, int batch, int H, int V, int reduce_cast,
                    int32_t* out_ids, float* out_best, void* workspace, size_t ws_bytes, void* out_logits,
                    int out_dtype, int64_t out_stride, void* stream) {
  clear_error();
  const char* who = mode == MODE_GREEDY ? "lm_head_w4_top1" : "lm_head_w4_logits";
  if (!hidden || !packed || (mode == MODE_GREEDY ? (const void*)out_ids : out_logits) == nullptr) {
    set_error("%s: null hidden/weight/output", who);
    return NVJSEL_EINVAL;
  }
  if (batch <= 0) { set_error("%s requires non-empty dimensions (batch=%d)", who, batch); return NVJSEL_EINVAL; }
  const int rc = w4_check_shape(who, V, H, group);
  if (rc != NVJSEL_OK) return rc;
  if (!valid_dtype(hidden_dtype)) { set_error("%s: unsupported hidden dtype %d", who, hidden_dtype); return NVJSEL_EINVAL; }
  if (scale_dtype != NVJSEL_BF16 && scale_dtype != NVJSEL_F16) {
    set_error("%s: scales must be bf16 or f16", who);
    return NVJSEL_EINVAL;
  }
  if (reduce_cast < 0 || reduce_cast > 2) { set_error("%s: reduce_cast must be 0, 1 or 2", who); return NVJSEL_EINVAL; }
  const W4Layout lay = w4_layout(V, H, group, has_zeros != 0);
  if (((uintptr_t)packed & 15) || packed_bytes < lay.total) {
    set_error("%s: packed weight of %zu bytes (16-byte aligned) where %zu are needed", who, packed_bytes, lay.total);
    return NVJSEL_EINVAL;
  }
  if (mode == MODE_GREEDY) {
    const size_t need = nvjsel_lm_head_workspace_size(batch);
    if (!workspace || ws_bytes < need) {
      set_error("%s: workspace %zu bytes < required %zu", who, ws_bytes, need);
      return NVJSEL_EWORKSPACE;
    }
  } else {
    if (!valid_dtype(out_dtype)) { set_error("%s: out dtype must be f32, bf16 or f16", who); return NVJSEL_EINVAL; }
    if (out_stride < V) { set_error("%s: out row stride < vocab", who); return NVJSEL_EINVAL; }
  }
  W4Args a{};
  a.packed = (const uint8_t*)packed;
  a.hidden_dtype = hidden_dtype;
  a.scale_dtype = scale_dtype;
  a.zeros = has_zeros != 0;
  a.V = V;
  a.H = H;
  a.reduce_cast = reduce_cast;
  a.out_dtype = out_dtype;
  a.out_stride = out_stride;
  a.counter = mode == MODE_GREEDY ? (unsigned int*)((char*)workspace + align_up((size_t)batch * 8, 256)) : nullptr;
  std::unique_lock<std::mutex> lock(launch_mutex(), std::defer_lock);
  if (mode == MODE_GREEDY) lock.lock();  // logits take no workspace
  const int most = kW4Rows;
  for (int b0 = 0; b0 < batch; b0 += most) {
    a.B = batch - b0 < most ? batch - b0 : most;
    a.hidden = (const char*)hidden + (size_t)b0 * H * dtype_size(hidden_dtype);
    if (mode == MODE_GREEDY) {
      a.row_keys = (unsigned long long*)workspace + b0;
      a.out_ids = out_ids + b0;
      a.out_best = out_best ? out_best + b0 : nullptr;
    } else {
      a.out_logits = (char*)out_logits + (size_t)b0 * (size_t)out_stride * dtype_size(out_dtype);
    }
    const auto pass = mode == MODE_GREEDY ? (hidden_dtype == DT_F32    ? w4_greedy_f32
                                             : hidden_dtype == DT_BF16 ? w4_greedy_bf16
                                                                       : w4_greedy_f16)
                                          : (hidden_dtype == DT_F32    ? w4_logits_f32
                                             : hidden_dtype == DT_BF16 ? w4_logits_bf16
                                                                       : w4_logits_f16);
    const int e = pass(a, group, (hipStream_t)stream);
    if (e != NVJSEL_OK) return e;
  }
  return NVJSEL_OK;
}

}  // namespace nvjsel

using namespace nvjsel;

extern "C" size_t nvjsel_w4_packed_size(int vocab, int hidden_dim, int group, int has_zeros) {
  if (vocab <= 0 || hidden_dim <= 0 || (group != 32 && group != 64 && group != 128) || hidden_dim % group) return 0;
  return w4_layout(vocab, hidden_dim, group, has_zeros != 0).total;
}

extern "C" int nvjsel_w4_pack(const void* qweight, const void* scales, const void* zeros, int vocab, int hidden_dim,
                              int group, void* packed, size_t packed_bytes, void* stream) {
  clear_error();
  if (!qweight || !scales || !packed) return fail(NVJSEL_EINVAL, "w4_pack: null pointer");
  const int rc = w4_check_shape("w4_pack", vocab, hidden_dim, group);
  if (rc != NVJSEL_OK) return rc;
  const W4Layout lay = w4_layout(vocab, hidden_dim, group, zeros != nullptr);
  if (((uintptr_t)packed & 15) || packed_bytes < lay.total) {
    set_error("w4_pack: packed weight of %zu bytes (16-byte aligned) where %zu are needed", packed_bytes, lay.total);
    return NVJSEL_EINVAL;
  }
  const size_t blocks = (size_t)lay.tiles * lay.kblocks, most = (size_t)device_cu_count() * 32;
  hipLaunchKernelGGL(w4_pack_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, (hipStream_t)stream,
                     (const uint8_t*)qweight, (const uint16_t*)scales, (const uint8_t*)zeros, vocab, hidden_dim, group,
                     (uint8_t*)packed);
  NVJSEL_CHECK_LAUNCH("w4_pack_kernel");
  return NVJSEL_OK;
}

extern "C" int nvjsel_w4_quantize(const void* weight, int weight_dtype, int64_t row_stride, int64_t col_stride, int vocab,
                                  int hidden_dim, int group, int scale_dtype, void* qweight, void* scales, void* zeros,
                                  void* stream) {
  clear_error();
  if (!weight || !qweight || !scales) return fail(NVJSEL_EINVAL, "w4_quantize: null pointer");
  const int rc = w4_check_shape("w4_quantize", vocab, hidden_dim, group);
  if (rc != NVJSEL_OK) return rc;
  if (!valid_dtype(weight_dtype)) return fail(NVJSEL_EINVAL, "w4_quantize: unsupported weight dtype");
  if (scale_dtype != NVJSEL_BF16 && scale_dtype != NVJSEL_F16)
    return fail(NVJSEL_EINVAL, "w4_quantize: scales must be bf16 or f16");
  if (row_stride < 1 || col_stride < 1) return fail(NVJSEL_EINVAL, "w4_quantize: strides must be positive");
  const size_t items = ((size_t)vocab * (hidden_dim / group) + 3) / 4, most = (size_t)device_cu_count() * 32;
  hipLaunchKernelGGL(w4_quantize_kernel, dim3((unsigned)(items < most ? items : most)), dim3(256), 0,
                     (hipStream_t)stream, weight, weight_dtype, row_stride, col_stride, vocab, hidden_dim, group,
                     scale_dtype, (uint8_t*)qweight, (uint16_t*)scales, (uint8_t*)zeros);
  NVJSEL_CHECK_LAUNCH("w4_quantize_kernel");
  return NVJSEL_OK;
}

extern "C" int nvjsel_lm_head_w4_top1(const void* hidden, int hidden_dtype, const void* packed, size_t packed_bytes,
                                      int scale_dtype, int has_zeros, int group, int batch, int hidden_dim, int vocab,
                                      int reduce_cast, int32_t* out_ids, float* out_best, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  return w4_entry(MODE_GREEDY, hidden, hidden_dtype, packed, packed_bytes, scale_dtype, has_zeros, group, batch,
                  hidden_dim, vocab, reduce_cast, out_ids, out_best, workspace, workspace_bytes, nullptr, DT_F32, 0,
                  stream);
}

extern "C" int nvjsel_lm_head_w4_logits(const void* hidden, int hidden_dtype, const void* packed, size_t packed_bytes,
                                        int scale_dtype, int has_zeros, int group, int batch, int hidden_dim, int vocab,
                                        int reduce_cast, void* out_logits, int out_dtype, int64_t out_row_stride,
                                        void* stream) {
  return w4_entry(MODE_LOGITS, hidden, hidden_dtype, packed, packed_bytes, scale_dtype, has_zeros, group, batch,
                  hidden_dim, vocab, reduce_cast, nullptr, nullptr, nullptr, 0, out_logits, out_dtype, out_row_stride,
                  stream);
}
