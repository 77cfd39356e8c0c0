// The staged GEMM of lm_head_ring.h: greedy, logits and sampling.
#include "lm_head_ring.h"

namespace nvjsel {

template <int WT, int MODE, int NBR, int NS>
static int launch_ring_rows(const LmArgs& a, hipStream_t stream) {
  using S = RingShape<MODE, NBR, NS>;
  const int rows = ring_share(a.V, device_cu_count());  // every block reads the same share of W, contiguous
  hipLaunchKernelGGL((lm_head_ring_kernel<WT, MODE, NBR, NS>), dim3((a.V + rows - 1) / rows), dim3(S::NW * 64), 0, stream,
                     a, rows, ScoreArgs{});
  NVJSEL_CHECK_LAUNCH("lm_head_ring_kernel");
  return NVJSEL_OK;
}

template <int WT, int MODE>
static int launch_ring_mode(const LmArgs& a, hipStream_t stream) {
  if (a.B <= 32) return launch_ring_rows<WT, MODE, 32, 1>(a, stream);
  if (a.B <= 64) return launch_ring_rows<WT, MODE, 64, 1>(a, stream);
  if (a.B <= 128) return launch_ring_rows<WT, MODE, 128, 1>(a, stream);
  if constexpr (MODE != MODE_SAMPLE) return launch_ring_rows<WT, MODE, 256, 1>(a, stream);
  return fail(NVJSEL_EINVAL, "launch_ring: at most 128 sampled rows per pass");
}

template <int MODE>
static int launch_ring_f32(const LmArgs& a, hipStream_t stream) {
  if (a.B <= 32) return launch_ring_rows<DT_BF16, MODE, 32, 3>(a, stream);
  if (a.B <= 64) return launch_ring_rows<DT_BF16, MODE, 64, 3>(a, stream);
  return fail(NVJSEL_EINVAL, "launch_ring: at most 64 rows of f32 activations per pass");
}

int launch_ring(int mode, const LmArgs& a, hipStream_t stream) {
  auto by_mode = [&](auto fn) -> int {
    if (mode == MODE_GREEDY) return fn(std::integral_constant<int, MODE_GREEDY>{});
    if (mode == MODE_SAMPLE) return fn(std::integral_constant<int, MODE_SAMPLE>{});
    return fn(std::integral_constant<int, MODE_LOGITS>{});
  };
  if (a.hidden_dtype == DT_F32) return by_mode([&](auto M) { return launch_ring_f32<decltype(M)::value>(a, stream); });
  if (a.weight_dtype == DT_F16) return by_mode([&](auto M) { return launch_ring_mode<DT_F16, decltype(M)::value>(a, stream); });
  return by_mode([&](auto M) { return launch_ring_mode<DT_BF16, decltype(M)::value>(a, stream); });
}

}  // namespace nvjsel
