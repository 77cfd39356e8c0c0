// Beam search's selection over beams and vocabulary (beam_select.h), and the
// reordering of the beams' states that follows it.
#include "beam_select.h"

namespace nvjsel {

static size_t beam_bytes(int batch, int beams, int shares, int cap) {
  return kBeamRequests * 4 + (size_t)batch * beams * shares * (sizeof(BeamPart) + cap * sizeof(uint2));
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
  typedef typename std::conditional<VEC == 16, row_u32x4, uint32_t>::type Vec;
  typedef typename std::conditional<VEC == 16, row_u32x4_any, row_u32_any>::type Any;
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
  beam_split(batch * beams, kBeamLists / beams, vocab, k, dtype, &shares, &share, &cap, &group);
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
  beam_split(batch * beams, kBeamLists / beams, vocab, k, dtype, &a.shares, &a.share, &a.cap, &a.group);
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
  std::lock_guard<std::mutex> lock(launch_mutex());
  if (dtype == DT_F32) return launch_beam<DT_F32, LP_NONE>(a, s);
  if (dtype == DT_BF16) return launch_beam<DT_BF16, LP_NONE>(a, s);
  return launch_beam<DT_F16, LP_NONE>(a, s);
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
