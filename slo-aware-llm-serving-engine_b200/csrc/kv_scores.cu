// Accumulated attention weights of cached keys, the second half of the scored decode:
//
//   scores[row, h, t] = decay * scores[row, h, t] + sum_{g in group h} 2^(x[g, t] - lse[g])
//
// x and lse are the log2-domain scores and denominators that the decode kernels store
// (4 G bytes a token and head against the K and V rows' 144 to 512, so that K is not
// read a second time).  One thread takes four tokens of one head and adds its group
// in order: no atomics, the same sum on every run.  The bf16 / f16 decode stores a row of
// tokens per head, the 4-bit decode the heads of a token side by side (what their
// accumulators make contiguous); both are read here.  The kernel may start before those
// that store them have ended, so what they store is loaded through L2 (__ldcg) and not
// through the read-only path.  They are stored to stay in L2 and loaded to leave it (447
// -> 439 us for the scored decode below).  Bound by the latency of its loads, largely
// from L2: 21 us for 256 x 8 heads of 512-4,096 tokens (G 4, 113 MB).
#include "common.cuh"

namespace slokv {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 4;  // tokens of a thread

struct ScoreParams {
  float *scores;
  int64_t row_stride, head_stride;
  int32_t width, num_rows;
  const int32_t *rows;
  const float *logits;
  int64_t logits_stride;
  const float *lse;
  const int32_t *lens;
  int32_t hkv, group, cap;
  float decay;
  uint32_t *err;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The scores' last use: their lines may go first.
__device__ __forceinline__ float4 load_last4(const float *p, uint64_t policy) {
  float4 v;
  asm volatile("ld.global.cg.L2::cache_hint.v4.f32 {%0, %1, %2, %3}, [%4], %5;"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "l"(p), "l"(policy));
  return v;
}
__device__ __forceinline__ float2 load_last2(const float *p, uint64_t policy) {
  float2 v;
  asm volatile("ld.global.cg.L2::cache_hint.v2.f32 {%0, %1}, [%2], %3;"
               : "=f"(v.x), "=f"(v.y)
               : "l"(p), "l"(policy));
  return v;
}

// kPairs: logits are [batch, hkv, logits_stride, group padded to even]; else [batch, hq,
// logits_stride], and kVec: score and logit rows allow 16-byte accesses.
template <bool kPairs, bool kVec>
__global__ void __launch_bounds__(kThreads) kv_scores_accumulate_kernel(const ScoreParams p) {
  const int32_t b = blockIdx.z, h = blockIdx.y;
  wait_prerequisites();
  int32_t len = __ldg(p.lens + b);
  const int32_t row = p.rows ? __ldg(p.rows + b) : b;
  const bool first = blockIdx.x == 0 && h == 0 && threadIdx.x == 0;
  if (row < 0 || row >= p.num_rows) {
    if (first && row != -1) record_error(p.err, SLOKV_DEVERR_SLOT_RANGE);
    return;
  }
  if (len > p.cap) {
    if (first) record_error(p.err, SLOKV_DEVERR_CONTEXT_LEN);
    len = p.cap;
  }
  const int64_t pair = static_cast<int64_t>(b) * p.hkv + h;
  const float *lse = p.lse + pair * p.group;
  float *score = p.scores + row * p.row_stride + h * p.head_stride;
  const uint64_t last = l2_evict_first_policy();
  if constexpr (kPairs) {
    // a warp's lanes take neighbouring tokens, whose heads lie side by side
    const int32_t heads = (p.group + 1) / 2 * 2;
    const int32_t t0 = blockIdx.x * kThreads * kPer + threadIdx.x;
    if (t0 >= len) return;
    const float *lg = p.logits + (pair * p.logits_stride + t0) * heads;
    const int64_t step = static_cast<int64_t>(kThreads) * heads;
    float w[kPer] = {0.f, 0.f, 0.f, 0.f}, before[kPer] = {0.f, 0.f, 0.f, 0.f};
    if (p.decay != 0.f) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (t0 + i * kThreads < len) before[i] = score[t0 + i * kThreads];
    }
#pragma unroll 2
    for (int g = 0; g < p.group; g += 2) {
      // a head whose every score is -inf has no weights; nor has the padding
      const float d0 = __ldcg(lse + g), d1 = g + 1 < p.group ? __ldcg(lse + g + 1) : -INFINITY;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (t0 + i * kThreads < len) {
          const float2 x = load_last2(lg + i * step + g, last);
          if (d0 != -INFINITY) w[i] += exp2_fast(x.x - d0);
          if (d1 != -INFINITY) w[i] += exp2_fast(x.y - d1);
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (t0 + i * kThreads < len) score[t0 + i * kThreads] = fmaf(p.decay, before[i], w[i]);
    return;
  } else {
    const int32_t t = (blockIdx.x * kThreads + threadIdx.x) * kPer;
    if (t >= len) return;
    const int32_t n = min(kPer, len - t);
    float w[kPer] = {0.f, 0.f, 0.f, 0.f};
    const float *lg = p.logits + pair * p.group * p.logits_stride + t;
    float4 before = make_float4(0.f, 0.f, 0.f, 0.f);
    if (kVec && n == kPer && p.decay != 0.f) before = *reinterpret_cast<const float4 *>(score + t);
#pragma unroll 4
    for (int g = 0; g < p.group; ++g, lg += p.logits_stride) {
      const float d = __ldcg(lse + g);
      if (d == -INFINITY) continue;
      float x[kPer];
      if (kVec && n == kPer) {
        const float4 v = load_last4(lg, last);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = i < n ? __ldcg(lg + i) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kPer; ++i) w[i] += exp2_fast(x[i] - d);
    }
    float *s = score + t;
    if (kVec && n == kPer) {
      *reinterpret_cast<float4 *>(s) =
          make_float4(fmaf(p.decay, before.x, w[0]), fmaf(p.decay, before.y, w[1]),
                      fmaf(p.decay, before.z, w[2]), fmaf(p.decay, before.w, w[3]));
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i < n) s[i] = p.decay != 0.f ? fmaf(p.decay, s[i], w[i]) : w[i];
    }
  }
}

}  // namespace
}  // namespace slokv

extern "C" int slokv_kv_scores_accumulate(float *scores, int64_t row_stride, int64_t head_stride,
                                          int32_t width, int32_t num_score_rows,
                                          const int32_t *score_rows, const float *logits,
                                          int64_t logits_stride, int32_t logits_pairs,
                                          const float *lse, const int32_t *context_lens, int32_t batch,
                                          int32_t num_q_heads, int32_t num_kv_heads,
                                          int64_t max_context, float decay, uint32_t *dev_error,
                                          void *stream) {
  using namespace slokv;
  if (batch < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
      width < 0 || num_score_rows < 0 || max_context < 0)
    return SLOKV_ERR_INVALID_ARG;
  if (batch == 0 || width == 0) return SLOKV_OK;
  if (!scores || !logits || !lse || !context_lens || logits_stride <= 0)
    return SLOKV_ERR_INVALID_ARG;
  if (batch > 65535 || num_kv_heads > 65535) return SLOKV_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(logits)) & 3u)
    return SLOKV_ERR_ALIGNMENT;
  ScoreParams p;
  p.scores = scores;
  p.row_stride = row_stride;
  p.head_stride = head_stride;
  p.width = width;
  p.num_rows = num_score_rows;
  p.rows = score_rows;
  p.logits = logits;
  p.logits_stride = logits_stride;
  p.lse = lse;
  p.lens = context_lens;
  p.hkv = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  int64_t cap = width < logits_stride ? width : logits_stride;
  if (max_context < cap) cap = max_context;
  p.cap = static_cast<int32_t>(cap);
  p.decay = decay;
  p.err = dev_error;
  if (cap == 0) return SLOKV_OK;
  if (cap > (1 << 30)) return SLOKV_ERR_UNSUPPORTED;  // a position plus a CTA's span fits 32 bits
  const bool vec = !((reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(logits)) & 15u) &&
                   !((row_stride | head_stride | logits_stride) & 3);
  const dim3 grid(static_cast<unsigned>((cap + kThreads * kPer - 1) / (kThreads * kPer)),
                  static_cast<unsigned>(num_kv_heads), static_cast<unsigned>(batch));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (logits_pairs && (reinterpret_cast<uintptr_t>(logits) & 7u)) return SLOKV_ERR_ALIGNMENT;
  auto *kernel = logits_pairs ? kv_scores_accumulate_kernel<true, false>
                 : vec        ? kv_scores_accumulate_kernel<false, true>
                              : kv_scores_accumulate_kernel<false, false>;
  return launch_dependent(kernel, grid, dim3(kThreads), 0, st, p) == cudaSuccess ? SLOKV_OK
                                                                                : SLOKV_ERR_CUDA;
}
