// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence b, kv head h) with n = context_lens[b] > keep tokens: the last `recent`
// stay, and of the others the keep - recent of the highest score (ties: the lowest
// position; NaN counts as -inf).  A kept token below position `keep` stays where it
// is; the kept tokens at or past `keep` fill the holes below it, both in order.  Every
// source lies at or past `keep` and every destination below it, so the moves are
// independent of each other, each moved row is read and written once, and nothing else
// is touched.  Keys carry their rotary position, so attention does not mind the order.
//
// kv_evict_select_kernel, one CTA per (b, h): the scores become unsigned keys of the
// same order (kept in shared memory up to kSmemKeys tokens, else read again through
// L2), a radix select over 4 x 8 bits finds the key of the last token that stays, and
// three ordered passes with warp votes (each warp owns a contiguous piece) rank ties,
// holes and moved tokens.  It writes the move list and compacts the score row.
// kv_evict_move_kernel then copies the rows, spread over the whole GPU.
#include "common.cuh"
#include "int4_page.cuh"

namespace slokv {
namespace {

using namespace kv4;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kSmemKeys = 8192;     // 32 KiB: four CTAs a multiprocessor
constexpr int kCopies = 8;          // histogram copies, so that equal keys collide less
constexpr int kMoveThreads = 256;
constexpr int kMovesPerCta = 64;

struct EvictParams {
  uint8_t *k_cache, *v_cache;
  int64_t k_bs, v_bs;               // block strides, bytes
  int32_t num_blocks, block_size, hkv;
  int32_t row_bytes;                // bytes of a (token, head) row; 0: a 4-bit pool
  const int32_t *tables;
  int64_t bt_stride;
  const int32_t *lens;
  float *scores;
  int64_t row_stride, head_stride;
  int32_t num_rows;
  const int32_t *rows;
  int32_t cap, keep, recent;
  int32_t *new_lens;
  int32_t *index;                   // [batch, hkv, keep] or null
  int32_t *counts;                  // [batch * hkv] moves of each pair
  int32_t *moves;                   // [batch * hkv][2][max_moves]: destinations, sources
  int32_t max_moves;
  uint32_t *err;
};

// A float as an unsigned key of the same order; -0 as +0, NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) f = -INFINITY;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kThreads) kv_evict_select_kernel(const EvictParams p) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t hist[kCopies][256];
  __shared__ uint32_t sh_prefix, sh_left;
  __shared__ uint32_t piece[3][kWarps];   // ties, holes, moved tokens of each warp's piece
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv;
  const int32_t n = __ldg(p.lens + b);
  const int32_t row = p.rows ? __ldg(p.rows + b) : b;
  const bool known = row >= 0 && row < p.num_rows;
  const bool fits = n <= p.cap;
  if (tid == 0 && h == 0) {
    if (!known && row != -1) record_error(p.err, SLOKV_DEVERR_SLOT_RANGE);
    if (!fits) record_error(p.err, SLOKV_DEVERR_CONTEXT_LEN);
    p.new_lens[b] = known && fits && n > p.keep ? p.keep : n;
  }
  int32_t *index = p.index ? p.index + static_cast<int64_t>(blockIdx.x) * p.keep : nullptr;
  if (index)
    for (int32_t i = tid; i < p.keep; i += kThreads) index[i] = i < n ? i : -1;
  if (!known || !fits || n <= p.keep) {
    if (tid == 0) p.counts[blockIdx.x] = 0;
    return;
  }
  float *score = p.scores + row * p.row_stride + h * p.head_stride;
  const int32_t old = n - p.recent;             // tokens that have to earn their place
  const uint32_t need = p.keep - p.recent;      // how many of them do (need < old)
  const bool in_smem = old <= kSmemKeys;
  if (in_smem)
    for (int32_t t = tid; t < old; t += kThreads) keys[t] = order_key(score[t]);
  auto key = [&](int32_t t) { return in_smem ? keys[t] : order_key(score[t]); };

  // ---- the need-th largest key: 8 bits a pass, most significant first ----
  uint32_t prefix = 0, left = need;             // left: places for keys that share the prefix
  for (int shift = 24; need && shift >= 0; shift -= 8) {
    for (int i = tid; i < kCopies * 256; i += kThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    for (int32_t t = tid; t < old; t += kThreads) {
      const uint32_t k = key(t);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[warp % kCopies][(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {
      // lane l owns bins 255 - 8 l .. 248 - 8 l, the highest first
      uint32_t bin[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bin[i] = 0;
        for (int q = 0; q < kCopies; ++q) bin[i] += hist[q][255 - 8 * lane - i];
        sum += bin[i];
      }
      uint32_t above = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, above, o);
        if (lane >= o) above += v;
      }
      above -= sum;
      if (above < left && left <= above + sum) {  // exactly one lane
        uint32_t rest = left - above;
        int i = 0;
        while (rest > bin[i]) rest -= bin[i++];
        sh_prefix = prefix | (static_cast<uint32_t>(255 - 8 * lane - i) << shift);
        sh_left = rest;
      }
    }
    __syncthreads();
    prefix = sh_prefix;
    left = sh_left;
  }
  __syncthreads();                              // the keys are in place (need == 0: no pass ran)

  // ---- ordered ranks: warp w owns tokens [lo, hi) ----
  const int32_t per = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int32_t lo = min(n, warp * per), hi = min(n, lo + per);
  const uint32_t below = (1u << lane) - 1u;
  uint32_t ties = 0;
  if (need)
    for (int32_t t0 = lo; t0 < hi; t0 += 32) {
      const int32_t t = t0 + lane;
      ties += __popc(__ballot_sync(0xffffffffu, t < min(hi, old) && key(t) == prefix));
    }
  if (lane == 0) piece[0][warp] = ties;
  __syncthreads();
  uint32_t tie_base = 0;
  for (int w = 0; w < warp; ++w) tie_base += piece[0][w];
  // kept[t]: recent, above the threshold key, or one of its first `left` holders
  auto kept_at = [&](int32_t t, uint32_t &base) {
    const bool in = t < hi, cand = in && t < old && need;
    const uint32_t k = cand ? key(t) : 0u;
    const bool tie = cand && k == prefix;
    const uint32_t votes = __ballot_sync(0xffffffffu, tie);
    const bool keep = in && (t >= old || (cand && k > prefix) ||
                             (tie && base + __popc(votes & below) < left));
    base += __popc(votes);
    return keep;
  };
  uint32_t base = tie_base, holes = 0, moved = 0;
  for (int32_t t0 = lo; t0 < hi; t0 += 32) {
    const int32_t t = t0 + lane;
    const bool k = kept_at(t, base);
    holes += __popc(__ballot_sync(0xffffffffu, t < hi && t < p.keep && !k));
    moved += __popc(__ballot_sync(0xffffffffu, t >= p.keep && k));
  }
  if (lane == 0) {
    piece[1][warp] = holes;
    piece[2][warp] = moved;
  }
  __syncthreads();
  uint32_t hole_at = 0, move_at = 0, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      hole_at += piece[1][w];
      move_at += piece[2][w];
    }
    total += piece[1][w];
  }
  int32_t *dst = p.moves + static_cast<int64_t>(blockIdx.x) * 2 * p.max_moves;
  int32_t *src = dst + p.max_moves;
  base = tie_base;
  for (int32_t t0 = lo; t0 < hi; t0 += 32) {
    const int32_t t = t0 + lane;
    const bool k = kept_at(t, base);
    const bool hole = t < hi && t < p.keep && !k, mover = t >= p.keep && k;
    const uint32_t hv = __ballot_sync(0xffffffffu, hole), mv = __ballot_sync(0xffffffffu, mover);
    if (hole) dst[hole_at + __popc(hv & below)] = t;
    if (mover) src[move_at + __popc(mv & below)] = t;
    hole_at += __popc(hv);
    move_at += __popc(mv);
  }
  if (tid == 0) p.counts[blockIdx.x] = static_cast<int32_t>(total);
  __syncthreads();
  for (uint32_t i = tid; i < total; i += kThreads) {
    const int32_t to = dst[i], from = src[i];
    score[to] = score[from];
    if (index) index[to] = from;
  }
  __syncthreads();
  for (int32_t t = p.keep + tid; t < n; t += kThreads) score[t] = 0.f;
}

__global__ void __launch_bounds__(kMoveThreads) kv_evict_move_kernel(const EvictParams p) {
  const int32_t pair = blockIdx.x, b = pair / p.hkv, h = pair % p.hkv;
  const int32_t count = __ldg(p.counts + pair);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t *dst = p.moves + static_cast<int64_t>(pair) * 2 * p.max_moves;
  const int32_t *src = dst + p.max_moves;
  const int32_t *table = p.tables + static_cast<int64_t>(b) * p.bt_stride;
  const int32_t stop = min(count, static_cast<int32_t>(blockIdx.y + 1) * kMovesPerCta);
  for (int32_t i = blockIdx.y * kMovesPerCta + warp; i < stop; i += kMoveThreads / 32) {
    const int32_t to = __ldg(dst + i), from = __ldg(src + i);
    const int32_t tb = __ldg(table + to / p.block_size), fb = __ldg(table + from / p.block_size);
    if (tb < 0 || tb >= p.num_blocks || fb < 0 || fb >= p.num_blocks) {
      if (lane == 0) record_error(p.err, SLOKV_DEVERR_BLOCK_RANGE);
      continue;
    }
    const int32_t to_off = to % p.block_size, from_off = from % p.block_size;
    if (p.row_bytes) {
      const int64_t head = static_cast<int64_t>(h) * p.row_bytes;
      const int64_t token = static_cast<int64_t>(p.hkv) * p.row_bytes;
      const int half = p.row_bytes / 16;        // 16-byte pieces of a row; K's first, then V's
      for (int c = lane; c < 2 * half; c += 32) {
        const bool v = c >= half;
        uint8_t *cache = v ? p.v_cache : p.k_cache;
        const int64_t bs = v ? p.v_bs : p.k_bs, at = head + (v ? c - half : c) * 16;
        const uint4 w = *reinterpret_cast<const uint4 *>(cache + fb * bs + from_off * token + at);
        *reinterpret_cast<uint4 *>(cache + tb * bs + to_off * token + at) = w;
      }
    } else if (lane < 10) {                     // 5 lanes a side: 4 x 16 B of codes, 8 B of parameters
      const bool v = lane >= 5;
      const int c = v ? lane - 5 : lane;
      uint8_t *cache = v ? p.v_cache : p.k_cache;
      const int64_t bs = v ? p.v_bs : p.k_bs;
      const int64_t head = static_cast<int64_t>(h) * p.block_size * kRowBytes;
      const uint8_t *f = cache + fb * bs + head;
      uint8_t *t = cache + tb * bs + head;
      if (c < 4)
        *reinterpret_cast<uint4 *>(t + code_offset(to_off) + 16 * c) =
            *reinterpret_cast<const uint4 *>(f + code_offset(from_off) + 16 * c);
      else
        *reinterpret_cast<uint2 *>(t + param_offset(to_off)) =
            *reinterpret_cast<const uint2 *>(f + param_offset(from_off));
    }
  }
}

// Most tokens of a pair that can move: they fill holes below keep from positions past it.
int64_t most_moves(int64_t keep, int64_t cap) {
  const int64_t past = cap - keep;
  return past <= 0 ? 0 : (past < keep ? past : keep);
}

size_t evict_workspace(int64_t pairs, int64_t keep, int64_t cap) {
  return static_cast<size_t>(pairs) * (1 + 2 * most_moves(keep, cap)) * sizeof(int32_t);
}

}  // namespace
}  // namespace slokv

extern "C" size_t slokv_kv_evict_workspace_bytes(int32_t batch, int32_t num_kv_heads, int32_t keep,
                                                 int32_t score_width) {
  if (batch <= 0 || num_kv_heads <= 0 || keep <= 0 || score_width < 0) return 0;
  return slokv::evict_workspace(static_cast<int64_t>(batch) * num_kv_heads, keep, score_width);
}

extern "C" int slokv_kv_evict(void *k_cache, void *v_cache, int64_t k_block_stride_bytes,
                              int64_t v_block_stride_bytes, int32_t num_blocks, int32_t block_size,
                              int32_t num_kv_heads, int32_t head_dim, int32_t cache_dtype,
                              const int32_t *block_tables, int64_t block_table_stride,
                              int32_t max_blocks_per_seq, const int32_t *context_lens,
                              int32_t batch, float *scores, int64_t score_row_stride,
                              int64_t score_head_stride, int32_t score_width,
                              int32_t num_score_rows, const int32_t *score_rows, int32_t keep,
                              int32_t recent, int32_t *new_lens, int32_t *index, void *workspace,
                              size_t workspace_bytes, uint32_t *dev_error, void *stream) {
  using namespace slokv;
  if (batch < 0 || num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || keep <= 0 ||
      recent < 0 || recent > keep || score_width < 0 || num_score_rows < 0)
    return SLOKV_ERR_INVALID_ARG;
  const bool q4 = cache_dtype == SLOKV_DTYPE_INT4;
  int elem = 0;
  if (cache_dtype == SLOKV_DTYPE_BF16 || cache_dtype == SLOKV_DTYPE_F16) elem = 2;
  if (cache_dtype == SLOKV_DTYPE_F32) elem = 4;
  if (head_dim != kHeadDim || (!q4 && !elem) || (q4 && block_size % kTileTokens))
    return SLOKV_ERR_UNSUPPORTED;
  if (batch == 0) return SLOKV_OK;
  if (!k_cache || !v_cache || !block_tables || !context_lens || !scores || !new_lens ||
      max_blocks_per_seq <= 0)
    return SLOKV_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15u) ||
      ((k_block_stride_bytes | v_block_stride_bytes) & 15) ||
      (reinterpret_cast<uintptr_t>(scores) & 3u))
    return SLOKV_ERR_ALIGNMENT;
  const int64_t pairs = static_cast<int64_t>(batch) * num_kv_heads;
  int64_t cap = static_cast<int64_t>(max_blocks_per_seq) * block_size;
  if (score_width < cap) cap = score_width;
  const int64_t most = most_moves(keep, cap);
  const int64_t chunks = (most + kMovesPerCta - 1) / kMovesPerCta;
  if (pairs > 0x7fffffff || chunks > 65535) return SLOKV_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < evict_workspace(pairs, keep, score_width))
    return SLOKV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 3u) return SLOKV_ERR_ALIGNMENT;

  EvictParams p;
  p.k_cache = static_cast<uint8_t *>(k_cache);
  p.v_cache = static_cast<uint8_t *>(v_cache);
  p.k_bs = k_block_stride_bytes;
  p.v_bs = v_block_stride_bytes;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.hkv = num_kv_heads;
  p.row_bytes = q4 ? 0 : kHeadDim * elem;
  p.tables = block_tables;
  p.bt_stride = block_table_stride;
  p.lens = context_lens;
  p.scores = scores;
  p.row_stride = score_row_stride;
  p.head_stride = score_head_stride;
  p.num_rows = num_score_rows;
  p.rows = score_rows;
  p.cap = static_cast<int32_t>(cap);
  p.keep = keep;
  p.recent = recent;
  p.new_lens = new_lens;
  p.index = index;
  p.max_moves = static_cast<int32_t>(most_moves(keep, score_width));
  p.counts = static_cast<int32_t *>(workspace);
  p.moves = p.counts + pairs;
  p.err = dev_error;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t smem = sizeof(uint32_t) * (cap < kSmemKeys ? cap : kSmemKeys);
  kv_evict_select_kernel<<<static_cast<unsigned>(pairs), kThreads, smem, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return SLOKV_ERR_CUDA;
  if (most == 0) return SLOKV_OK;
  const dim3 grid(static_cast<unsigned>(pairs), static_cast<unsigned>(chunks));
  kv_evict_move_kernel<<<grid, kMoveThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? SLOKV_OK : SLOKV_ERR_CUDA;
}
