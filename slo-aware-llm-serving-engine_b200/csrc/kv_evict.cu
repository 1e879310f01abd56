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
// L2), a radix select of at most 4 x 8 bits finds the key of the last token that stays, and
// warp votes turn the row into 32-token words (each warp owns a contiguous piece), from
// which ties, holes and moved tokens are ranked.  It writes the move list and compacts
// the score row.  Bound by its barriers and votes, not by its 9 MB: 27 us for 1,024 pairs of
// 512-4,096 tokens.  Long rows are bound by their one CTA: eight pairs of 98,000 tokens take
// 207 us with their moves (0.5 us of score bytes).
//
// kv_evict_move_kernel then copies the rows, spread over the whole GPU: a warp looks up
// eight moves and loads their K and V rows before it stores any.  HBM-bound: 90 us at
// 5.6 TB/s of scattered 256-byte rows for the same pairs cut to 1,024 tokens (136 us with
// one move at a time).
#include "common.cuh"
#include "int4_page.cuh"

namespace slokv {
namespace {

using namespace kv4;

constexpr int kSmemKeys = 8192;     // 32 KiB
constexpr int kCopies = 4;          // histogram copies, so that equal keys collide less
constexpr int kMoveThreads = 256;
constexpr int kMovesPerWarp = 8;
constexpr int kMovesPerCta = kMoveThreads / 32 * kMovesPerWarp;

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

template <int kThreads>
__global__ void __launch_bounds__(kThreads) kv_evict_select_kernel(const EvictParams p) {
  constexpr int kWarps = kThreads / 32;
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t hist[kCopies][256];
  __shared__ uint32_t sh_prefix, sh_left, sh_done;
  __shared__ uint32_t piece[3][kWarps];   // ties, holes, moved tokens of each warp's piece
  launch_dependents();  // the move kernel
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
  if (index)   // unsigned: keep may be 2^31 - 1, and a signed i would wrap below it
    for (uint32_t i = tid; i < static_cast<uint32_t>(p.keep); i += kThreads)
      index[i] = static_cast<int32_t>(i) < n ? static_cast<int32_t>(i) : -1;
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
  bool done = need == 0;                        // every key that shares the prefix stays
  for (int shift = 24; !done && shift >= 0; shift -= 8) {
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
        sh_done = rest == bin[i];
      }
    }
    __syncthreads();
    prefix = sh_prefix;
    left = sh_left;
    done = sh_done;
  }
  __syncthreads();                              // the keys are in place (need == 0: no pass ran)

  // ---- ordered ranks, 32 tokens to a word; warp w owns the words [lo, hi) ----
  // A key of at least `least` stays, and of the holders of the key `prefix` the first `left`.
  const uint32_t least = need == 0 ? 0xffffffffu : done ? prefix : prefix + 1;
  const bool ties_exist = !done;
  const int32_t words = (n + 31) / 32, per = (words + kWarps - 1) / kWarps;
  const int32_t lo = min(words, warp * per), hi = min(words, lo + per);
  const uint32_t below = (1u << lane) - 1u;
  // Lane i gets what the tokens of word w0 + i are: certain to stay, or ties.
  uint32_t sure = 0, tie = 0;
  auto classify = [&](int32_t w0) {
    sure = tie = 0;
    const int32_t stop = min(32, hi - w0);
    for (int32_t i = 0; i < stop; ++i) {
      const int32_t t = (w0 + i) * 32 + lane;
      const uint32_t k = t < old ? key(t) : 0u;
      const uint32_t a = __ballot_sync(0xffffffffu, t < n && (t >= old || k >= least));
      const uint32_t b = __ballot_sync(0xffffffffu, ties_exist && t < old && k == prefix);
      if (lane == i) {
        sure = a;
        tie = b;
      }
    }
  };
  auto inclusive = [&](uint32_t v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += x;
    }
    return v;
  };
  // Holes and moved tokens of lane i's word, given the ties before the group of words.
  uint32_t hole = 0, mover = 0;
  auto place = [&](int32_t w0, uint32_t &tie_base) {
    const uint32_t upto = inclusive(__popc(tie));
    const uint32_t before = tie_base + upto - __popc(tie);
    uint32_t some = tie;
    const uint32_t room = before < left ? left - before : 0u;
    if (room == 0) some = 0;
    while (__popc(some) > room) some &= ~(0x80000000u >> __clz(some));  // one word at most
    tie_base += __shfl_sync(0xffffffffu, upto, 31);
    const int32_t t0 = (w0 + lane) * 32;
    auto mask_below = [&](int32_t limit) {
      return limit >= t0 + 32 ? 0xffffffffu : limit <= t0 ? 0u : (1u << (limit - t0)) - 1u;
    };
    const bool mine = w0 + lane < hi;
    const uint32_t stays = sure | some, under = mask_below(p.keep);
    hole = mine ? ~stays & mask_below(n) & under : 0u;
    mover = mine ? stays & ~under : 0u;
  };
  const bool single = per <= 32;                // one group of words: classified once
  uint32_t ties = 0;
  for (int32_t w0 = lo; w0 < hi; w0 += 32) {
    classify(w0);
    ties += __shfl_sync(0xffffffffu, inclusive(__popc(tie)), 31);
  }
  if (lane == 0) piece[0][warp] = ties;
  __syncthreads();
  uint32_t tie_base = 0;
  for (int w = 0; w < warp; ++w) tie_base += piece[0][w];
  uint32_t base = tie_base, holes = 0, moved = 0;
  for (int32_t w0 = lo; w0 < hi; w0 += 32) {
    if (!single) classify(w0);
    place(w0, base);
    holes += __popc(hole);
    moved += __popc(mover);
  }
  holes = __reduce_add_sync(0xffffffffu, holes);
  moved = __reduce_add_sync(0xffffffffu, moved);
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
  for (int32_t w0 = lo; w0 < hi; w0 += 32) {
    if (!single) {
      classify(w0);
      place(w0, base);
    }
    const int32_t stop = min(32, hi - w0);
    for (int32_t i = 0; i < stop; ++i) {
      const uint32_t hv = __shfl_sync(0xffffffffu, hole, i), mv = __shfl_sync(0xffffffffu, mover, i);
      const int32_t t = (w0 + i) * 32 + lane;
      if ((hv >> lane) & 1u) dst[hole_at + __popc(hv & below)] = t;
      if ((mv >> lane) & 1u) src[move_at + __popc(mv & below)] = t;
      hole_at += __popc(hv);
      move_at += __popc(mv);
    }
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
  wait_prerequisites();
  // (the selection's output: through L2, since this kernel may have started before it)
  const int32_t count = __ldcg(p.counts + pair);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t *dst = p.moves + static_cast<int64_t>(pair) * 2 * p.max_moves;
  const int32_t *src = dst + p.max_moves;
  const int32_t *table = p.tables + static_cast<int64_t>(b) * p.bt_stride;
  // lanes 0 .. 7 look up the warp's moves, then all their rows are loaded before any is stored
  const int32_t first = blockIdx.y * kMovesPerCta + warp * kMovesPerWarp;
  if (first >= count) return;
  int32_t tb = -1, fb = 0, to_off = 0, from_off = 0;
  if (lane < kMovesPerWarp && first + lane < count) {
    const int32_t to = __ldcg(dst + first + lane), from = __ldcg(src + first + lane);
    const int32_t to_page = to / p.block_size, from_page = from / p.block_size;
    tb = __ldg(table + to_page);
    fb = __ldg(table + from_page);
    to_off = to - to_page * p.block_size;
    from_off = from - from_page * p.block_size;
    if (tb < 0 || tb >= p.num_blocks || fb < 0 || fb >= p.num_blocks) {
      record_error(p.err, SLOKV_DEVERR_BLOCK_RANGE);
      tb = -1;
    }
  }
  if (p.row_bytes) {
    const int64_t head = static_cast<int64_t>(h) * p.row_bytes;
    const int64_t token = static_cast<int64_t>(p.hkv) * p.row_bytes;
    const int half = p.row_bytes / 16;          // 16-byte pieces of a row; K's first, then V's
    for (int c = lane; c < 2 * half; c += 32) {  // 16 or 32 pieces a side: all lanes alike
      uint8_t *cache = c >= half ? p.v_cache : p.k_cache;
      const int64_t bs = c >= half ? p.v_bs : p.k_bs;
      const int64_t at = head + (c >= half ? c - half : c) * 16;
      uint4 w[kMovesPerWarp];
#pragma unroll
      for (int i = 0; i < kMovesPerWarp; ++i) {
        const int32_t t = __shfl_sync(0xffffffffu, tb, i), f = __shfl_sync(0xffffffffu, fb, i);
        const int32_t fo = __shfl_sync(0xffffffffu, from_off, i);
        if (t >= 0) w[i] = *reinterpret_cast<const uint4 *>(cache + f * bs + fo * token + at);
      }
#pragma unroll
      for (int i = 0; i < kMovesPerWarp; ++i) {
        const int32_t t = __shfl_sync(0xffffffffu, tb, i), o = __shfl_sync(0xffffffffu, to_off, i);
        if (t >= 0) *reinterpret_cast<uint4 *>(cache + t * bs + o * token + at) = w[i];
      }
    }
  } else {
    // a 4-bit row is 9 pieces of 8 bytes a side: the lanes take (move, piece) pairs
    const int64_t head = static_cast<int64_t>(h) * p.block_size * kRowBytes;
    constexpr int kPieces = 18, kSteps = (kMovesPerWarp * kPieces + 31) / 32;
    uint2 w[kSteps];
#pragma unroll
    for (int pass = 0; pass < 2; ++pass)
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int item = lane + 32 * k, i = item / kPieces, c = item % kPieces;
        const int32_t t = __shfl_sync(0xffffffffu, tb, i & 7), f = __shfl_sync(0xffffffffu, fb, i & 7);
        const int32_t to = __shfl_sync(0xffffffffu, to_off, i & 7);
        const int32_t fo = __shfl_sync(0xffffffffu, from_off, i & 7);
        if (i >= kMovesPerWarp || t < 0) continue;
        const bool v = c >= 9;
        const int q = v ? c - 9 : c;
        uint8_t *cache = (v ? p.v_cache : p.k_cache) + head;
        const int64_t bs = v ? p.v_bs : p.k_bs;
        const int32_t off = pass ? to : fo;
        uint2 *at = reinterpret_cast<uint2 *>(cache + (pass ? t : f) * bs +
                                              (q < 8 ? code_offset(off) + 8 * q : param_offset(off)));
        if (pass)
          *at = w[k];
        else
          w[k] = *at;
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
  if (pairs > 0x7fffffff || chunks > 65535 || cap > (1 << 30)) return SLOKV_ERR_UNSUPPORTED;
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
  // 256 threads: eight CTAs a multiprocessor hide each other's barriers (128 x 8 pairs of
  // 2304 tokens: 34 us against 42 with 512, before the ranks were taken from words, now
  // 27); rows that do not fit in shared memory, which few pairs have, take 1024.
  if (cap <= kSmemKeys)
    kv_evict_select_kernel<256><<<static_cast<unsigned>(pairs), 256, smem, st>>>(p);
  else
    kv_evict_select_kernel<1024><<<static_cast<unsigned>(pairs), 1024, smem, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return SLOKV_ERR_CUDA;
  if (most == 0) return SLOKV_OK;
  const dim3 grid(static_cast<unsigned>(pairs), static_cast<unsigned>(chunks));
  return launch_dependent(kv_evict_move_kernel, grid, dim3(kMoveThreads), 0, st, p) == cudaSuccess
             ? SLOKV_OK
             : SLOKV_ERR_CUDA;
}
