// Paged GQA decode attention over the 4-bit pool (layout: int4_page.cuh).
//
//   K[t] = mK_g + sK_g c,  V[t] = mV_g + sV_g c     (g: 64-dim group, c: 4-bit code)
//   S[h, t] = scale * sum_g ( sK_tg (q . c)_g + mK_tg (sum_d q)_g )
//   out[h]  = sum_t p_t V[t] / sum_t p_t,  p_t = 2^(S log2(e) - running max)
//
// Bound by HBM in principle (144 bytes a token and head, 4 G 128 FMA) and by issue and ALU
// slots in fact: unpacking a code costs more than loading it.  So the codes go to the
// tensor cores as they are, scale and minimum are applied to the score tile and to the
// probabilities instead of to the 128 dims, and no code is ever rounded.
// Measured: 128 sequences of 1,024-8,192 tokens, 8 KV heads of 4, bf16: 118 us = 5.77 TB/s
// at 1,965 MHz (89 % of the copy rate), 136-140 us in a loop of seconds under the 1,000 W cap;
// 15 warp instructions a token and head (K and V), half of them ALU.
//
// QK^T (m16n8k16, f16, S^T = K q^T: A = K codes, 16 tokens; B = q, 8 heads).  A code in bits
// 0-3 of an f16 is the subnormal c 2^-24, in bits 4-7 it is 16 c 2^-24: two masks and one
// shift turn a word of 8 codes into four f16x2 operands, exactly.  q rows are brought to
// 2^14 <= max |q| < 2^15 by a power of two (the dims that meet the 16 c codes to a
// sixteenth of that), which the fp32 result undoes with the 2^24.  The minimum's term is
// one bf16 MMA for 16 tokens: the parameter words are its A operand as they lie in the
// page, q's group sums in three bf16 pieces its B.
//
// PV (m16n8k16, f16, out^T = V^T P^T: A = V codes, 16 dims; B = P^T, 8 heads).  Heads are
// the columns of both products, so no MMA row is wasted on a small group, and a lane's
// score and output columns are the same two heads.  movmatrix turns the score tile into the
// B operand; a prmt pairs the codes of two tokens.  Of the two codes in a byte the low one
// is masked out and the high one taken together with it (c0 + 16 c1, also linear in an
// f16's bits): sum r c1 = (sum r (c0 + 16 c1) - sum r c0) / 16 loses nothing, the division
// by 16 shrinking the larger sum's rounding as well, and saves a mask (116 -> 114 us).
//
// The probabilities carry the V scale, r = f16(p s_g):  out = sum_t r c + sum_t p m.  Half
// a step of r is 2^-11, an eighth of a bf16 output's (1.8e-3 off in all, 1.7e-3 of it the
// output's).  An f16 output rounds as finely as r does, so for those r is two f16 (the
// second takes what the first leaves) and the product runs twice: 2.1e-4 off, the output's
// own, instead of 5e-4 with one, at 137 us instead of 118.  f16
// has 5 exponent bits and the scales' range is fp32's: the reference that the scores are
// exponentiated against is not the running maximum but lies 15 - ceil(log2 max(s, |m|))
// below it, the maximum over the tokens seen so far.  r is then at most 2^15 and keeps
// its 11 bits down to 2^-29 of the largest value (or of 2^-60, if that is more); the sum
// of p is taken against the same reference, so the quotient does not see it.
//
// Work split: the 64-token tiles of all (sequence, kv head) segments, in that order, cut
// into equal contiguous ranges, one per warp slot; slot s is warp s / grid of CTA s % grid,
// so that a few tiles still use every SM.  A segment inside one range is finished in place,
// the others leave (reference, sum, acc) partials that the merge kernel combines.  Each
// warp owns a ring of 9,216-byte stages; lane 0 issues two bulk copies a tile (K and V
// tile are contiguous), with the next page's block id loaded a page ahead.  12 warps with two
// stages: 8 with three took 131 us instead of 122 then, 16 with K and V tiles apart (128
// registers, spills) 139 instead of 116.
#include "common.cuh"
#include "decode_worklist.cuh"
#include "int4_page.cuh"

#include <type_traits>

namespace slokv {
namespace decode4 {

using decode::fast_exp2;
using decode::kAccOff;
using decode::kD;
using decode::kMaxBatch;
using decode::kRowFloats;
using kv4::kParamOff;
using kv4::kRowBytes;
using kv4::kTileBytes;
using kv4::min_of;
using kv4::scale_of;

constexpr int kTile = kv4::kTileTokens;
constexpr int kStages = 2;
constexpr int kStage = 2 * kTileBytes;                    // K tile, V tile

constexpr int kFlush = 8;                                 // tiles between two moves out of o
constexpr int kSkip = 4;                                  // sequences per entry of the tile prefix

// Warps of a CTA by the query-head columns (kN x 8): twice the accumulators at kN = 2 need
// the larger register share of 8 warps, and spill a little even so (128 sequences of 1,024-8,192
// tokens, 721 MB, 16 heads a KV head: 212 us in bf16, 260 in f16; 8 heads: 137 in bf16).
constexpr int warps_of(int kN) { return kN == 1 ? 12 : 8; }
constexpr int ring_bytes(int warps) { return warps * kStages * kStage; }

struct Params {
  void *out;
  int64_t out_sb, out_sh;
  const void *q;
  int64_t q_sb, q_sh;
  const uint8_t *k_cache, *v_cache;
  int64_t k_bs, v_bs;                 // block strides, bytes
  const int32_t *block_tables;
  int64_t bt_stride;
  int32_t max_blocks;
  const int32_t *context_lens;
  int32_t batch;
  int32_t num_blocks, block_size, hkv, group;
  float scale_log2;
  float *partials;                    // [nslots][2][group][kRowFloats]
  int4 *jobs;                         // [nslots]: segment (b, h, first slot, last slot) of the warp
                                      // slot's head partial (x = -1: it has none)
  const int32_t *table_rows;          // table row of each sequence, or null: its own index
  float *logits;                      // scored: [batch, hkv, logits_stride, logits_heads] log2-
                                      // domain scores (logits_heads: the group, padded to even)
  float *lse;                         // scored: [batch, hq] log2 of the softmax denominator
  int32_t logits_stride, logits_heads;
  uint32_t *err;
  int32_t nslots;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes,
                                          uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1], %2, [%3], %4;" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}

// Shared-memory loads as plain C++, which the compiler may schedule between the waits.
__device__ __forceinline__ uint4 lds128(const uint8_t *p) {
  return *reinterpret_cast<const uint4 *>(p);
}
__device__ __forceinline__ uint2 lds64(const uint8_t *p) {
  return *reinterpret_cast<const uint2 *>(p);
}
__device__ __forceinline__ uint32_t lds32(const uint8_t *p) {
  return *reinterpret_cast<const uint32_t *>(p);
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}

// Without "volatile": the compiler may interleave independent MMAs.
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with a zero C.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void mma_bf16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// x in the high half as the bf16 nearest to it; x becomes what that leaves.
__device__ __forceinline__ uint32_t split_bf16(float &x) {
  const uint32_t hi = static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(x))) << 16;
  x -= __uint_as_float(hi);
  return hi;
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// ---- work list ----------------------------------------------------------------

// Cached tokens of sequence b, within the table's reach.
__device__ __forceinline__ int32_t seq_len(const Params &p, int32_t b) {
  const int32_t len = max(0, __ldg(p.context_lens + b));
  const int64_t cap = static_cast<int64_t>(p.max_blocks) * p.block_size;
  return len > cap ? static_cast<int32_t>(cap) : len;
}

__device__ __forceinline__ int32_t seq_tiles(const Params &p, int32_t b) {
  return (seq_len(p, b) + kTile - 1) / kTile;
}

// prefix[i] = tiles before sequence kSkip i, for i up to ceil(batch / kSkip); the last
// entry is the total.  Called by all threads of the CTA.
__device__ void build_prefix(const Params &p, int32_t *prefix) {
  __shared__ int32_t warp_sums[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int32_t n = (p.batch + kSkip - 1) / kSkip;
  int32_t carry = 0;
  for (int32_t i0 = 0; i0 < n; i0 += blockDim.x) {
    const int32_t i = i0 + tid;
    int32_t own = 0;
#pragma unroll
    for (int k = 0; k < kSkip; ++k) {
      const int32_t b = i * kSkip + k;
      if (i < n && b < p.batch) own += seq_tiles(p, b) * p.hkv;
    }
    int32_t v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t x = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += x;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    int32_t before = carry, all = carry;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) before += warp_sums[w];
      all += warp_sums[w];
    }
    if (i < n) prefix[i] = before + v - own;
    carry = all;
    __syncthreads();
  }
  if (tid == 0) prefix[n] = carry;
  __syncthreads();
}

struct TileRef {
  int32_t b, h, j, nt, seg_start;  // sequence, kv head, tile of the segment, its tiles, its first
};

// Locate global tile t.
__device__ __forceinline__ TileRef locate(const Params &p, const int32_t *prefix, int32_t t) {
  int32_t lo = 0, hi = (p.batch + kSkip - 1) / kSkip - 1;
  while (lo < hi) {
    const int32_t mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= t) lo = mid; else hi = mid - 1;
  }
  TileRef r;
  r.b = lo * kSkip;
  int32_t first = prefix[lo];
  r.nt = seq_tiles(p, r.b);
  while (first + r.nt * p.hkv <= t) {
    first += r.nt * p.hkv;
    r.nt = seq_tiles(p, ++r.b);
  }
  r.h = (t - first) / r.nt;
  r.j = t - first - r.h * r.nt;
  r.seg_start = first + r.h * r.nt;
  return r;
}

// Equal contiguous ranges of `total` tiles over min(total, nslots) slots.
struct Split {
  int32_t slots, chunk, rem;
  __device__ __forceinline__ Split(int32_t total, int32_t nslots) {
    slots = min(total, nslots);
    chunk = slots ? total / slots : 0;
    rem = total - chunk * slots;
  }
  __device__ __forceinline__ int32_t start(int32_t s) const { return s * chunk + min(s, rem); }
  __device__ __forceinline__ int32_t owner(int32_t t) const {
    const int32_t pivot = rem * (chunk + 1);
    return t < pivot ? t / (chunk + 1) : rem + (t - pivot) / chunk;
  }
};

// The next tile that a warp's producer lane issues, in work-list order.
struct Cursor {
  const uint8_t *k, *v;  // the tile; k null: its page lies outside the pool
  int32_t in_page;       // tiles left in the page, this one included
  int32_t b, h, page;    // sequence, kv head, page of the segment
  int32_t left;          // tiles left in the segment, this one included
  int32_t ahead;         // block id of the page that follows in the range
};

__device__ __forceinline__ int32_t table_entry(const Params &p, int32_t b, int32_t page) {
  if (p.table_rows) b = __ldg(p.table_rows + b);
  return __ldg(p.block_tables + static_cast<int64_t>(b) * p.bt_stride + page);
}

// The sequence after b that has tokens, whose first tile is tile t of the work list: the
// neighbour, or behind a gap, however long, the one that the prefix gives.  (140 sequences
// of 512 tokens padded to 256: 33 us when each warp walks the gap, 29.6 us so; three
// sequences of 8,192: 323 and 29 us.)
__device__ __forceinline__ int32_t next_seq(const Params &p, const int32_t *prefix, int32_t b,
                                            int32_t t) {
  return seq_len(p, b + 1) ? b + 1 : locate(p, prefix, t).b;
}

// Enter page c.page of segment (c.b, c.h), whose block id is `blk`, at its tile `first`,
// tile t of the work list, and load the id of the page after it if the range, which ends
// at `end`, reaches it: the segment's next, else the first page of the next segment.
__device__ __forceinline__ void cursor_page(Cursor &c, const Params &p, const int32_t *prefix,
                                            int32_t blk, int32_t first, int32_t t, int32_t end,
                                            int tiles_per_block) {
  c.k = c.v = nullptr;
  if (blk >= 0 && blk < p.num_blocks) {
    const int64_t at = static_cast<int64_t>(c.h) * p.block_size * kRowBytes +
                       static_cast<int64_t>(first) * kTileBytes;
    c.k = p.k_cache + blk * p.k_bs + at;
    c.v = p.v_cache + blk * p.v_bs + at;
  } else {
    record_error(p.err, SLOKV_DEVERR_BLOCK_RANGE);
  }
  c.in_page = min(tiles_per_block - first, c.left);
  if (t + c.in_page >= end) return;
  int32_t b = c.b, page = c.page + 1;
  if (c.in_page == c.left) {
    page = 0;
    if (c.h + 1 == p.hkv) b = next_seq(p, prefix, b, t + c.in_page);
  }
  c.ahead = table_entry(p, b, page);
}

__device__ __forceinline__ void cursor_init(Cursor &c, const Params &p, const int32_t *prefix,
                                            const TileRef &r, int32_t t, int32_t end,
                                            int tiles_per_block) {
  c.b = r.b;
  c.h = r.h;
  c.page = r.j / tiles_per_block;
  c.left = r.nt - r.j;
  cursor_page(c, p, prefix, table_entry(p, c.b, c.page), r.j - c.page * tiles_per_block, t, end,
              tiles_per_block);
}

// Step to the following tile, tile t of the work list; call only if it is in the range.
__device__ __forceinline__ void cursor_next(Cursor &c, const Params &p, const int32_t *prefix,
                                            int32_t t, int32_t end, int tiles_per_block) {
  --c.left;
  if (--c.in_page) {
    if (c.k) {
      c.k += kTileBytes;
      c.v += kTileBytes;
    }
    return;
  }
  ++c.page;
  if (!c.left) {
    c.page = 0;
    if (++c.h == p.hkv) {
      c.h = 0;
      c.b = next_seq(p, prefix, c.b, t);
    }
    c.left = seq_tiles(p, c.b);
  }
  cursor_page(c, p, prefix, c.ahead, 0, t, end, tiles_per_block);
}

// Issue the copies of the cursor's tile into `stage`.  A page outside the pool is not
// read: the stage completes empty and the return value is false.
__device__ __forceinline__ bool issue_tile(const Cursor &c, uint32_t ring, uint32_t bars, int stage,
                                           uint64_t policy) {
  const uint32_t bar = bars + stage * 8;
  if (!c.k) {
    mbar_arrive(bar);
    return false;
  }
  const uint32_t dst = ring + stage * kStage;
  fence_proxy_async_smem();
  mbar_arrive_expect_tx(bar, kStage);
  bulk_load(dst, c.k, kTileBytes, bar, policy);
  bulk_load(dst + kTileBytes, c.v, kTileBytes, bar, policy);
  return true;
}

// kN: query-head columns in units of 8 (group <= 8 * kN).
template <typename T, int kN, bool kScored>
__global__ void __launch_bounds__(warps_of(kN) * 32, 1) paged_decode_int4_kernel(const Params p) {
  using MO = Mma<T>;
  constexpr int kWarps = warps_of(kN), kRingBytes = ring_bytes(kWarps);
  constexpr int kParts = std::is_same<T, __half>::value ? 2 : 1;  // f16 pieces of p s
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 127u) & ~127u;
  uint8_t *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars_all = base + kRingBytes;
  int32_t *prefix = reinterpret_cast<int32_t *>(base_ptr + kRingBytes + kWarps * kStages * 8);

  launch_dependents();  // the merge kernel
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;

  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(bars_all + (warp * kStages + i) * 8, 1);
    fence_barrier_init();
  }
  build_prefix(p, prefix);  // contains __syncthreads

  const int32_t total = prefix[(p.batch + kSkip - 1) / kSkip];
  const int G = p.group;

  // Sequences with no context (graph padding rows) produce zeros.
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const int32_t len = __ldg(p.context_lens + b);
    if (len > static_cast<int64_t>(p.max_blocks) * p.block_size && threadIdx.x == 0)
      record_error(p.err, SLOKV_DEVERR_CONTEXT_LEN);
    if (len > 0 || (len < 0 && p.table_rows)) continue;  // (expanded rows: -1 is not ours to write)
    T *ob = static_cast<T *>(p.out) + static_cast<int64_t>(b) * p.out_sb;
    for (int i = threadIdx.x; i < p.hkv * G * kD; i += blockDim.x) {
      const int row = i / kD, d = i - row * kD;
      reinterpret_cast<uint16_t *>(ob + row * p.out_sh)[d] = 0;
    }
  }

  const Split split(total, p.nslots);
  const int32_t s = warp * gridDim.x + blockIdx.x;
  int4 job = make_int4(-1, 0, 0, 0);  // rewritten on every call
  if (s >= split.slots) {
    if (lane == 0) p.jobs[s] = job;
    return;
  }
  const int32_t a = split.start(s), e = split.start(s + 1);

  const uint32_t ring = base + warp * kStages * kStage;
  const uint32_t bars = bars_all + warp * kStages * 8;
  const uint64_t policy = l2_evict_first_policy();
  const int tiles_per_block = p.block_size / kTile;

  TileRef r = locate(p, prefix, a);
  Cursor cur = {};                  // lane 0: the tile that is issued next
  uint32_t empty = 0;               // lane 0: stages whose page lies outside the pool
  if (lane == 0) {
    cursor_init(cur, p, prefix, r, a, e, tiles_per_block);
    for (int i = 0; i < kStages && a + i < e; ++i) {
      if (!issue_tile(cur, ring, bars, i, policy)) empty |= 1u << i;
      if (a + i + 1 < e) cursor_next(cur, p, prefix, a + i + 1, e, tiles_per_block);
    }
  }
  __syncwarp();

  // Token of row n of an 8-token group: 2c -> c, 2c + 1 -> 4 + (c ^ 1).  Two neighbouring
  // rows then lie in shared memory rows of unlike parity, so that the 16-byte K loads
  // (two rows a quarter warp) do not collide and the V loads do so in pairs only.
  const int tok_k = (g & 1) ? 4 + ((g >> 1) ^ 1) : (g >> 1);
  const int tok_e = c, tok_o = 4 + (c ^ 1);

  int32_t t = a;
  while (t < e) {
    if (t != a) r = locate(p, prefix, t);
    const int32_t seg_end = r.seg_start + r.nt;
    const int32_t piece_end = min(seg_end, e);
    const int32_t len = seq_len(p, r.b);

    // q of head 8 rr + g of kv head r.h, f16, in the dim order of the codes: chunk c of a
    // code row holds dims 16c .. 16c + 15 of group 0 (words x, z) and of group 1 (words y,
    // w).  k-step 4 grp + 2 half takes the nibbles (0, 4), (2, 6) of the word, k-step + 1
    // the nibbles (1, 5), (3, 7), which the masks leave 16 times larger.
    uint32_t qb[kN][8][2];
    // B of the minimum's MMA: its A holds a token's (scale, minimum) words as they are, k = 2c
    // the scale and k = 2c + 1 the minimum of group c & 1, so B has zeros against the scales
    // and, against the minima, the group's sum of q in three bf16 pieces (24 bits).
    uint32_t qm[kN][2];
    float unscale[kN][2];   // accumulator unit -> log2-domain score, of the same heads
#pragma unroll
    for (int rr = 0; rr < kN; ++rr) {
      const int head = g + 8 * rr;
      const T *qr = static_cast<const T *>(p.q) + static_cast<int64_t>(r.b) * p.q_sb +
                    static_cast<int64_t>(r.h * G + head) * p.q_sh;
      float x[2][2][8];
      float amax = 0.f;
#pragma unroll
      for (int grp = 0; grp < 2; ++grp)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            const int d = 64 * grp + 16 * c + 8 * half + k;
            const uint32_t w = head < G ? *reinterpret_cast<const uint32_t *>(qr + d) : 0u;
            const float2 f = MO::unpack(w);
            x[grp][half][k] = f.x;
            x[grp][half][k + 1] = f.y;
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int ex = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
      const int k2 = min(max(14 - ex, -103), 110);
      // a negative softmax scale goes into q, so that the scores' order is the logits'
      const float mul = copysignf(__uint_as_float(static_cast<uint32_t>(k2 + 127) << 23), p.scale_log2);
      // (not 0 for a scale of 0: it multiplies the -inf of masked tokens)
      const float un = fmaxf(fabsf(p.scale_log2) * __uint_as_float(static_cast<uint32_t>(24 - k2 + 127) << 23),
                             1.17549435e-38f);
      unscale[rr][0] = __shfl_sync(0xffffffffu, un, 8 * c);
      unscale[rr][1] = __shfl_sync(0xffffffffu, un, 8 * c + 4);
      float qsum[2];
#pragma unroll
      for (int grp = 0; grp < 2; ++grp) {
        float sum = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float *v = x[grp][half];
          const int ks = 4 * grp + 2 * half;
          const float lo = mul * 0.0625f;
          qb[rr][ks][0] = Mma<__half>::pack(v[0] * mul, v[4] * mul);
          qb[rr][ks][1] = Mma<__half>::pack(v[2] * mul, v[6] * mul);
          qb[rr][ks + 1][0] = Mma<__half>::pack(v[1] * lo, v[5] * lo);
          qb[rr][ks + 1][1] = Mma<__half>::pack(v[3] * lo, v[7] * lo);
#pragma unroll
          for (int k = 0; k < 8; ++k) sum += v[k] * mul;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qsum[grp] = sum * 5.9604644775390625e-8f;  // 2^-24: the unit of the codes
      }
      float rest = c & 1 ? qsum[1] : qsum[0];
      const uint32_t q_hi = split_bf16(rest), q_mid = split_bf16(rest), q_lo = split_bf16(rest);
      qm[rr][0] = c < 2 ? q_hi : q_mid;
      qm[rr][1] = c < 2 ? q_lo : 0u;
    }

    // out^T accumulators: o[rr][4 grp + k][x] is dim 64 grp + 8 g + k (+ 4 for x >= 2) of head
    // 8 rr + 2 c + (x & 1), for odd k 16 times that and the even dim before it; vz: sum of p m
    // over this lane's tokens.  m: running maximum score, ref: what the scores are
    // exponentiated against.
    // moved_o: what was moved out of o, per group and head: the sums are o + moved_o (byte
    // sums o + 17 moved_o).
    float o[kN][8][4], vz[kN][2][2], moved_o[kN][2][2], m[kN][2], ref[kN][2], l[kN][2];
    // ceil(log2) of the largest V scale or minimum so far; at least -60, so that the sum of
    // p <= 2^75 stays finite over any context (V values all zero)
    int sexp = -60;
#pragma unroll
    for (int rr = 0; rr < kN; ++rr) {
#pragma unroll
      for (int n = 0; n < 8; ++n) o[rr][n][0] = o[rr][n][1] = o[rr][n][2] = o[rr][n][3] = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        vz[rr][n][0] = vz[rr][n][1] = moved_o[rr][n][0] = moved_o[rr][n][1] = 0.f;
        m[rr][n] = ref[rr][n] = -INFINITY;
        l[rr][n] = 0.f;
      }
    }

    for (int32_t tt = t; tt < piece_end; ++tt) {
      const int32_t idx = tt - a;
      const int stage = idx % kStages;
      const uint32_t parity = (idx / kStages) & 1;
      const int32_t j = tt - r.seg_start;
      if (!mbar_wait(bars + stage * 8, parity)) {
        if (lane == 0) record_error(p.err, SLOKV_DEVERR_TIMEOUT);
        // the copies that are still in flight into this ring, each wait bounded
        for (int i = 1; i < kStages && tt + i < e; ++i)
          mbar_wait(bars + (idx + i) % kStages * 8, ((idx + i) / kStages) & 1);
        if (lane == 0) p.jobs[s] = make_int4(-1, 0, 0, 0);
        return;
      }
      const int valid = min(kTile, len - j * kTile);
      uint8_t *kb = base_ptr + (warp * kStages + stage) * kStage;
      const uint8_t *vb = kb + kTileBytes;
      const bool hole = (__shfl_sync(0xffffffffu, empty, 0) >> stage) & 1u;
      if (hole || valid < kTile) {
        // Parameters of rows past the context (stale bytes, possibly NaN) and of pages
        // outside the pool read as zero; the codes are finite whatever they hold.
        uint8_t *pp = kb + kParamOff;
        for (int i = (hole ? 0 : valid) + lane; i < kTile; i += 32) {
          *reinterpret_cast<uint2 *>(pp + i * 8) = make_uint2(0u, 0u);
          *reinterpret_cast<uint2 *>(pp + kTileBytes + i * 8) = make_uint2(0u, 0u);
        }
        __syncwarp();
      }

      float *lg = nullptr;
      int room = 0;
      // (made anew for each tile: held across the loop its registers cost 1.5 %)
      const uint64_t keep = kScored ? l2_evict_last_policy() : 0;
      if constexpr (kScored) {
        room = min(valid, p.logits_stride - j * kTile);
        const int64_t row = (static_cast<int64_t>(r.b) * p.hkv + r.h) * p.logits_stride + j * kTile;
        lg = p.logits + row * p.logits_heads + 2 * c;
      }

      // ---- scores of 64 tokens x 8 kN heads, in the accumulators' unit ----
      float sc[kN][4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 w0 = lds128(kb + (16 * i + tok_k) * 64 + c * 16);
        const uint4 w1 = lds128(kb + (16 * i + 8 + tok_k) * 64 + c * 16);
        float acc[kN][2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int grp = 0; grp < 2; ++grp) {
            const uint32_t x0 = half ? (grp ? w0.w : w0.z) : (grp ? w0.y : w0.x);
            const uint32_t x1 = half ? (grp ? w1.w : w1.z) : (grp ? w1.y : w1.x);
            const uint32_t h0 = x0 >> 8, h1 = x1 >> 8;
            const int ks = 4 * grp + 2 * half;
#pragma unroll
            for (int rr = 0; rr < kN; ++rr) {
              if (half == 0)
                mma_f16_first(acc[rr][grp], x0 & 0x000f000fu, x1 & 0x000f000fu, h0 & 0x000f000fu,
                              h1 & 0x000f000fu, qb[rr][ks][0], qb[rr][ks][1]);
              else
                mma_f16(acc[rr][grp], x0 & 0x000f000fu, x1 & 0x000f000fu, h0 & 0x000f000fu,
                        h1 & 0x000f000fu, qb[rr][ks][0], qb[rr][ks][1]);
              mma_f16(acc[rr][grp], x0 & 0x00f000f0u, x1 & 0x00f000f0u, h0 & 0x00f000f0u,
                      h1 & 0x00f000f0u, qb[rr][ks + 1][0], qb[rr][ks + 1][1]);
            }
          }
        const uint32_t mw0 = lds32(kb + kParamOff + (16 * i + tok_k) * 8 + (c & 1) * 4);
        const uint32_t mw1 = lds32(kb + kParamOff + (16 * i + 8 + tok_k) * 8 + (c & 1) * 4);
#pragma unroll
        for (int rr = 0; rr < kN; ++rr)
          mma_bf16_first(sc[rr][i], mw0, mw1, mw0, mw1, qm[rr][0], qm[rr][1]);
#pragma unroll
        for (int row = 0; row < 2; ++row) {
          const uint2 pw = lds64(kb + kParamOff + (16 * i + 8 * row + tok_k) * 8);
          const float s0 = scale_of(pw.x), s1 = scale_of(pw.y);
#pragma unroll
          for (int rr = 0; rr < kN; ++rr)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              sc[rr][i][2 * row + x] = fmaf(s0, acc[rr][0][2 * row + x],
                                            fmaf(s1, acc[rr][1][2 * row + x], sc[rr][i][2 * row + x]));
          if constexpr (kScored) {
            // head pairs innermost: the lanes of 8 tokens write one contiguous run
            const int tok = 16 * i + 8 * row + tok_k;
#pragma unroll
            for (int rr = 0; rr < kN; ++rr)
              if (tok < room && 8 * rr + 2 * c < G)
                store_pair(lg + tok * p.logits_heads + 8 * rr, sc[rr][i][2 * row] * unscale[rr][0],
                           sc[rr][i][2 * row + 1] * unscale[rr][1], keep);
          }
        }
      }
      if (valid < kTile) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int row = 0; row < 2; ++row)
            if (16 * i + 8 * row + tok_k >= valid) {
#pragma unroll
              for (int rr = 0; rr < kN; ++rr) sc[rr][i][2 * row] = sc[rr][i][2 * row + 1] = -INFINITY;
            }
      }
      // ---- online softmax ----
      {
        // positive bf16 order as their bits, and both halves of a word count
        const uint2 p0 = lds64(vb + kParamOff + lane * 8), p1 = lds64(vb + kParamOff + (lane + 32) * 8);
        const uint32_t abs2 = 0x7fff7fffu;
        uint32_t top = __vmaxu2(__vmaxu2(p0.x & abs2, p0.y & abs2), __vmaxu2(p1.x & abs2, p1.y & abs2));
        top = __reduce_max_sync(0xffffffffu, max(top >> 16, top & 0xffffu));
        if (top >= 0x7f80u) {  // NaN parameters do not count
          const uint32_t w[4] = {p0.x & abs2, p0.y & abs2, p1.x & abs2, p1.y & abs2};
          top = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if ((w[i] & 0xffffu) < 0x7f80u) top = max(top, w[i] & 0xffffu);
            if ((w[i] >> 16) < 0x7f80u) top = max(top, w[i] >> 16);
          }
          top = __reduce_max_sync(0xffffffffu, top);
        }
        sexp = max(sexp, static_cast<int>(top >> 7) - 126);
      }
      const float under = static_cast<float>(15 - sexp);
      bool moved = false;
      float alpha[kN][2];
#pragma unroll
      for (int rr = 0; rr < kN; ++rr)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float mx = fmaxf(sc[rr][0][x], sc[rr][0][2 + x]);
#pragma unroll
          for (int i = 1; i < 4; ++i) mx = fmaxf(mx, fmaxf(sc[rr][i][x], sc[rr][i][2 + x]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          m[rr][x] = fmaxf(m[rr][x], mx * unscale[rr][x]);
          const float now = (m[rr][x] == -INFINITY ? 0.f : m[rr][x]) - under;
          alpha[rr][x] = fast_exp2(ref[rr][x] - now);
          moved |= now != ref[rr][x];
          ref[rr][x] = now;
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int rr = 0; rr < kN; ++rr) {
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            o[rr][n][0] *= alpha[rr][0];
            o[rr][n][1] *= alpha[rr][1];
            o[rr][n][2] *= alpha[rr][0];
            o[rr][n][3] *= alpha[rr][1];
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            vz[rr][n][0] *= alpha[rr][0];
            vz[rr][n][1] *= alpha[rr][1];
            moved_o[rr][n][0] *= alpha[rr][0];
            moved_o[rr][n][1] *= alpha[rr][1];
            l[rr][n] *= alpha[rr][n];
          }
        }
      }

      // ---- out^T += V^T P^T, 16 tokens a step ----
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t pb[kParts][kN][2][2];  // [piece][head columns][group][b0 | b1]
#pragma unroll
        for (int row = 0; row < 2; ++row) {
          const uint2 pw = lds64(vb + kParamOff + (16 * i + 8 * row + tok_k) * 8);
          const float s0 = scale_of(pw.x), s1 = scale_of(pw.y), m0 = min_of(pw.x), m1 = min_of(pw.y);
#pragma unroll
          for (int rr = 0; rr < kN; ++rr) {
            float pr[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              pr[x] = fast_exp2(fmaf(sc[rr][i][2 * row + x], unscale[rr][x], -ref[rr][x]));
              l[rr][x] += pr[x];
              vz[rr][0][x] = fmaf(pr[x], m0, vz[rr][0][x]);
              vz[rr][1][x] = fmaf(pr[x], m1, vz[rr][1][x]);
            }
            const uint32_t r0 = Mma<__half>::pack(pr[0] * s0, pr[1] * s0);
            const uint32_t r1 = Mma<__half>::pack(pr[0] * s1, pr[1] * s1);
            pb[0][rr][0][row] = movmatrix_trans(r0);
            pb[0][rr][1][row] = movmatrix_trans(r1);
            if constexpr (kParts == 2) {
              const float2 f0 = Mma<__half>::unpack(r0), f1 = Mma<__half>::unpack(r1);
              pb[1][rr][0][row] = movmatrix_trans(
                  Mma<__half>::pack(fmaf(pr[0], s0, -f0.x), fmaf(pr[1], s0, -f0.y)));
              pb[1][rr][1][row] = movmatrix_trans(
                  Mma<__half>::pack(fmaf(pr[0], s1, -f1.x), fmaf(pr[1], s1, -f1.y)));
            }
          }
        }
        const uint2 e0 = lds64(vb + (16 * i + tok_e) * 64 + g * 8);
        const uint2 o0 = lds64(vb + (16 * i + tok_o) * 64 + g * 8);
        const uint2 e1 = lds64(vb + (16 * i + 8 + tok_e) * 64 + g * 8);
        const uint2 o1 = lds64(vb + (16 * i + 8 + tok_o) * 64 + g * 8);
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
          const uint32_t x0 = grp ? e0.y : e0.x, y0 = grp ? o0.y : o0.x;
          const uint32_t x1 = grp ? e1.y : e1.x, y1 = grp ? o1.y : o1.x;
          const uint32_t lo0 = prmt(x0, y0, 0x5410u), hi0 = prmt(x0, y0, 0x7632u);
          const uint32_t lo1 = prmt(x1, y1, 0x5410u), hi1 = prmt(x1, y1, 0x7632u);
          // k even: the low nibble of a byte; k odd: the whole byte, low + 16 high
          uint32_t av[4][4] = {{lo0, hi0, lo1, hi1}};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            av[3][x] = prmt(av[0][x], 0u, 0x4341u);
            av[2][x] = av[3][x] & 0x000f000fu;
            av[1][x] = av[0][x] & 0x00ff00ffu;
            av[0][x] &= 0x000f000fu;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int rr = 0; rr < kN; ++rr)
#pragma unroll
              for (int part = 0; part < kParts; ++part)
                mma_f16(o[rr][4 * grp + k], av[k][0], av[k][1], av[k][2], av[k][3],
                        pb[part][rr][grp][0], pb[part][rr][grp][1]);
        }
      }
      // The codes are not negative, so o grows with the tokens while out need not, and the
      // MMA's additions truncate: the mean of 19,000 values in one run was 6.4e-3 off.  Every
      // kFlush tiles a lane moves the sum of one of its dims out of all of them, which leaves
      // their differences in o and 2.4e-3 (the output's rounding), for 114 -> 117 us.
      if ((tt - t) % kFlush == kFlush - 1) {
#pragma unroll
        for (int rr = 0; rr < kN; ++rr)
#pragma unroll
          for (int grp = 0; grp < 2; ++grp)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float y = o[rr][4 * grp][x];
              moved_o[rr][grp][x] += y;
#pragma unroll
              for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int up = 0; up < 2; ++up)
                  o[rr][4 * grp + k][2 * up + x] = fmaf(k & 1 ? -17.f : -1.f, y, o[rr][4 * grp + k][2 * up + x]);
            }
      }
      __syncwarp();
      if (lane == 0 && tt + kStages < e) {
        empty &= ~(1u << stage);
        if (!issue_tile(cur, ring, bars, stage, policy)) empty |= 1u << stage;
        if (tt + kStages + 1 < e) {
          cursor_next(cur, p, prefix, tt + kStages + 1, e, tiles_per_block);
        }
      }
      __syncwarp();
    }

    // ---- finish the piece ----
    const bool whole = (t == r.seg_start) && (piece_end == seg_end);
    const int slot_idx = (t == a && t > r.seg_start) ? 0 : 1;
    if (!whole && slot_idx == 0)
      job = make_int4(r.b, r.h, split.owner(r.seg_start), split.owner(seg_end - 1));
    float *pb = p.partials + (static_cast<int64_t>(s) * 2 + slot_idx) * G * kRowFloats;
#pragma unroll
    for (int rr = 0; rr < kN; ++rr)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) {
          l[rr][x] += __shfl_xor_sync(0xffffffffu, l[rr][x], d);
          vz[rr][0][x] += __shfl_xor_sync(0xffffffffu, vz[rr][0][x], d);
          vz[rr][1][x] += __shfl_xor_sync(0xffffffffu, vz[rr][1][x], d);
        }
        const int head = 8 * rr + 2 * c + x;
        if (head >= G) continue;
        const float lh = l[rr][x];
        const float inv = whole ? (lh > 0.f ? 1.f / lh : (lh == 0.f ? 0.f : lh)) : 1.f;
        if (g == 0) {
          if (!whole) {
            pb[head * kRowFloats] = ref[rr][x];
            pb[head * kRowFloats + 1] = lh;
          } else if (kScored) {
            p.lse[static_cast<int64_t>(r.b) * p.hkv * G + r.h * G + head] = ref[rr][x] + log2f(lh);
          }
        }
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
          // 2^24 undoes the codes' unit; an odd dim is its byte's sum less the even one's, / 16
          const float z = fmaf(16777216.f, moved_o[rr][grp][x], vz[rr][grp][x]);
          float v[8];
#pragma unroll
          for (int k = 0; k < 4; k += 2)
#pragma unroll
            for (int up = 0; up < 2; ++up) {
              const float low = o[rr][4 * grp + k][2 * up + x], byte = o[rr][4 * grp + k + 1][2 * up + x];
              v[k + 4 * up] = fmaf(16777216.f, low, z) * inv;
              v[k + 4 * up + 1] = fmaf(1048576.f, byte - low, z) * inv;
            }
          const int d = 64 * grp + 8 * g;
          if (whole) {
            uint32_t *ob = reinterpret_cast<uint32_t *>(
                static_cast<T *>(p.out) + static_cast<int64_t>(r.b) * p.out_sb +
                static_cast<int64_t>(r.h * G + head) * p.out_sh + d);
#pragma unroll
            for (int k = 0; k < 4; ++k) ob[k] = MO::pack(v[2 * k], v[2 * k + 1]);
          } else {
            float4 *row_acc = reinterpret_cast<float4 *>(pb + head * kRowFloats + kAccOff + d);
            row_acc[0] = make_float4(v[0], v[1], v[2], v[3]);
            row_acc[1] = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
      }
    t = piece_end;
  }
  if (lane == 0) p.jobs[s] = job;
}

// Combine the partials of every segment that straddles warp ranges.  Its pieces are the tail
// partial of slot s_lo and the head partials of slots s_lo + 1 .. s_hi.  One CTA per warp
// slot; the s_hi - s_lo CTAs of a segment share its (head, 32 dims) units, so that a long
// context cut into hundreds of pieces is read by many CTAs.  Eight threads take a unit's
// dims, as float4; the 32 such groups of a CTA are P pieces x 32 / P units at a time (P: the
// pieces, rounded up to a power of two), and the P partial sums meet by shuffles (4 to a
// warp) and in shared memory.
constexpr int kMergeThreads = 256;
constexpr int kMergeGroups = kMergeThreads / 8;

struct Merged {
  float m, l;
  float4 v;
};

__device__ __forceinline__ void merge_into(Merged &x, const Merged &y) {
  const float mn = fmaxf(x.m, y.m);
  const float a = x.m == -INFINITY ? 0.f : fast_exp2(x.m - mn);
  const float b = y.m == -INFINITY ? 0.f : fast_exp2(y.m - mn);
  x.m = mn;
  x.l = x.l * a + y.l * b;
  x.v = make_float4(x.v.x * a + y.v.x * b, x.v.y * a + y.v.y * b, x.v.z * a + y.v.z * b,
                    x.v.w * a + y.v.w * b);
}

template <typename T, bool kScored>
__global__ void __launch_bounds__(kMergeThreads) paged_decode_int4_merge_kernel(const Params p) {
  __shared__ Merged part[kMergeGroups][8];
  wait_prerequisites();
  const int32_t s = blockIdx.x;
  const int4 job = p.jobs[s];
  if (job.x < 0) return;
  const int G = p.group;
  const int32_t s_lo = job.z, pieces = job.w - s_lo + 1, sharers = pieces - 1;
  int P = 2;
  while (P < kMergeGroups && P < pieces) P *= 2;
  const int group = threadIdx.x >> 3, dim4 = threadIdx.x & 7, first = group % P;
  const int units = G * (kD / 32);
  for (int u0 = s - s_lo - 1; u0 < units; u0 += sharers * (kMergeGroups / P)) {
    const int u = u0 + (group / P) * sharers;
    const int head = u / (kD / 32), d = (u % (kD / 32)) * 32 + dim4 * 4;
    Merged x = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    if (u < units) {
#pragma unroll 2
      for (int32_t i = first; i < pieces; i += P) {
        const float *row = p.partials +
                           ((static_cast<int64_t>(s_lo + i) * 2 + (i == 0 ? 1 : 0)) * G + head) * kRowFloats;
        Merged y;
        const float2 ml = *reinterpret_cast<const float2 *>(row);
        y.m = ml.x;
        y.l = ml.y;
        y.v = *reinterpret_cast<const float4 *>(row + kAccOff + d);
        merge_into(x, y);
      }
    }
#pragma unroll
    for (int o = 8; o <= 16; o <<= 1) {
      Merged y;
      y.m = __shfl_xor_sync(0xffffffffu, x.m, o);
      y.l = __shfl_xor_sync(0xffffffffu, x.l, o);
      y.v.x = __shfl_xor_sync(0xffffffffu, x.v.x, o);
      y.v.y = __shfl_xor_sync(0xffffffffu, x.v.y, o);
      y.v.z = __shfl_xor_sync(0xffffffffu, x.v.z, o);
      y.v.w = __shfl_xor_sync(0xffffffffu, x.v.w, o);
      if (o < P * 8) merge_into(x, y);
    }
    if (P > 4) {
      if (first % 4 == 0) part[group][dim4] = x;
      __syncthreads();
      if (first == 0)
        for (int k = 4; k < P; k += 4) merge_into(x, part[group + k][dim4]);
      __syncthreads();
    }
    if (first == 0 && u < units) {
      const float inv = x.l > 0.f ? 1.f / x.l : (x.l == 0.f ? 0.f : x.l);
      uint32_t *ow = reinterpret_cast<uint32_t *>(
          static_cast<T *>(p.out) + static_cast<int64_t>(job.x) * p.out_sb +
          static_cast<int64_t>(job.y * G + head) * p.out_sh + d);
      ow[0] = Mma<T>::pack(x.v.x * inv, x.v.y * inv);
      ow[1] = Mma<T>::pack(x.v.z * inv, x.v.w * inv);
      if (kScored && d == 0)
        p.lse[static_cast<int64_t>(job.x) * p.hkv * G + job.y * G + head] = x.m + log2f(x.l);
    }
  }
}

int device_sms(int dev) {
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
    return -1;
  return n;
}

int warps_for(int group) { return warps_of(group <= 8 ? 1 : 2); }

size_t partial_bytes_for(int sms, int group) {
  return static_cast<size_t>(sms) * warps_for(group) * 2 * group * kRowFloats * sizeof(float);
}

size_t workspace_bytes_for(int sms, int group) {
  return partial_bytes_for(sms, group) + static_cast<size_t>(sms) * warps_for(group) * sizeof(int4);
}

size_t smem_bytes(int warps, int batch) {
  return 128 + ring_bytes(warps) + warps * kStages * 8 +
         ((static_cast<size_t>(batch) + kSkip - 1) / kSkip + 1) * sizeof(int32_t);
}

template <typename T, int kN, bool kScored>
int launch(const Params &p, int sms, cudaStream_t stream) {
  constexpr int kWarps = warps_of(kN);
  static std::atomic<uint64_t> done{0};
  const bool ok = once_per_device(done, [] {
    return cudaFuncSetAttribute(paged_decode_int4_kernel<T, kN, kScored>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(smem_bytes(kWarps, kMaxBatch))) == cudaSuccess;
  });
  if (!ok) return SLOKV_ERR_CUDA;
  paged_decode_int4_kernel<T, kN, kScored><<<sms, kWarps * 32, smem_bytes(kWarps, p.batch),
                                            stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return SLOKV_ERR_CUDA;
  return launch_dependent(paged_decode_int4_merge_kernel<T, kScored>,
                          dim3(static_cast<unsigned>(p.nslots)), dim3(kMergeThreads), 0, stream,
                          p) == cudaSuccess
             ? SLOKV_OK
             : SLOKV_ERR_CUDA;
}

template <typename T>
int pick(const Params &p, bool scored, int sms, cudaStream_t st) {
  if (p.group <= 8)
    return scored ? launch<T, 1, true>(p, sms, st) : launch<T, 1, false>(p, sms, st);
  return scored ? launch<T, 2, true>(p, sms, st) : launch<T, 2, false>(p, sms, st);
}

}  // namespace decode4
}  // namespace slokv

extern "C" size_t slokv_paged_decode_int4_workspace_bytes(int32_t device, int32_t num_q_heads,
                                                          int32_t num_kv_heads,
                                                          int32_t head_dim) {
  using namespace slokv::decode4;
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return 0;
  if (head_dim != kD || num_q_heads / num_kv_heads > 16) return 0;
  int dev = device;
  if (dev < 0 && cudaGetDevice(&dev) != cudaSuccess) return 0;
  const int sms = device_sms(dev);
  return sms > 0 ? workspace_bytes_for(sms, num_q_heads / num_kv_heads) : 0;
}

extern "C" int slokv_paged_decode_int4(void *out, int64_t out_stride_b, int64_t out_stride_h,
                                       const void *q, int64_t q_stride_b, int64_t q_stride_h,
                                       const void *k_cache, const void *v_cache,
                                       int64_t k_block_stride, int64_t v_block_stride,
                                       int32_t num_blocks, int32_t block_size,
                                       int32_t num_q_heads, int32_t num_kv_heads,
                                       int32_t head_dim, const int32_t *block_tables,
                                       int64_t block_table_stride, int32_t max_blocks_per_seq,
                                       const int32_t *table_rows, const int32_t *context_lens,
                                       int32_t batch, float softmax_scale, int32_t q_dtype,
                                       float *logits,
                                       int64_t logits_stride, float *lse, void *workspace,
                                       size_t workspace_bytes, uint32_t *dev_error,
                                       void *stream) {
  using namespace slokv;
  using namespace slokv::decode4;
  if (batch < 0 || num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || num_q_heads <= 0)
    return SLOKV_ERR_INVALID_ARG;
  if (batch == 0) return SLOKV_OK;
  if (batch > kMaxBatch || head_dim != kD) return SLOKV_ERR_UNSUPPORTED;
  if (q_dtype != SLOKV_DTYPE_BF16 && q_dtype != SLOKV_DTYPE_F16) return SLOKV_ERR_UNSUPPORTED;
  if (num_q_heads % num_kv_heads) return SLOKV_ERR_INVALID_ARG;
  const int group = num_q_heads / num_kv_heads;
  if (group > 16 || block_size % kTile) return SLOKV_ERR_UNSUPPORTED;
  if (max_blocks_per_seq > 0 &&
      !decode::tiles_fit(batch, num_kv_heads, max_blocks_per_seq, block_size, kTile))
    return SLOKV_ERR_UNSUPPORTED;
  if (!out || !q || !k_cache || !v_cache || !block_tables || !context_lens ||
      max_blocks_per_seq <= 0 || (logits != nullptr) != (lse != nullptr))
    return SLOKV_ERR_INVALID_ARG;
  if (logits && (logits_stride <= 0 || logits_stride > 0x7fffffff)) return SLOKV_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(logits) & 7u) return SLOKV_ERR_ALIGNMENT;
  const int64_t run = static_cast<int64_t>(num_kv_heads) * block_size * kRowBytes;
  if (((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15u) ||
      ((k_block_stride | v_block_stride) & 15) || k_block_stride < run || v_block_stride < run)
    return SLOKV_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 3u)
    return SLOKV_ERR_ALIGNMENT;
  if ((q_stride_b | q_stride_h | out_stride_b | out_stride_h) & 1) return SLOKV_ERR_ALIGNMENT;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return SLOKV_ERR_CUDA;
  const int sms = device_sms(dev);
  if (sms <= 0) return SLOKV_ERR_CUDA;
  if (!workspace || workspace_bytes < workspace_bytes_for(sms, group)) return SLOKV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15u) return SLOKV_ERR_ALIGNMENT;

  Params p;
  p.out = out;
  p.out_sb = out_stride_b;
  p.out_sh = out_stride_h;
  p.q = q;
  p.q_sb = q_stride_b;
  p.q_sh = q_stride_h;
  p.k_cache = static_cast<const uint8_t *>(k_cache);
  p.v_cache = static_cast<const uint8_t *>(v_cache);
  p.k_bs = k_block_stride;
  p.v_bs = v_block_stride;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.max_blocks = max_blocks_per_seq;
  p.context_lens = context_lens;
  p.batch = batch;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.hkv = num_kv_heads;
  p.group = group;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.partials = static_cast<float *>(workspace);
  p.jobs = reinterpret_cast<int4 *>(static_cast<char *>(workspace) + partial_bytes_for(sms, group));
  p.table_rows = table_rows;
  p.logits = logits;
  p.logits_heads = (group + 1) / 2 * 2;
  p.lse = lse;
  p.logits_stride = static_cast<int32_t>(logits_stride);
  p.err = dev_error;
  p.nslots = sms * warps_for(group);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return q_dtype == SLOKV_DTYPE_BF16 ? pick<__nv_bfloat16>(p, logits != nullptr, sms, st)
                                     : pick<__half>(p, logits != nullptr, sms, st);
}
