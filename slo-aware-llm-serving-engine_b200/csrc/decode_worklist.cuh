// Work list of the persistent decode kernels: the tiles (kTile tokens) of every
// (sequence, kv head) segment in the order (b, kv head, tile), split into equal
// contiguous ranges, one per warp slot.  `P` is a kernel's parameter block with
// context_lens, batch, max_blocks, block_size and hkv.
#pragma once

#include "common.cuh"

namespace slokv {
namespace decode {

constexpr int kD = 128;                         // head_dim
constexpr int kRowFloats = kD + 4;              // partial row: m, l, pad, pad, acc[kD]
constexpr int kAccOff = 4;                      // acc starts 16-byte aligned
constexpr int kMaxBatch = 8192;

// Whether the work list of every table row filled to its reach counts in 32 bits.
inline bool tiles_fit(int64_t batch, int64_t hkv, int64_t max_blocks, int64_t block_size, int tile) {
  const int64_t segments = batch * hkv;
  return segments <= 0x7fffffff &&
         (max_blocks * block_size + tile - 1) / tile <= 0x7fffffff / segments;
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Number of tiles of sequence b (its segment length per kv head).
template <int kTile, typename P>
__device__ __forceinline__ int32_t seq_tiles(const P &p, int b, uint32_t *err_bits) {
  int32_t len = __ldg(p.context_lens + b);
  if (len <= 0) return 0;
  const int64_t cap = static_cast<int64_t>(p.max_blocks) * p.block_size;
  if (len > cap) {
    *err_bits |= SLOKV_DEVERR_CONTEXT_LEN;
    len = static_cast<int32_t>(cap);
  }
  return (len + kTile - 1) / kTile;
}

template <typename P>
__device__ __forceinline__ int32_t seq_len_clamped(const P &p, int b) {
  int32_t len = __ldg(p.context_lens + b);
  const int64_t cap = static_cast<int64_t>(p.max_blocks) * p.block_size;
  return len > cap ? static_cast<int32_t>(cap) : len;
}

// Exclusive prefix over sequences of (tiles_b * hkv) into prefix[0..batch].
// Called by all threads of the CTA.
template <int kTile, typename P>
__device__ void build_prefix(const P &p, int32_t *prefix, uint32_t *err_bits) {
  __shared__ int32_t warp_sums[32];
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int per = (p.batch + nthr - 1) / nthr;
  const int lo = min(tid * per, p.batch), hi = min(lo + per, p.batch);
  int32_t local = 0;
  for (int b = lo; b < hi; ++b) local += seq_tiles<kTile>(p, b, err_bits) * p.hkv;
  // inclusive scan of `local` across the CTA
  const int lane = tid & 31, warp = tid >> 5;
  int32_t v = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    int32_t t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    const int nw = nthr >> 5;
    int32_t w = lane < nw ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      int32_t t = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += t;
    }
    if (lane < nw) warp_sums[lane] = w;
  }
  __syncthreads();
  int32_t run = v - local + (warp > 0 ? warp_sums[warp - 1] : 0);
  for (int b = lo; b < hi; ++b) {
    prefix[b] = run;
    uint32_t dummy = 0;
    run += seq_tiles<kTile>(p, b, &dummy) * p.hkv;
  }
  if (tid == nthr - 1) prefix[p.batch] = run;
  __syncthreads();
}

struct TileRef {
  int32_t b, h, j, nt, seg_start;
};

// Locate global tile t: largest b with prefix[b] <= t.
template <typename P>
__device__ __forceinline__ TileRef locate(const P &p, const int32_t *prefix, int64_t t) {
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= t) lo = mid; else hi = mid - 1;
  }
  TileRef r;
  r.b = lo;
  r.nt = (prefix[lo + 1] - prefix[lo]) / p.hkv;
  const int32_t rel = static_cast<int32_t>(t - prefix[lo]);
  r.h = rel / r.nt;
  r.j = rel - r.h * r.nt;
  r.seg_start = prefix[lo] + r.h * r.nt;
  return r;
}

__device__ __forceinline__ int64_t range_start(int64_t s, int64_t total, int64_t nslots) {
  return (s * total) / nslots;
}

// Slot that owns global tile t (max s with range_start(s) <= t).
__device__ __forceinline__ int64_t owner_slot(int64_t t, int64_t total, int64_t nslots) {
  int64_t s = (t * nslots) / total;
  if (s >= nslots) s = nslots - 1;
  while (s + 1 < nslots && range_start(s + 1, total, nslots) <= t) ++s;
  while (s > 0 && range_start(s, total, nslots) > t) --s;
  return s;
}

}  // namespace decode
}  // namespace slokv
