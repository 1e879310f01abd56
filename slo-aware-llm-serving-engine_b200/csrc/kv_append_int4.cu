// Quantising paged append to the 4-bit KV pool, the read-back of single rows and the
// widening of cached rows for prefill.
//
// Contract, per token, kv head and group of 64 dims (every step IEEE fp32):
//   mn = min x, mx = max x
//   scale = bf16((mx - mn) / 15), minimum = bf16(mn)
//   code = scale > 0 ? clamp(rint((x - minimum) / scale), 0, 15) : 0
// The value is within half a scale of x, except that f16 and fp32 groups with |min| > 7 (mx -
// mn) clamp where bf16(min) misses min: within 2^-8 (|min| + mx - mn).
// A group with a NaN or an infinity, or whose range overflows fp32, is stored with a
// NaN scale (its values read as NaN) and flags SLOKV_DEVERR_NONFINITE.  A token's
// parameters are its own, so nothing stored before is touched and a page needs no
// reset when it changes hands.
//
// Append: eight lanes per row of 128 dims, 16 dims a lane: two 16-byte loads, a two-step
// shuffle min / max over the 4 lanes of a group, one exchange between the groups' lanes and an
// 8-byte store (the eight lanes' stores are the row's 64 contiguous bytes).  A CTA takes 16
// tokens of one head, K and V, so its rows are neighbours in the page.  Issue-bound: 14 us
// for 6211 tokens of 8 heads (33 MB, 5 us of HBM) at 104 warp instructions a row; 31 us with
// a division a value and 8 dims a lane.  So the quotient is a multiplication by an
// approximate 1 / scale, 2^-22 of itself off; a value that this leaves within 2^-16 of a
// border between two codes is divided, and the codes are always those of the true
// division.
//
// Read-back and widening: eight lanes per row, each with the 8 bytes that hold 8 dims
// of either group, so that the 16-byte stores of a row are contiguous.  Bound by the
// latency of the small loads (widening 4 rows of 16,000 tokens in all, 8 heads: 20 us for
// 86 MB), so all of a thread's rows are loaded before the first is stored (30 us without).
#include "common.cuh"
#include "int4_page.cuh"

#include <type_traits>

namespace slokv {
namespace {

using namespace kv4;

constexpr int kThreads = 256;
constexpr int kRowsPerCta = kThreads / 8;

template <typename T>
__device__ __forceinline__ float widen(T x);
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float widen<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float widen<float>(float x) { return x; }

// Eight consecutive elements of a row; kVec: the address is 16-byte aligned.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T *p, float *x) {
  if constexpr (kVec && sizeof(T) == 2) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(p));
    const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = widen(e[i]);
  } else if constexpr (kVec) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p));
    const float4 b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = widen(p[i]);
  }
}

// n / d for 0 <= n < 2^31 without a division (the round-up method of Granlund and
// Montgomery, 1994): q = (n + high32(n m)) >> l with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1.
struct FastDiv {
  uint32_t m, l;
  explicit FastDiv(uint32_t d) {
    l = 0;
    while ((1ull << l) < d) ++l;
    m = static_cast<uint32_t>((((1ull << l) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int32_t operator()(int32_t n) const {
    const uint32_t u = static_cast<uint32_t>(n);
    return static_cast<int32_t>((u + __umulhi(u, m)) >> l);
  }
};

__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes of 8 values of a group with minimum m and scale s > 0, the k-th in bits 4k ..;
// inv: 1 / s, approximately.  kExact: m is the minimum itself, so x >= m, and s >= range /
// 15 (1 - 2^-8) gives quotients below 15.1: no code needs clamping.  (Scales below 2^-120,
// which bf16 may hold less exactly, always divide: inv is NaN for them.  None is above
// 2^125, so the reciprocal is a normal number.)
template <bool kExact>
__device__ __forceinline__ uint32_t encode8(const float *x, float m, float s, float inv) {
  const float magic = 12582912.f;    // 1.5 * 2^23: adding it rounds to an integer
  uint32_t word = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float d = __fsub_rn(x[i], m);
    const float t = __fmaf_rn(d, inv, magic);
    int32_t bits = __float_as_int(t);  // magic's bits plus the code
    // not within 0.5 - 2^-16 of the integer (four times what 15 2^-22 is off), or NaN
    if (!(fabsf(__fmaf_rn(d, inv, -__fsub_rn(t, magic))) <= 0.49998474f))
      bits = __float_as_int(magic + fminf(fmaxf(rintf(__fdiv_rn(d, s)), 0.f), 15.f));
    if (!kExact) bits = min(max(bits, __float_as_int(magic)), __float_as_int(magic) + 15);
    word = word * 16u + static_cast<uint32_t>(bits);
  }
  return word - 0x3f400000u;         // the sum of magic's bits (0x4b400000) 16^i, modulo 2^32
}

constexpr int kTokensPerCta = kRowsPerCta / 2;  // K and V

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads)
    kv_append_int4_kernel(const T *__restrict__ key, int64_t key_stride, int64_t key_head,
                          const T *__restrict__ value, int64_t value_stride, int64_t value_head,
                          uint8_t *__restrict__ k_cache, uint8_t *__restrict__ v_cache,
                          int64_t k_block_stride, int64_t v_block_stride,
                          const int32_t *__restrict__ slots, int32_t tokens, int32_t hkv,
                          int32_t block_size, int32_t num_blocks, FastDiv by_hkv, FastDiv by_block,
                          uint32_t *err) {
  const int lane = threadIdx.x & 31, sub = lane & 7;
  // a warp holds K and V of two tokens; every lane takes part in the shuffles
  const bool is_v = lane & 8;
  const int32_t chunk = by_hkv(blockIdx.x), h = blockIdx.x - chunk * hkv;
  const int32_t t = chunk * kTokensPerCta + (threadIdx.x >> 4);
  const int32_t slot = t < tokens ? __ldg(slots + t) : -1;
  const int32_t blk = by_block(max(slot, 0)), off = slot - blk * block_size;
  const bool live = slot >= 0 && blk < num_blocks;
  if (!live && slot != -1 && sub == 0) record_error(err, SLOKV_DEVERR_SLOT_RANGE);
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
  if (live) {
    const T *src = is_v ? value + t * value_stride + h * value_head
                        : key + t * key_stride + h * key_head;
    src += sub * 16;
    load8<T, kVec>(src, x);
    load8<T, kVec>(src + 8, x + 8);
  }
  float mn = x[0], mx = x[0], zero = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    mn = fminf(mn, x[i]);
    mx = fmaxf(mx, x[i]);
    zero = __fmaf_rn(x[i], 0.f, zero);  // NaN where a value is not finite
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const uint32_t votes = __ballot_sync(0xffffffffu, zero != zero);
  bool bad = (votes >> (lane & 28)) & 0xfu;
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(mx, mn), 15.f));
  const __nv_bfloat16 mb = __float2bfloat16_rn(mn);
  const float s = __bfloat162float(sb), m = __bfloat162float(mb);
  bad |= !isfinite(s) || !isfinite(m);
  uint32_t w0 = 0, w1 = 0;
  if (!bad && s > 0.f) {
    constexpr bool kExact = std::is_same<T, __nv_bfloat16>::value;  // other minima may round up
    const float inv = s < 7.5e-37f ? __int_as_float(0x7fffffff) : rcp_fast(s);
    w0 = encode8<kExact>(x, m, s, inv);
    w1 = encode8<kExact>(x + 8, m, s, inv);
  }
  // lane j of group 0 has the row's stored words 4j, 4j + 2 and lane j of group 1 4j + 1, 4j + 3
  const int grp = sub >> 2, j = sub & 3;
  const uint32_t other = __shfl_xor_sync(0xffffffffu, grp ? w0 : w1, 4);
  if (!live) return;
  uint8_t *run = (is_v ? v_cache + blk * v_block_stride : k_cache + blk * k_block_stride) +
                 static_cast<int64_t>(h) * block_size * kRowBytes;
  *reinterpret_cast<uint2 *>(run + code_offset(off) + 16 * j + 8 * grp) =
      grp ? make_uint2(other, w1) : make_uint2(w0, other);
  if (j == 0) {
    const uint32_t lo = bad ? 0x7fffu : __bfloat16_as_ushort(sb);
    const uint32_t hi = bad ? 0u : __bfloat16_as_ushort(mb);
    *reinterpret_cast<uint32_t *>(run + param_offset(off) + 4 * grp) = lo | (hi << 16);
    if (bad) record_error(err, SLOKV_DEVERR_NONFINITE);
  }
}

constexpr int kWideRows = kThreads / 8;   // rows at a time of the read-back and the widening

// What lane i of eight holds of a row: dims 8i .. 8i + 7 of either group, and both groups'
// parameters.
struct Piece {
  uint2 code, par;
};

__device__ __forceinline__ Piece load_piece(const uint8_t *run, int32_t off, int i) {
  return {__ldg(reinterpret_cast<const uint2 *>(run + code_offset(off) + 8 * i)),
          __ldg(reinterpret_cast<const uint2 *>(run + param_offset(off)))};
}

__device__ __forceinline__ void piece_values(const Piece &p, int grp, float (&v)[8]) {
  const uint32_t w = grp ? p.code.y : p.code.x, pw = grp ? p.par.y : p.par.x;
  const float s = scale_of(pw), m = min_of(pw);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = fmaf(s, static_cast<float>((w >> (4 * k)) & 15u), m);
}

// fp32 values of the rows at `slots` (-1 or outside the pool: zeros).
__global__ void __launch_bounds__(kThreads)
    int4_decode_kernel(const uint8_t *__restrict__ cache, int64_t block_stride,
                       const int32_t *__restrict__ slots, int32_t tokens, int32_t hkv,
                       int32_t block_size, int32_t num_blocks, float *__restrict__ out,
                       uint32_t *err) {
  const int i = threadIdx.x & 7;
  const int32_t chunk = blockIdx.x / hkv, h = blockIdx.x - chunk * hkv;
  const int32_t t = chunk * kWideRows + (threadIdx.x >> 3);
  if (t >= tokens) return;
  const int32_t slot = __ldg(slots + t);
  const int32_t blk = slot / block_size;
  Piece p = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
  if (slot >= 0 && blk < num_blocks)
    p = load_piece(cache + blk * block_stride + static_cast<int64_t>(h) * block_size * kRowBytes,
                   slot - blk * block_size, i);
  else if (slot != -1 && i == 0)
    record_error(err, SLOKV_DEVERR_SLOT_RANGE);
  float *o = out + (static_cast<int64_t>(t) * hkv + h) * kHeadDim + i * 8;
#pragma unroll
  for (int grp = 0; grp < 2; ++grp) {
    float v[8];
    piece_values(p, grp, v);
    reinterpret_cast<float4 *>(o + 64 * grp)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(o + 64 * grp)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// Widen the cached tokens of a prefill call's rows to bf16 / f16: token t of row r goes to
// page r * pages + t / 128 of 128-token pages [.., 128, hkv, 128], whose table is written
// beside them.  One CTA per (page, head, side).  A page that the row reaches is
// written whole (zeros past its last key and for a block id outside the pool: the
// prefill loads whole pages); the others are left alone.
//
// f16: a row of finite f16 can read back past 65,504: its minimum is rounded to bf16 (up by
// 128 at most, down to -65,536) and so is its scale (half a step is 32 at most, 15 scales 480),
// which makes 65,504 + 608 = 66,112 at most.  Those values are clamped, towards what was
// stored; larger ones, of pools written in other types, become infinite and are flagged.
constexpr int kWidePage = 128;
constexpr float kF16Max = 65504.f, kF16Reach = 66112.f;

template <typename T>
__global__ void __launch_bounds__(kThreads)
    int4_rows_widen_kernel(const uint8_t *__restrict__ k_cache, const uint8_t *__restrict__ v_cache,
                           int64_t k_block_stride, int64_t v_block_stride, int32_t num_blocks,
                           int32_t block_size, int32_t hkv, const int32_t *__restrict__ tables,
                           int64_t bt_stride, int32_t max_blocks, const int32_t *__restrict__ cu_k,
                           int32_t pages, T *__restrict__ dst_k, T *__restrict__ dst_v,
                           int32_t *__restrict__ dst_table, uint32_t *err) {
  const int32_t page = blockIdx.x % pages, r = blockIdx.x / pages;
  const int32_t h = blockIdx.y;
  const bool is_v = blockIdx.z;
  const bool first = h == 0 && !is_v && threadIdx.x == 0;
  if (first) dst_table[blockIdx.x] = blockIdx.x;
  int64_t keys = static_cast<int64_t>(__ldg(cu_k + r + 1)) - __ldg(cu_k + r);
  const int64_t t0 = static_cast<int64_t>(page) * kWidePage;
  if (t0 >= keys) return;
  const int64_t reach = static_cast<int64_t>(max_blocks) * block_size;
  if (keys > reach) {                             // keys past the table read as zeros
    if (first && page == 0) record_error(err, SLOKV_DEVERR_CONTEXT_LEN);
    keys = reach;
  }
  const uint8_t *cache = is_v ? v_cache : k_cache;
  const int64_t stride = is_v ? v_block_stride : k_block_stride;
  T *dst = (is_v ? dst_v : dst_k) +
           (static_cast<int64_t>(blockIdx.x) * kWidePage * hkv + h) * kHeadDim;
  const int i = threadIdx.x & 7;
  constexpr int kSteps = kWidePage / kWideRows;
  Piece piece[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {              // all loads before the first store
    piece[k] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
    const int64_t t = t0 + k * kWideRows + (threadIdx.x >> 3);
    if (t >= keys) continue;
    const int32_t col = static_cast<int32_t>(t) / block_size;
    const int32_t blk = __ldg(tables + r * bt_stride + col);
    if (blk >= 0 && blk < num_blocks)
      piece[k] = load_piece(cache + blk * stride + static_cast<int64_t>(h) * block_size * kRowBytes,
                            static_cast<int32_t>(t) - col * block_size, i);
    else if (i == 0)
      record_error(err, SLOKV_DEVERR_BLOCK_RANGE);
  }
  bool past = false;                              // a value that f16 cannot hold
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    T *o = dst + static_cast<int64_t>(k * kWideRows + (threadIdx.x >> 3)) * hkv * kHeadDim + i * 8;
#pragma unroll
    for (int grp = 0; grp < 2; ++grp) {
      float v[8];
      piece_values(piece[k], grp, v);
      if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {             // (NaN passes both tests unchanged)
          past |= fabsf(v[e]) > kF16Reach;
          if (fabsf(v[e]) <= kF16Reach) v[e] = fminf(fmaxf(v[e], -kF16Max), kF16Max);
        }
      }
      uint4 w;
      w.x = Mma<T>::pack(v[0], v[1]);
      w.y = Mma<T>::pack(v[2], v[3]);
      w.z = Mma<T>::pack(v[4], v[5]);
      w.w = Mma<T>::pack(v[6], v[7]);
      *reinterpret_cast<uint4 *>(o + 64 * grp) = w;
    }
  }
  if (past) record_error(err, SLOKV_DEVERR_NONFINITE);
}

// The queries of a short prefill as decode rows: query token i of row r attends to the
// first k_len - q_len + i + 1 cached tokens of table row r.  Tokens that no row names get
// the length -1.
__global__ void int4_rows_expand_kernel(const int32_t *__restrict__ cu_q,
                                        const int32_t *__restrict__ cu_k, int32_t rows,
                                        int32_t tokens, int32_t *__restrict__ table_rows,
                                        int32_t *__restrict__ lens) {
  const int32_t t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= tokens) return;
  // the last row that starts at or before t
  int32_t lo = 0, hi = rows - 1;
  while (lo < hi) {
    const int32_t mid = (lo + hi + 1) >> 1;
    if (__ldg(cu_q + mid) <= t) lo = mid; else hi = mid - 1;
  }
  const int32_t first = __ldg(cu_q + lo), last = __ldg(cu_q + lo + 1);
  const bool named = t >= first && t < last;
  const int32_t keys = __ldg(cu_k + lo + 1) - __ldg(cu_k + lo);
  table_rows[t] = lo;
  lens[t] = named ? max(0, keys - (last - t) + 1) : -1;
}

bool pool_ok(const void *base, int64_t block_stride, int32_t hkv, int32_t block_size) {
  return !(reinterpret_cast<uintptr_t>(base) & 15u) && !(block_stride & 15) &&
         block_stride >= static_cast<int64_t>(hkv) * block_size * kRowBytes;
}

// Whether every row's 8-element pieces lie on 16-byte boundaries.
bool vec_ok(const void *p, int64_t stride, int64_t head, int elem) {
  return !(reinterpret_cast<uintptr_t>(p) & 15u) && !((stride * elem) & 15) && !((head * elem) & 15);
}

}  // namespace
}  // namespace slokv

extern "C" int slokv_kv_append_int4(const void *key, int64_t key_row_stride,
                                    int64_t key_head_stride, const void *value,
                                    int64_t value_row_stride, int64_t value_head_stride,
                                    void *k_cache, void *v_cache, int64_t k_block_stride,
                                    int64_t v_block_stride, const int32_t *slot_mapping,
                                    int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim,
                                    int32_t block_size, int32_t num_blocks, int32_t in_dtype,
                                    uint32_t *dev_error, void *stream) {
  using namespace slokv;
  if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks <= 0 || block_size <= 0)
    return SLOKV_ERR_INVALID_ARG;
  if (head_dim != kHeadDim || block_size % kTileTokens) return SLOKV_ERR_UNSUPPORTED;
  if (in_dtype != SLOKV_DTYPE_BF16 && in_dtype != SLOKV_DTYPE_F16 && in_dtype != SLOKV_DTYPE_F32)
    return SLOKV_ERR_UNSUPPORTED;
  if (num_tokens == 0) return SLOKV_OK;
  if (!key || !value || !k_cache || !v_cache || !slot_mapping) return SLOKV_ERR_INVALID_ARG;
  if (!pool_ok(k_cache, k_block_stride, num_kv_heads, block_size) ||
      !pool_ok(v_cache, v_block_stride, num_kv_heads, block_size))
    return SLOKV_ERR_ALIGNMENT;
  const int elem = in_dtype == SLOKV_DTYPE_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & (elem - 1))
    return SLOKV_ERR_ALIGNMENT;
  const int64_t chunks = (static_cast<int64_t>(num_tokens) + kTokensPerCta - 1) / kTokensPerCta;
  if (chunks * num_kv_heads > 0x7fffffff) return SLOKV_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(chunks * num_kv_heads);
  const bool vec = vec_ok(key, key_row_stride, key_head_stride, elem) &&
                   vec_ok(value, value_row_stride, value_head_stride, elem);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel, auto tag) {
    using T = decltype(tag);
    kernel<<<grid, kThreads, 0, st>>>(
        static_cast<const T *>(key), key_row_stride, key_head_stride,
        static_cast<const T *>(value), value_row_stride, value_head_stride,
        static_cast<uint8_t *>(k_cache), static_cast<uint8_t *>(v_cache), k_block_stride,
        v_block_stride, slot_mapping, num_tokens, num_kv_heads, block_size, num_blocks,
        FastDiv(num_kv_heads), FastDiv(block_size), dev_error);
    return cudaGetLastError() == cudaSuccess ? SLOKV_OK : SLOKV_ERR_CUDA;
  };
  if (in_dtype == SLOKV_DTYPE_BF16)
    return vec ? go(kv_append_int4_kernel<__nv_bfloat16, true>, __nv_bfloat16())
               : go(kv_append_int4_kernel<__nv_bfloat16, false>, __nv_bfloat16());
  if (in_dtype == SLOKV_DTYPE_F16)
    return vec ? go(kv_append_int4_kernel<__half, true>, __half())
               : go(kv_append_int4_kernel<__half, false>, __half());
  return vec ? go(kv_append_int4_kernel<float, true>, float())
             : go(kv_append_int4_kernel<float, false>, float());
}

extern "C" int slokv_int4_decode(const void *cache, int64_t block_stride,
                                 const int32_t *slot_mapping, int32_t num_tokens,
                                 int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                 int32_t num_blocks, float *out, uint32_t *dev_error,
                                 void *stream) {
  using namespace slokv;
  if (num_tokens < 0 || num_kv_heads <= 0 || num_blocks <= 0 || block_size <= 0)
    return SLOKV_ERR_INVALID_ARG;
  if (head_dim != kHeadDim || block_size % kTileTokens) return SLOKV_ERR_UNSUPPORTED;
  if (num_tokens == 0) return SLOKV_OK;
  if (!cache || !slot_mapping || !out) return SLOKV_ERR_INVALID_ARG;
  if (!pool_ok(cache, block_stride, num_kv_heads, block_size) ||
      (reinterpret_cast<uintptr_t>(out) & 15u))
    return SLOKV_ERR_ALIGNMENT;
  const int64_t chunks = (static_cast<int64_t>(num_tokens) + kWideRows - 1) / kWideRows;
  if (chunks * num_kv_heads > 0x7fffffff) return SLOKV_ERR_UNSUPPORTED;
  int4_decode_kernel<<<static_cast<unsigned>(chunks * num_kv_heads), kThreads, 0,
                       static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t *>(cache), block_stride, slot_mapping, num_tokens, num_kv_heads,
      block_size, num_blocks, out, dev_error);
  return cudaGetLastError() == cudaSuccess ? SLOKV_OK : SLOKV_ERR_CUDA;
}

extern "C" int slokv_int4_rows_widen(const void *k_cache, const void *v_cache,
                                     int64_t k_block_stride, int64_t v_block_stride,
                                     int32_t num_blocks, int32_t block_size, int32_t num_kv_heads,
                                     int32_t head_dim, const int32_t *block_tables,
                                     int64_t block_table_stride, int32_t max_blocks_per_seq,
                                     const int32_t *cu_seqlens_k, int32_t num_rows,
                                     int32_t pages_per_row, void *dst_k, void *dst_v,
                                     int32_t *dst_table, int32_t dst_dtype, uint32_t *dev_error,
                                     void *stream) {
  using namespace slokv;
  if (num_rows < 0 || pages_per_row < 0 || num_kv_heads <= 0 || num_blocks <= 0 || block_size <= 0)
    return SLOKV_ERR_INVALID_ARG;
  if (head_dim != kHeadDim || block_size % kTileTokens) return SLOKV_ERR_UNSUPPORTED;
  if (dst_dtype != SLOKV_DTYPE_BF16 && dst_dtype != SLOKV_DTYPE_F16) return SLOKV_ERR_UNSUPPORTED;
  if (num_rows == 0 || pages_per_row == 0) return SLOKV_OK;
  if (!k_cache || !v_cache || !block_tables || !cu_seqlens_k || !dst_k || !dst_v || !dst_table ||
      max_blocks_per_seq <= 0)
    return SLOKV_ERR_INVALID_ARG;
  if (!pool_ok(k_cache, k_block_stride, num_kv_heads, block_size) ||
      !pool_ok(v_cache, v_block_stride, num_kv_heads, block_size) ||
      ((reinterpret_cast<uintptr_t>(dst_k) | reinterpret_cast<uintptr_t>(dst_v)) & 15u))
    return SLOKV_ERR_ALIGNMENT;
  const int64_t pages = static_cast<int64_t>(num_rows) * pages_per_row;
  if (pages > 0x7fffffff || num_kv_heads > 65535) return SLOKV_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(pages), static_cast<unsigned>(num_kv_heads), 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kernel, auto tag) {
    using T = decltype(tag);
    kernel<<<grid, kThreads, 0, st>>>(
        static_cast<const uint8_t *>(k_cache), static_cast<const uint8_t *>(v_cache),
        k_block_stride, v_block_stride, num_blocks, block_size, num_kv_heads, block_tables,
        block_table_stride, max_blocks_per_seq, cu_seqlens_k, pages_per_row,
        static_cast<T *>(dst_k), static_cast<T *>(dst_v), dst_table, dev_error);
    return cudaGetLastError() == cudaSuccess ? SLOKV_OK : SLOKV_ERR_CUDA;
  };
  return dst_dtype == SLOKV_DTYPE_BF16 ? go(int4_rows_widen_kernel<__nv_bfloat16>, __nv_bfloat16())
                                       : go(int4_rows_widen_kernel<__half>, __half());
}

extern "C" int slokv_int4_rows_expand(const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k,
                                      int32_t num_rows, int32_t num_tokens, int32_t *table_rows,
                                      int32_t *context_lens, void *stream) {
  using namespace slokv;
  if (num_rows < 0 || num_tokens < 0) return SLOKV_ERR_INVALID_ARG;
  if (num_rows == 0 || num_tokens == 0) return SLOKV_OK;
  if (!cu_seqlens_q || !cu_seqlens_k || !table_rows || !context_lens) return SLOKV_ERR_INVALID_ARG;
  int4_rows_expand_kernel<<<static_cast<unsigned>((num_tokens + 127ll) / 128), 128, 0,
                            static_cast<cudaStream_t>(stream)>>>(
      cu_seqlens_q, cu_seqlens_k, num_rows, num_tokens, table_rows, context_lens);
  return cudaGetLastError() == cudaSuccess ? SLOKV_OK : SLOKV_ERR_CUDA;
}
