"""4-bit KV cache: quantising store, decode and prefill attention, read-back.

One side of a pool is uint8 [num_blocks, num_kv_heads, block_size * 72]
(block_size a multiple of 64, head_dim 128; layout and rounding rules in
include/slokv.h): 64 code bytes and 8 parameter bytes per token and head
against 256 bytes in bf16 and 128 in FP8.  Each token carries its own scale and
minimum per 64 dims, so a store touches nothing but its own tokens and pages
change hands without a reset.

The functions are the counterparts of store_kvcache, flash_attn_with_kvcache
and flash_attn_varlen_func.  They run on the current stream of the tensors'
device, never synchronise, and take their scratch from torch's caching
allocator per call, so calls on several streams and graphs replayed side by
side do not share any.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import SlokvError, buffers, check, lib, require_cuda, stream_ptr
from .kvcache import _i32_contig, _varlen_attention

HEAD_DIM = 128
TILE_TOKENS = 64
ROW_BYTES = 72          # 64 bytes of codes, 2 x (scale, minimum) in bf16
_WIDE_PAGE = 128        # tokens of a page that rows are widened to for prefill


def is_int4_cache(cache: torch.Tensor) -> bool:
    """One side of a 4-bit pool (an FP8 pool's uint8 codes have four dims)."""
    return cache.dtype == torch.uint8 and cache.dim() == 3


def int4_pool_shape(num_blocks: int, block_size: int, num_kv_heads: int):
    """Shape of one side of a 4-bit pool."""
    if block_size <= 0 or block_size % TILE_TOKENS:
        raise SlokvError(f"a 4-bit pool's block_size must be a multiple of {TILE_TOKENS}")
    return (num_blocks, num_kv_heads, block_size * ROW_BYTES)


def int4_geometry(k_cache: torch.Tensor, v_cache: torch.Tensor):
    """(num_blocks, block_size, num_kv_heads) of a 4-bit pool, checked."""
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not is_int4_cache(c):
            raise SlokvError(f"{name} must be a uint8 4-bit pool [num_blocks, num_kv_heads, "
                             f"block_size * {ROW_BYTES}]")
        if c.shape[2] == 0 or c.shape[2] % (TILE_TOKENS * ROW_BYTES):
            raise SlokvError(f"{name}: the last dim must be block_size * {ROW_BYTES} bytes, "
                             f"block_size a multiple of {TILE_TOKENS}")
        if c.stride(2) != 1 or (c.shape[1] > 1 and c.stride(1) != c.shape[2]):
            raise SlokvError(f"{name} blocks must be contiguous")
        if c.shape[0] > 1 and c.stride(0) < c.shape[1] * c.shape[2]:
            raise SlokvError(f"{name} blocks must not overlap")
    if v_cache.shape != k_cache.shape:
        raise SlokvError("k_cache and v_cache shapes differ")
    return k_cache.shape[0], k_cache.shape[2] // ROW_BYTES, k_cache.shape[1]


def _block_stride(c: torch.Tensor) -> int:
    return c.stride(0) if c.shape[0] > 1 else c.shape[1] * c.shape[2]


def store_kvcache_int4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Quantising store into the 4-bit pool (store_kvcache's counterpart).

    key / value: [N, Hkv, 128] bf16, f16 or fp32 (the same type), any row and head
    strides with a contiguous last dim (views of a fused qkv projection too);
    slot_mapping: [N] int32, -1 skips the token, the other slots distinct.
    """
    if key.dim() != 3 or value.shape != key.shape:
        raise SlokvError("key and value must be [tokens, heads, head_dim] of one shape")
    N, H, D = key.shape
    if D != HEAD_DIM:
        raise SlokvError(f"the 4-bit pool has head_dim {HEAD_DIM}, not {D}")
    if key.dtype != value.dtype or key.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise SlokvError("key and value must both be bf16, f16 or fp32")
    if key.stride(-1) != 1 or value.stride(-1) != 1:
        raise SlokvError("key and value need a contiguous last dimension")
    NB, bs, Hkv = int4_geometry(k_cache, v_cache)
    if Hkv != H:
        raise SlokvError(f"the pool has {Hkv} KV heads, key / value {H}")
    dev = require_cuda(key, value, k_cache, v_cache, slot_mapping)
    _i32_contig("slot_mapping", slot_mapping)
    if slot_mapping.numel() != N:
        raise SlokvError("slot_mapping must have one entry per token")
    if N == 0:
        return
    with torch.cuda.device(dev):
        check(lib().slokv_kv_append_int4(
            key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0),
            value.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), _block_stride(k_cache),
            _block_stride(v_cache), slot_mapping.data_ptr(), N, H, D, bs, NB,
            _lib.dtype_code(key.dtype), buffers.error_word(dev).data_ptr(), stream_ptr(dev)),
            "kv_append_int4")


def int4_decode(cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """fp32 values [N, Hkv, 128] of the rows at `slots` ([N] int32) of one side of a
    4-bit pool (e4m3_decode's counterpart); slot -1 gives zeros."""
    NB, bs, H = int4_geometry(cache, cache)
    dev = require_cuda(cache, slots)
    _i32_contig("slots", slots)
    out = torch.empty(slots.numel(), H, HEAD_DIM, dtype=torch.float32, device=dev)
    if slots.numel():
        with torch.cuda.device(dev):
            check(lib().slokv_int4_decode(
                cache.data_ptr(), _block_stride(cache), slots.data_ptr(), slots.numel(), H,
                HEAD_DIM, bs, NB, out.data_ptr(), buffers.error_word(dev).data_ptr(),
                stream_ptr(dev)), "int4_decode")
    return out


def check_decode_args(q, cache_seqlens, block_table, out, head_dim):
    """Argument checks that the paged decodes of this package's 4-bit and scored
    paths share; returns (batch, query heads, out)."""
    if q.dim() != 4 or q.shape[1] != 1 or q.shape[3] != head_dim:
        raise SlokvError(f"paged decode expects q of shape [batch, 1, heads, {head_dim}]")
    if q.dtype not in (torch.bfloat16, torch.float16) or q.stride(-1) != 1:
        raise SlokvError("q must be bf16 or f16 with a contiguous last dimension")
    B, _, Hq, _ = q.shape
    _i32_contig("cache_seqlens", cache_seqlens)
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(-1) != 1:
        raise SlokvError("block_table must be int32 [batch, pages] with a contiguous last dim")
    if block_table.shape[0] < B or cache_seqlens.numel() < B:
        raise SlokvError("block_table / cache_seqlens have fewer rows than q")
    if block_table.shape[1] == 0:
        raise SlokvError("block_table has no columns")
    if out is None:
        out = torch.empty(B, 1, Hq, head_dim, dtype=q.dtype, device=q.device)
    elif out.dtype != q.dtype or out.shape != q.shape or out.stride(-1) != 1 or not out.is_cuda:
        raise SlokvError("out must match q's shape, dtype and device with a contiguous last dim")
    return B, Hq, out


def _decode_int4(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, out,
                 logits=None, lse=None):
    NB, bs, Hkv = int4_geometry(k_cache, v_cache)
    dev = require_cuda(q, k_cache, v_cache, cache_seqlens, block_table, out)
    B, Hq, out = check_decode_args(q, cache_seqlens, block_table, out, HEAD_DIM)
    if B == 0:
        return out
    scale = float(softmax_scale) if softmax_scale is not None else HEAD_DIM ** -0.5
    with torch.cuda.device(dev):
        nbytes = lib().slokv_paged_decode_int4_workspace_bytes(-1, Hq, Hkv, HEAD_DIM)
        if nbytes == 0:
            raise SlokvError(f"unsupported 4-bit decode geometry Hq={Hq} Hkv={Hkv}")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        check(lib().slokv_paged_decode_int4(
            out.data_ptr(), out.stride(0), out.stride(2), q.data_ptr(), q.stride(0), q.stride(2),
            k_cache.data_ptr(), v_cache.data_ptr(), _block_stride(k_cache),
            _block_stride(v_cache), NB, bs, Hq, Hkv, HEAD_DIM, block_table.data_ptr(),
            block_table.stride(0), block_table.shape[1], cache_seqlens.data_ptr(), B, scale,
            _lib.dtype_code(q.dtype), None if logits is None else logits.data_ptr(),
            0 if logits is None else logits.stride(1), None if lse is None else lse.data_ptr(),
            ws.data_ptr(), nbytes, buffers.error_word(dev).data_ptr(), stream_ptr(dev)),
            "paged_decode_int4")
    return out


def flash_attn_with_kvcache_int4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                 cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                                 softmax_scale: float | None = None, causal: bool = True,
                                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Paged decode over the 4-bit pool (flash_attn_with_kvcache's counterpart).

    q: [B, 1, Hq, 128] bf16 or f16, at most 16 query heads per KV head, 4-byte
    aligned with even strides; cache_seqlens: [B] int32 including the token stored this
    step (0: the row's output is zero); block_table: [B, W] int32.
    """
    return _decode_int4(q, k_cache, v_cache, cache_seqlens, block_table, softmax_scale, out)


def flash_attn_varlen_func_int4(q, k_cache, v_cache, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
                                max_seqlen_k, softmax_scale=None, causal=True, block_table=None,
                                out=None):
    """Causal varlen attention over a 4-bit pool's pages (block_table required).

    Arguments as flash_attn_varlen_func's paged form, any block_size that the pool
    allows.  The rows' cached tokens are widened once to q's type (one rounding) in a
    scratch of rows x ceil(max_seqlen_k / 128) pages, which the tcgen05 prefill then
    reads: 16 times the prefill's own page reads at most when a chunk is a few
    tokens, a few per cent of its time when it is a thousand.
    """
    if block_table is None:
        raise SlokvError("4-bit varlen attention reads the pool: block_table is required")
    if not causal:
        raise SlokvError("only causal varlen attention is implemented (the engine's only use)")
    if q.dim() != 3 or q.shape[2] != HEAD_DIM or q.dtype not in (torch.bfloat16, torch.float16) \
            or q.stride(-1) != 1:
        raise SlokvError(f"q must be bf16/f16 [tokens, heads, {HEAD_DIM}] with a contiguous last "
                         "dim")
    NB, bs, Hkv = int4_geometry(k_cache, v_cache)
    dev = require_cuda(q, k_cache, v_cache, cu_seqlens_q, cu_seqlens_k, block_table, out)
    _i32_contig("cu_seqlens_q", cu_seqlens_q)
    _i32_contig("cu_seqlens_k", cu_seqlens_k)
    if cu_seqlens_k.numel() != cu_seqlens_q.numel():
        raise SlokvError("cu_seqlens_q and cu_seqlens_k differ in length")
    rows = cu_seqlens_q.numel() - 1
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(-1) != 1 \
            or block_table.shape[0] < rows:
        raise SlokvError("block_table must be int32 [rows, pages] with a contiguous last dim")
    if q.shape[1] % Hkv:
        raise SlokvError("query heads must divide by the KV heads")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype or out.shape != q.shape or out.stride(-1) != 1:
        raise SlokvError("out must match q's shape and dtype with a contiguous last dim")
    if q.shape[0] == 0 or rows <= 0 or int(max_seqlen_q) <= 0:
        return out
    pages = max(1, (int(max_seqlen_k) + _WIDE_PAGE - 1) // _WIDE_PAGE)
    with torch.cuda.device(dev):
        wide = torch.empty(2, rows * pages, _WIDE_PAGE, Hkv, HEAD_DIM, dtype=q.dtype, device=dev)
        table = torch.empty(rows, pages, dtype=torch.int32, device=dev)
        check(lib().slokv_int4_rows_widen(
            k_cache.data_ptr(), v_cache.data_ptr(), _block_stride(k_cache),
            _block_stride(v_cache), NB, bs, Hkv, HEAD_DIM, block_table.data_ptr(),
            block_table.stride(0), block_table.shape[1], cu_seqlens_k.data_ptr(), rows, pages,
            wide[0].data_ptr(), wide[1].data_ptr(), table.data_ptr(), _lib.dtype_code(q.dtype),
            buffers.error_word(dev).data_ptr(), stream_ptr(dev)), "int4_rows_widen")
        return _varlen_attention(q, wide[0], wide[1], cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
                                 softmax_scale, causal, table, out, None)
