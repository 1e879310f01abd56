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
from ._lib import SlokvError, buffers, check, lib, on_device, require_cuda
from .kvcache import _i32_contig

HEAD_DIM = 128
TILE_TOKENS = 64
ROW_BYTES = 72          # 64 bytes of codes, 2 x (scale, minimum) in bf16
_WIDE_PAGE = 128        # tokens of a page that rows are widened to for prefill
_WIDE_BYTES = 1 << 30   # scratch of widened rows; more rows than fit run in groups

# A prefill call of at most SHORT_CHUNK query tokens a row, or SHORT_CALL in all, runs as
# decode rows (8 KV heads of 4, us, prefill / decode rows, L cached tokens: 1 row of 64
# on L 4000 82 / 63, of 128 79 / 110; 8 rows of 16 115 / 109, of 32 113 / 202; 64 rows
# of 4 793 / 204, of 16 783 / 783).
SHORT_CHUNK, SHORT_CALL = 16, 64
_MAX_DECODE_ROWS, _MAX_GROUP = 8192, 16   # of the decode kernel

_Q_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_STORE_DTYPES = {**_Q_DTYPES, torch.float32: _lib.DTYPE_F32}


def is_int4_cache(cache: torch.Tensor) -> bool:
    """One side of a 4-bit pool (an FP8 pool's uint8 codes have four dims)."""
    return cache.dtype == torch.uint8 and cache.dim() == 3


def int4_pool_shape(num_blocks: int, block_size: int, num_kv_heads: int):
    """Shape of one side of a 4-bit pool."""
    if block_size <= 0 or block_size % TILE_TOKENS:
        raise SlokvError(f"a 4-bit pool's block_size must be a multiple of {TILE_TOKENS}")
    return (num_blocks, num_kv_heads, block_size * ROW_BYTES)


def int4_geometry(k_cache: torch.Tensor, v_cache: torch.Tensor):
    """(num_blocks, block_size, num_kv_heads, K and V block strides in bytes) of a 4-bit
    pool, checked."""
    shape = k_cache.shape
    if v_cache.shape != shape:
        raise SlokvError("k_cache and v_cache shapes differ")
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8 or len(shape) != 3:
        raise SlokvError("k_cache / v_cache must be uint8 4-bit pools [num_blocks, "
                         f"num_kv_heads, block_size * {ROW_BYTES}]")
    nb, h, size = shape
    if size == 0 or size % (TILE_TOKENS * ROW_BYTES):
        raise SlokvError(f"a 4-bit pool's last dim must be block_size * {ROW_BYTES} bytes, "
                         f"block_size a multiple of {TILE_TOKENS}")
    k_block, k_head, k_one = k_cache.stride()
    v_block, v_head, v_one = v_cache.stride()
    if k_one != 1 or v_one != 1 or (h > 1 and (k_head != size or v_head != size)):
        raise SlokvError("a 4-bit pool's blocks must be contiguous")
    run = h * size
    if nb <= 1:
        k_block = v_block = run
    elif k_block < run or v_block < run:
        raise SlokvError("a 4-bit pool's blocks must not overlap")
    return nb, size // ROW_BYTES, h, k_block, v_block


def store_kvcache_int4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Quantising store into the 4-bit pool (store_kvcache's counterpart).

    key / value: [N, Hkv, 128] bf16, f16 or fp32 (the same type), any row and head
    strides with a contiguous last dim (views of a fused qkv projection too);
    slot_mapping: [N] int32, -1 skips the token, the other slots distinct.

    A value comes back within half a step (a fifteenth of its group's range, rounded), but
    f16 and fp32 groups whose |min| is more than 7 times their range come back within
    2^-8 (|min| + range): their minimum is kept in bf16.
    """
    if key.dim() != 3 or value.shape != key.shape:
        raise SlokvError("key and value must be [tokens, heads, head_dim] of one shape")
    N, H, D = key.shape
    if D != HEAD_DIM:
        raise SlokvError(f"the 4-bit pool has head_dim {HEAD_DIM}, not {D}")
    dtype = key.dtype
    if value.dtype != dtype or dtype not in _STORE_DTYPES:
        raise SlokvError("key and value must both be bf16, f16 or fp32")
    k_row, k_head, k_one = key.stride()
    v_row, v_head, v_one = value.stride()
    if k_one != 1 or v_one != 1:
        raise SlokvError("key and value need a contiguous last dimension")
    NB, bs, Hkv, k_block, v_block = int4_geometry(k_cache, v_cache)
    if Hkv != H:
        raise SlokvError(f"the pool has {Hkv} KV heads, key / value {H}")
    dev = require_cuda(key, value, k_cache, v_cache, slot_mapping)
    _i32_contig("slot_mapping", slot_mapping)
    if slot_mapping.numel() != N:
        raise SlokvError("slot_mapping must have one entry per token")
    if N == 0:
        return
    with on_device(dev) as stream:
        check(lib().slokv_kv_append_int4(
            key.data_ptr(), k_row, k_head, value.data_ptr(), v_row, v_head, k_cache.data_ptr(),
            v_cache.data_ptr(), k_block, v_block, slot_mapping.data_ptr(), N, H, D, bs, NB,
            _STORE_DTYPES[dtype], buffers.error_word(dev).data_ptr(), stream), "kv_append_int4")


def int4_decode(cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """fp32 values [N, Hkv, 128] of the rows at `slots` ([N] int32) of one side of a
    4-bit pool (e4m3_decode's counterpart); slot -1 gives zeros."""
    NB, bs, H, block, _ = int4_geometry(cache, cache)
    dev = require_cuda(cache, slots)
    _i32_contig("slots", slots)
    n = slots.numel()
    out = torch.empty(n, H, HEAD_DIM, dtype=torch.float32, device=dev)
    if n:
        with on_device(dev) as stream:
            check(lib().slokv_int4_decode(
                cache.data_ptr(), block, slots.data_ptr(), n, H, HEAD_DIM, bs, NB, out.data_ptr(),
                buffers.error_word(dev).data_ptr(), stream), "int4_decode")
    return out


def check_decode_args(q, cache_seqlens, block_table, out):
    """Argument checks that the paged decodes of this package's 4-bit and scored
    paths share; returns (batch, query heads, out)."""
    shape, dtype = q.shape, q.dtype
    if len(shape) != 4 or shape[1] != 1 or shape[3] != HEAD_DIM:
        raise SlokvError(f"paged decode expects q of shape [batch, 1, heads, {HEAD_DIM}]")
    B, Hq = shape[0], shape[2]
    if dtype not in _Q_DTYPES or q.stride(3) != 1:
        raise SlokvError("q must be bf16 or f16 with a contiguous last dimension")
    _i32_contig("cache_seqlens", cache_seqlens)
    table = block_table.shape
    if len(table) != 2 or block_table.dtype != torch.int32 or block_table.stride(1) != 1:
        raise SlokvError("block_table must be int32 [batch, pages] with a contiguous last dim")
    rows, width = table
    if rows < B or cache_seqlens.numel() < B:
        raise SlokvError("block_table / cache_seqlens have fewer rows than q")
    if width == 0:
        raise SlokvError("block_table has no columns")
    if out is None:
        out = torch.empty(B, 1, Hq, HEAD_DIM, dtype=dtype, device=q.device)
    elif out.dtype != dtype or out.shape != shape or out.stride(3) != 1:
        raise SlokvError("out must match q's shape and dtype with a contiguous last dim")
    return B, Hq, out


_workspace_bytes = {}   # (device, Hq, Hkv) -> bytes: a property of the device


def decode_int4_workspace_bytes(index: int, num_q_heads: int, num_kv_heads: int) -> int:
    key = (index, num_q_heads, num_kv_heads)
    n = _workspace_bytes.get(key)
    if n is None:
        n = lib().slokv_paged_decode_int4_workspace_bytes(index, num_q_heads, num_kv_heads,
                                                          HEAD_DIM)
        if n == 0:
            raise SlokvError(f"unsupported 4-bit decode geometry Hq={num_q_heads} "
                             f"Hkv={num_kv_heads}")
        _workspace_bytes[key] = n
    return n


def launch_decode_int4(q, k_cache, v_cache, pool, lens, block_table, scale, B, Hq, out, workspace,
                       nbytes, err, stream, logits=None, logits_stride=0, lse=None,
                       table_rows=None):
    """slokv_paged_decode_int4 on checked arguments; lens, workspace, logits, lse and
    table_rows are addresses; q / out [B, ..., Hq, 128]."""
    NB, bs, Hkv, k_block, v_block = pool
    qs, os = q.stride(), out.stride()
    check(lib().slokv_paged_decode_int4(
        out.data_ptr(), os[0], os[-2], q.data_ptr(), qs[0], qs[-2], k_cache.data_ptr(),
        v_cache.data_ptr(), k_block, v_block, NB, bs, Hq, Hkv, HEAD_DIM, block_table.data_ptr(),
        block_table.stride(0), block_table.shape[1], table_rows, lens, B, scale,
        _Q_DTYPES[q.dtype], logits, logits_stride, lse, workspace, nbytes, err, stream),
        "paged_decode_int4")


def flash_attn_with_kvcache_int4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                 cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                                 softmax_scale: float | None = None, causal: bool = True,
                                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Paged decode over the 4-bit pool (flash_attn_with_kvcache's counterpart).

    q: [B, 1, Hq, 128] bf16 or f16, at most 16 query heads per KV head, 4-byte
    aligned with even strides; cache_seqlens: [B] int32 including the token stored this
    step (0: the row's output is zero); block_table: [B, W] int32.
    """
    pool = int4_geometry(k_cache, v_cache)
    dev = require_cuda(q, k_cache, v_cache, cache_seqlens, block_table, out)
    B, Hq, out = check_decode_args(q, cache_seqlens, block_table, out)
    if B == 0:
        return out
    scale = HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale)
    with on_device(dev) as stream:
        nbytes = decode_int4_workspace_bytes(dev.index, Hq, pool[2])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        launch_decode_int4(q, k_cache, v_cache, pool, cache_seqlens.data_ptr(), block_table, scale,
                           B, Hq, out, ws.data_ptr(), nbytes, buffers.error_word(dev).data_ptr(), stream)
    return out


def _rows_on(x: torch.Tensor, align: int) -> bool:
    """Whether every (token, head) row of x, bf16 or f16, begins on a multiple of `align` bytes."""
    row, head, _ = x.stride()
    return not (x.data_ptr() | row * 2 | head * 2) & (align - 1)


def flash_attn_varlen_func_int4(q, k_cache, v_cache, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
                                max_seqlen_k, softmax_scale=None, causal=True, block_table=None,
                                out=None):
    """Causal varlen attention over a 4-bit pool's pages (block_table required).

    Arguments as flash_attn_varlen_func's paged form, any block_size that the pool
    allows.  q and out may be views at any address and stride with a contiguous last dim:
    one that the call's kernel does not take (short calls: rows on 4 bytes, others: on 16)
    goes through a contiguous copy.

    Short calls (SHORT_CHUNK, SHORT_CALL) run as decode rows, one a query token.  For
    longer ones the rows' cached tokens are widened once to q's type (one rounding; f16
    queries on a pool with values past f16's range, which no f16 rows leave in it, get
    infinities and the device error NONFINITE) in a scratch of at most 1 GiB (or one row
    of max_seqlen_k tokens), as many rows at a time as fit, which the tcgen05 prefill then
    reads: a few per cent of its time when a chunk is a thousand tokens.  There, as in
    flash_attn_varlen_func, a V row that is not finite (the store flags it) also reaches
    the queries of its 128-key tile that come before it.
    """
    if block_table is None:
        raise SlokvError("4-bit varlen attention reads the pool: block_table is required")
    if not causal:
        raise SlokvError("only causal varlen attention is implemented (the engine's only use)")
    if q.dim() != 3 or q.shape[2] != HEAD_DIM or q.dtype not in (torch.bfloat16, torch.float16) \
            or q.stride(-1) != 1:
        raise SlokvError(f"q must be bf16/f16 [tokens, heads, {HEAD_DIM}] with a contiguous last "
                         "dim")
    pool = int4_geometry(k_cache, v_cache)
    NB, bs, Hkv, k_block, v_block = pool
    dev = require_cuda(q, k_cache, v_cache, cu_seqlens_q, cu_seqlens_k, block_table, out)
    _i32_contig("cu_seqlens_q", cu_seqlens_q)
    _i32_contig("cu_seqlens_k", cu_seqlens_k)
    if cu_seqlens_k.numel() != cu_seqlens_q.numel():
        raise SlokvError("cu_seqlens_q and cu_seqlens_k differ in length")
    rows = cu_seqlens_q.numel() - 1
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(-1) != 1 \
            or block_table.shape[0] < rows:
        raise SlokvError("block_table must be int32 [rows, pages] with a contiguous last dim")
    Tq, Hq, _ = q.shape
    if Hq % Hkv:
        raise SlokvError("query heads must divide by the KV heads")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype or out.shape != q.shape or out.stride(-1) != 1:
        raise SlokvError("out must match q's shape and dtype with a contiguous last dim")
    max_seqlen_q, max_seqlen_k = int(max_seqlen_q), int(max_seqlen_k)
    if Tq == 0 or rows <= 0 or max_seqlen_q <= 0:
        return out
    if block_table.shape[1] == 0:
        raise SlokvError("block_table has no columns")
    short = ((max_seqlen_q <= SHORT_CHUNK or Tq <= SHORT_CALL) and Tq <= _MAX_DECODE_ROWS
             and Hq // Hkv <= _MAX_GROUP
             and Tq * Hkv * block_table.shape[1] * (bs // TILE_TOKENS) < 2 ** 31)
    if not _rows_on(q, 4 if short else 16):
        q = q.clone(memory_format=torch.contiguous_format)
    if not _rows_on(out, 4 if short else 16):
        # (a copy with out's content, since tokens of no row keep it)
        res = out.clone(memory_format=torch.contiguous_format)
        flash_attn_varlen_func_int4(q, k_cache, v_cache, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
                                    max_seqlen_k, softmax_scale, causal, block_table, res)
        return out.copy_(res)
    if short:
        scale = HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale)
        with on_device(dev) as stream:
            nbytes = decode_int4_workspace_bytes(dev.index, Hq, Hkv)
            ws = torch.empty(nbytes + 8 * Tq, dtype=torch.uint8, device=dev)
            table_rows, lens = ws.data_ptr() + nbytes, ws.data_ptr() + nbytes + 4 * Tq
            check(lib().slokv_int4_rows_expand(cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
                                               rows, Tq, table_rows, lens, stream),
                  "int4_rows_expand")
            launch_decode_int4(q, k_cache, v_cache, pool, lens, block_table, scale, Tq, Hq, out,
                               ws.data_ptr(), nbytes, buffers.error_word(dev).data_ptr(), stream,
                               table_rows=table_rows)
        return out
    pages = max(1, (max_seqlen_k + _WIDE_PAGE - 1) // _WIDE_PAGE)
    scale = HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale)
    dtype, err = _Q_DTYPES[q.dtype], buffers.error_word(dev).data_ptr()
    row_bytes = 2 * pages * _WIDE_PAGE * Hkv * HEAD_DIM * q.element_size()
    group = min(rows, max(1, _WIDE_BYTES // row_bytes))
    with on_device(dev) as stream:
        wide = torch.empty(2, group * pages, _WIDE_PAGE, Hkv, HEAD_DIM, dtype=q.dtype, device=dev)
        order = lib().slokv_paged_prefill_workspace_bytes(group, max_seqlen_q)
        scratch = torch.empty(4 * group * pages + order + 256, dtype=torch.uint8, device=dev)
        k_wide, v_wide, block = wide[0].data_ptr(), wide[1].data_ptr(), wide.stride(1)
        work = (scratch.data_ptr() + 255) // 256 * 256
        table = work + order
        for r in range(0, rows, group):      # several groups of rows share the scratch in turn
            n = min(group, rows - r)
            cu_q, cu_k = cu_seqlens_q.data_ptr() + 4 * r, cu_seqlens_k.data_ptr() + 4 * r
            check(lib().slokv_int4_rows_widen(
                k_cache.data_ptr(), v_cache.data_ptr(), k_block, v_block, NB, bs, Hkv, HEAD_DIM,
                block_table.data_ptr() + 4 * r * block_table.stride(0), block_table.stride(0),
                block_table.shape[1], cu_k, n, pages, k_wide, v_wide, table, dtype, err, stream),
                "int4_rows_widen")
            check(lib().slokv_paged_prefill(
                out.data_ptr(), out.stride(0), out.stride(1), q.data_ptr(), q.stride(0),
                q.stride(1), Tq, k_wide, v_wide, 0, 0, 0, block, block, cu_q, cu_k, n,
                max_seqlen_q, table, pages, pages, group * pages, _WIDE_PAGE, Hq, Hkv, HEAD_DIM,
                scale, dtype, None, work, order, err, stream), "paged_prefill")
    return out
