"""Cache eviction by accumulated attention weight.

`flash_attn_with_kvcache_scored` is a paged decode that also adds each key's
attention weight, summed over the query heads of its KV head, to a score table;
`kv_evict` cuts sequences down to the tokens that are recent or have the highest
scores, separately for every KV head, in place in their own pages.

Scores are fp32 [rows, num_kv_heads, width], one row per sequence and one column per
cached position; a caller zeroes a row when a sequence takes it.  `score_rows` maps
the batch to rows (-1: not scored, for padding rows); without it batch row b uses
score row b.  A bf16 / f16 pool or a 4-bit one (kvcache_int4) is read; eviction
also takes fp32 pools.  FP8 pools are refused: their scale is shared by a block, so
a token cannot move to another block as it is.

After an eviction a sequence's cache length and the position of its next token are
two numbers: the next token is stored at slot new_len, with the rotary position
that it has in the text.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import SlokvError, buffers, check, lib, require_cuda, stream_ptr
from .kvcache import _i32_contig
from .kvcache_int4 import (HEAD_DIM, _block_stride, _decode_int4, check_decode_args,
                           int4_geometry, is_int4_cache)


def _check_scores(scores, score_rows, batch, num_kv_heads):
    if scores.dim() != 3 or scores.dtype != torch.float32 or scores.stride(-1) != 1:
        raise SlokvError("scores must be fp32 [rows, num_kv_heads, width] with a contiguous last "
                         "dim")
    if scores.shape[1] != num_kv_heads:
        raise SlokvError(f"scores have {scores.shape[1]} KV heads, the pool {num_kv_heads}")
    if score_rows is None:
        if scores.shape[0] < batch:
            raise SlokvError("scores have fewer rows than the batch")
    else:
        _i32_contig("score_rows", score_rows)
        if score_rows.numel() < batch:
            raise SlokvError("score_rows has fewer entries than the batch")


def _dense_geometry(k_cache, v_cache, dtypes):
    """(num_blocks, block_size, num_kv_heads) of an unquantised pool, checked."""
    if k_cache.dim() != 4 or k_cache.shape[3] != HEAD_DIM or v_cache.shape != k_cache.shape:
        raise SlokvError(f"k_cache / v_cache must be [num_blocks, block_size, Hkv, {HEAD_DIM}] of "
                         "one shape")
    if k_cache.dtype not in dtypes or v_cache.dtype != k_cache.dtype:
        raise SlokvError(f"k_cache / v_cache must both be one of {dtypes} (FP8 pools are not "
                         "supported)")
    NB, bs, Hkv, D = k_cache.shape
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.stride(3) != 1 or c.stride(2) != D or c.stride(1) != Hkv * D:
            raise SlokvError(f"{name} blocks must be contiguous [block_size, Hkv, D]")
    return NB, bs, Hkv


def flash_attn_with_kvcache_scored(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                   scores: torch.Tensor, cache_seqlens: torch.Tensor,
                                   block_table: torch.Tensor, max_seqlen_k: int | None = None,
                                   softmax_scale: float | None = None, causal: bool = True,
                                   decay: float = 1.0, score_rows: torch.Tensor | None = None,
                                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Paged decode that accumulates attention weights.

    As flash_attn_with_kvcache (bf16 / f16 pool) or flash_attn_with_kvcache_int4, and
      scores[row, h, t] = decay * scores[row, h, t] + sum over h's query heads of softmax[t]
    for every cached position t of each sequence.  decay 1 accumulates, decay 0
    overwrites with this step's weights.  max_seqlen_k (default: scores' width) bounds
    the context lengths: it sizes the [B, Hq, max_seqlen_k] fp32 scratch, and positions
    past it or past scores' width are not scored (device error CONTEXT_LEN).  Two
    sequences of one call must not share a score row; shared blocks are fine.
    """
    four = is_int4_cache(k_cache)
    if four:
        NB, bs, Hkv = int4_geometry(k_cache, v_cache)
    else:
        NB, bs, Hkv = _dense_geometry(k_cache, v_cache, (torch.bfloat16, torch.float16))
        if q.dtype != k_cache.dtype:
            raise SlokvError("q and cache dtypes differ")
    dev = require_cuda(q, k_cache, v_cache, scores, cache_seqlens, block_table, score_rows, out)
    B, Hq, out = check_decode_args(q, cache_seqlens, block_table, out, HEAD_DIM)
    _check_scores(scores, score_rows, B, Hkv)
    if Hq % Hkv:
        raise SlokvError("query heads must divide by the KV heads")
    if B == 0:
        return out
    width = scores.shape[2] if max_seqlen_k is None else min(int(max_seqlen_k), scores.shape[2])
    if width <= 0:
        raise SlokvError("scores have no columns (or max_seqlen_k is not positive)")
    scale = float(softmax_scale) if softmax_scale is not None else HEAD_DIM ** -0.5
    with torch.cuda.device(dev):
        stride = (width + 3) // 4 * 4
        logits = torch.empty(B, Hq, stride, dtype=torch.float32, device=dev)
        lse = torch.empty(B, Hq, dtype=torch.float32, device=dev)
        err, stream = buffers.error_word(dev).data_ptr(), stream_ptr(dev)
        if four:
            _decode_int4(q, k_cache, v_cache, cache_seqlens, block_table, scale, out, logits, lse)
        else:
            nbytes = lib().slokv_paged_decode_workspace_bytes(-1, Hq, Hkv, HEAD_DIM)
            ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
            check(lib().slokv_paged_decode_logits(
                out.data_ptr(), out.stride(0), out.stride(2), q.data_ptr(), q.stride(0),
                q.stride(2), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0),
                v_cache.stride(0), NB, bs, Hq, Hkv, HEAD_DIM, block_table.data_ptr(),
                block_table.stride(0), block_table.shape[1], cache_seqlens.data_ptr(), B, scale,
                _lib.dtype_code(q.dtype), logits.data_ptr(), stride, lse.data_ptr(),
                ws.data_ptr(), nbytes, err, stream), "paged_decode_logits")
        check(lib().slokv_kv_scores_accumulate(
            scores.data_ptr(), scores.stride(0), scores.stride(1), width, scores.shape[0],
            None if score_rows is None else score_rows.data_ptr(), logits.data_ptr(), stride,
            lse.data_ptr(), cache_seqlens.data_ptr(), B, Hq, Hkv, block_table.shape[1] * bs,
            float(decay), err, stream), "kv_scores_accumulate")
    return out


def kv_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, scores: torch.Tensor,
             cache_seqlens: torch.Tensor, block_table: torch.Tensor, keep: int, recent: int,
             score_rows: torch.Tensor | None = None, return_index: bool = False):
    """Cut every sequence longer than `keep` tokens to `keep`, in place.

    Per sequence and KV head the last `recent` tokens stay, and of the others the
    keep - recent of the highest score (ties: the lowest position; NaN counts as -inf).
    Kept tokens below position keep stay in their slots; the others move, in order,
    into the freed slots below it, with their scores, and the rest of the score row is
    zeroed.  Returns the new lengths ([B] int32) and, with return_index, the position
    that each slot's token came from ([B, Hkv, keep] int32, -1 past the new length).

    The pages below position keep must belong to one sequence each (kv_block_copy
    shared ones first); those past it can be freed afterwards.
    """
    keep, recent = int(keep), int(recent)
    if keep < 1 or recent < 0 or recent > keep:
        raise SlokvError("kv_evict needs keep >= 1 and 0 <= recent <= keep")
    if is_int4_cache(k_cache):
        NB, bs, Hkv = int4_geometry(k_cache, v_cache)
        dtype, strides = _lib.DTYPE_INT4, (_block_stride(k_cache), _block_stride(v_cache))
    else:
        NB, bs, Hkv = _dense_geometry(k_cache, v_cache,
                                      (torch.bfloat16, torch.float16, torch.float32))
        es = k_cache.element_size()
        dtype = _lib.dtype_code(k_cache.dtype)
        strides = (k_cache.stride(0) * es, v_cache.stride(0) * es)
    dev = require_cuda(k_cache, v_cache, scores, cache_seqlens, block_table, score_rows)
    _i32_contig("cache_seqlens", cache_seqlens)
    B = cache_seqlens.numel()
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(-1) != 1 \
            or block_table.shape[0] < B or block_table.shape[1] == 0:
        raise SlokvError("block_table must be int32 [batch, pages] with a contiguous last dim")
    _check_scores(scores, score_rows, B, Hkv)
    new_lens = torch.empty(B, dtype=torch.int32, device=dev)
    index = torch.empty(B, Hkv, keep, dtype=torch.int32, device=dev) if return_index else None
    if B:
        with torch.cuda.device(dev):
            nbytes = lib().slokv_kv_evict_workspace_bytes(B, Hkv, keep, scores.shape[2])
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            check(lib().slokv_kv_evict(
                k_cache.data_ptr(), v_cache.data_ptr(), *strides, NB, bs, Hkv, HEAD_DIM, dtype,
                block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                cache_seqlens.data_ptr(), B, scores.data_ptr(), scores.stride(0),
                scores.stride(1), scores.shape[2], scores.shape[0],
                None if score_rows is None else score_rows.data_ptr(), keep, recent,
                new_lens.data_ptr(), None if index is None else index.data_ptr(), ws.data_ptr(),
                nbytes, buffers.error_word(dev).data_ptr(), stream_ptr(dev)), "kv_evict")
    return (new_lens, index) if return_index else new_lens
