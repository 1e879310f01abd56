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
from ._lib import SlokvError, buffers, check, lib, on_device, require_cuda
from .kvcache import _i32_contig
from .kvcache_int4 import (HEAD_DIM, check_decode_args, decode_int4_workspace_bytes, int4_geometry,
                           is_int4_cache, launch_decode_int4)


def _check_scores(scores, score_rows, batch, num_kv_heads):
    """(rows, width, row stride, head stride, score_rows' address) of a score table."""
    if scores.dim() != 3 or scores.dtype != torch.float32:
        raise SlokvError("scores must be fp32 [rows, num_kv_heads, width]")
    rows, heads, width = scores.shape
    row, head, one = scores.stride()
    if one != 1:
        raise SlokvError("scores need a contiguous last dimension")
    if heads != num_kv_heads:
        raise SlokvError(f"scores have {heads} KV heads, the pool {num_kv_heads}")
    if score_rows is None:
        if rows < batch:
            raise SlokvError("scores have fewer rows than the batch")
        return rows, width, row, head, None
    _i32_contig("score_rows", score_rows)
    if score_rows.numel() < batch:
        raise SlokvError("score_rows has fewer entries than the batch")
    return rows, width, row, head, score_rows.data_ptr()


def _dense_geometry(k_cache, v_cache, dtypes):
    """(num_blocks, block_size, num_kv_heads, K and V block strides in elements) of an
    unquantised pool, checked."""
    if k_cache.dim() != 4 or k_cache.shape[3] != HEAD_DIM or v_cache.shape != k_cache.shape:
        raise SlokvError(f"k_cache / v_cache must be [num_blocks, block_size, Hkv, {HEAD_DIM}] of "
                         "one shape")
    if k_cache.dtype not in dtypes or v_cache.dtype != k_cache.dtype:
        raise SlokvError(f"k_cache / v_cache must both be one of {list(dtypes)} (FP8 pools are not "
                         "supported)")
    NB, bs, Hkv, D = k_cache.shape
    ks, vs = k_cache.stride(), v_cache.stride()
    if ks[1:] != (Hkv * D, D, 1) or vs[1:] != (Hkv * D, D, 1):
        raise SlokvError("k_cache / v_cache blocks must be contiguous [block_size, Hkv, D]")
    return NB, bs, Hkv, ks[0], vs[0]


_DECODE_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_EVICT_DTYPES = {**_DECODE_DTYPES, torch.float32: _lib.DTYPE_F32}
_workspace_bytes = {}   # (device, Hq, Hkv) -> bytes of the bf16 / f16 decode


def _decode_workspace_bytes(index, num_q_heads, num_kv_heads):
    key = (index, num_q_heads, num_kv_heads)
    n = _workspace_bytes.get(key)
    if n is None:
        n = lib().slokv_paged_decode_workspace_bytes(index, num_q_heads, num_kv_heads, HEAD_DIM)
        if n == 0:
            raise SlokvError(f"unsupported decode geometry Hq={num_q_heads} Hkv={num_kv_heads}")
        _workspace_bytes[key] = n
    return n


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
    the context lengths: positions past it or past scores' width are not scored (device
    error CONTEXT_LEN).  The scratch is fp32 [B, Hq, min(max_seqlen_k, the block table's
    reach)].  Two sequences of one call must not share a score row; shared blocks are fine.
    """
    four = is_int4_cache(k_cache)
    if four:
        pool = int4_geometry(k_cache, v_cache)
    else:
        pool = _dense_geometry(k_cache, v_cache, _DECODE_DTYPES)
        if q.dtype != k_cache.dtype:
            raise SlokvError("q and cache dtypes differ")
    NB, bs, Hkv, k_block, v_block = pool
    dev = require_cuda(q, k_cache, v_cache, scores, cache_seqlens, block_table, score_rows, out)
    B, Hq, out = check_decode_args(q, cache_seqlens, block_table, out)
    rows, width, row, head, rows_ptr = _check_scores(scores, score_rows, B, Hkv)
    if Hq % Hkv:
        raise SlokvError("query heads must divide by the KV heads")
    if B == 0:
        return out
    if max_seqlen_k is not None:
        width = min(int(max_seqlen_k), width)
    if width <= 0:
        raise SlokvError("scores have no columns (or max_seqlen_k is not positive)")
    scale = HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale)
    reach = block_table.shape[1] * bs
    stride = (min(width, reach) + 3) // 4 * 4
    with on_device(dev) as stream:
        nbytes = (decode_int4_workspace_bytes if four else _decode_workspace_bytes)(dev.index, Hq,
                                                                                    Hkv)
        # one scratch: the decode's workspace, the scores of this step, their denominators
        logits_at = (nbytes + 255) // 256 * 256
        # (the 4-bit decode stores a KV head's heads side by side, padded to pairs)
        heads = Hkv * ((Hq // Hkv + 1) // 2 * 2) if four else Hq
        lse_at = logits_at + 4 * B * heads * stride
        scratch = torch.empty(lse_at + 4 * B * Hq, dtype=torch.uint8, device=dev)
        ws = scratch.data_ptr()
        logits, lse, err = ws + logits_at, ws + lse_at, buffers.error_word(dev).data_ptr()
        if four:
            launch_decode_int4(q, k_cache, v_cache, pool, cache_seqlens.data_ptr(), block_table,
                               scale, B, Hq, out, ws, nbytes, err, stream, logits, stride, lse)
        else:
            qs, os = q.stride(), out.stride()
            check(lib().slokv_paged_decode_logits(
                out.data_ptr(), os[0], os[2], q.data_ptr(), qs[0], qs[2], k_cache.data_ptr(),
                v_cache.data_ptr(), k_block, v_block, NB, bs, Hq, Hkv, HEAD_DIM,
                block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                cache_seqlens.data_ptr(), B, scale, _DECODE_DTYPES[q.dtype], logits, stride, lse, ws,
                nbytes, err, stream), "paged_decode_logits")
        check(lib().slokv_kv_scores_accumulate(
            scores.data_ptr(), row, head, width, rows, rows_ptr, logits, stride, int(four), lse,
            cache_seqlens.data_ptr(), B, Hq, Hkv, reach, float(decay), err, stream),
            "kv_scores_accumulate")
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

    The pages below position keep and the score rows must belong to one sequence each
    (kv_block_copy shared pages first); the pages past it can be freed afterwards.
    """
    keep, recent = int(keep), int(recent)
    if not 1 <= keep < 2 ** 31 or not 0 <= recent <= keep:
        raise SlokvError("kv_evict needs 1 <= keep < 2^31 and 0 <= recent <= keep")
    if is_int4_cache(k_cache):
        NB, bs, Hkv, k_block, v_block = int4_geometry(k_cache, v_cache)
        dtype = _lib.DTYPE_INT4
    else:
        NB, bs, Hkv, k_block, v_block = _dense_geometry(k_cache, v_cache, _EVICT_DTYPES)
        dtype, es = _EVICT_DTYPES[k_cache.dtype], k_cache.element_size()
        k_block, v_block = k_block * es, v_block * es
    dev = require_cuda(k_cache, v_cache, scores, cache_seqlens, block_table, score_rows)
    _i32_contig("cache_seqlens", cache_seqlens)
    B = cache_seqlens.numel()
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(1) != 1 \
            or block_table.shape[0] < B or block_table.shape[1] == 0:
        raise SlokvError("block_table must be int32 [batch, pages] with a contiguous last dim")
    rows, width, row, head, rows_ptr = _check_scores(scores, score_rows, B, Hkv)
    new_lens = torch.empty(B, dtype=torch.int32, device=dev)
    index = torch.empty(B, Hkv, keep, dtype=torch.int32, device=dev) if return_index else None
    if B:
        with on_device(dev) as stream:
            nbytes = lib().slokv_kv_evict_workspace_bytes(B, Hkv, keep, width)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            check(lib().slokv_kv_evict(
                k_cache.data_ptr(), v_cache.data_ptr(), k_block, v_block, NB, bs, Hkv, HEAD_DIM,
                dtype, block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                cache_seqlens.data_ptr(), B, scores.data_ptr(), row, head, width, rows, rows_ptr,
                keep, recent, new_lens.data_ptr(), None if index is None else index.data_ptr(),
                ws.data_ptr(), nbytes, buffers.error_word(dev).data_ptr(), stream), "kv_evict")
    return (new_lens, index) if return_index else new_lens
