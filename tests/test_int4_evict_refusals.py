"""Refusals of the 4-bit and eviction entry points that need no GPU: the C ABI's argument
checks and the Python checks that come before any device work."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(256)


def test_append_int4_arguments(pkg):
    lib = pkg._lib.lib()

    def call(n=4, h=2, d=128, bs=64, nb=3, dt=0, ptr=P, pool=P, stride=2 * 64 * 72):
        return lib.slokv_kv_append_int4(ptr, 256, 128, ptr, 256, 128, pool, pool, stride, stride, ptr,
                                        n, h, d, bs, nb, dt, None, None)
    assert call(n=0) == 0
    assert call(n=-1) == -1 and call(h=0) == -1 and call(nb=0) == -1 and call(bs=0) == -1
    assert call(d=64) == -3 and call(bs=96) == -3 and call(dt=3) == -3 and call(dt=9) == -3
    assert call(ptr=None) == -1 and call(pool=None) == -1
    assert call(stride=2 * 64 * 72 + 8) == -2              # 16-byte block strides
    assert call(stride=64 * 72) == -2                      # blocks that overlap
    assert call(pool=ctypes.c_void_p(264)) == -2
    assert call(ptr=ctypes.c_void_p(257)) == -2            # an odd address of a 2-byte type


def test_decode_rows_and_widen_arguments(pkg):
    lib = pkg._lib.lib()

    def rows(n=4, d=128, bs=64, out=P, cache=P):
        return lib.slokv_int4_decode(cache, 2 * 64 * 72, P, n, 2, d, bs, 3, out, None, None)
    assert rows(n=0) == 0 and rows(n=-1) == -1
    assert rows(d=64) == -3 and rows(bs=100) == -3
    assert rows(out=None) == -1 and rows(out=ctypes.c_void_p(260)) == -2 and rows(cache=None) == -1

    def widen(r=2, pages=2, d=128, bs=64, dt=0, dst=P, w=4):
        return lib.slokv_int4_rows_widen(P, P, 2 * 64 * 72, 2 * 64 * 72, 3, bs, 2, d, P, 4, w, P, r,
                                         pages, dst, dst, P, dt, None, None)
    assert widen(r=0) == 0 and widen(pages=0) == 0
    assert widen(r=-1) == -1 and widen(d=64) == -3 and widen(bs=32) == -3 and widen(dt=2) == -3
    assert widen(dst=None) == -1 and widen(w=0) == -1 and widen(dst=ctypes.c_void_p(264)) == -2


def test_decode_int4_arguments(pkg):
    lib = pkg._lib.lib()

    def call(hq=8, hkv=2, d=128, bs=64, dt=0, batch=3, q=P, cache=P, stride=2 * 64 * 72, osb=1024,
             logits=None, lse=None, ls=0, w=4):
        return lib.slokv_paged_decode_int4(P, osb, 128, q, 1024, 128, cache, cache, stride, stride, 3, bs,
                                           hq, hkv, d, P, 4, w, None, P, batch, 0.1, dt, logits, ls,
                                           lse, None, 0, None, None)
    assert call(batch=0) == 0 and call(batch=-1) == -1
    assert call(batch=8193) == -3 and call(d=64) == -3 and call(dt=2) == -3
    assert call(hq=7) == -1 and call(hq=34) == -3 and call(bs=96) == -3
    assert call(q=None) == -1 and call(w=0) == -1
    assert call(logits=P) == -1 and call(logits=P, lse=P, ls=0) == -1
    assert call(cache=ctypes.c_void_p(264)) == -2 and call(stride=2 * 64 * 72 + 4) == -2
    assert call(q=ctypes.c_void_p(258)) == -2 and call(osb=1023) == -2
    assert call(logits=ctypes.c_void_p(260), lse=P, ls=64) == -2
    ex = lambda r=1, t=1, a=P: lib.slokv_int4_rows_expand(a, P, r, t, P, P, None)
    assert ex(r=0) == 0 and ex(t=0) == 0 and ex(r=-1) == -1 and ex(t=-1) == -1 and ex(a=None) == -1
    assert lib.slokv_paged_decode_int4_workspace_bytes(0, 7, 2, 128) == 0
    assert lib.slokv_paged_decode_int4_workspace_bytes(0, 8, 2, 64) == 0
    assert lib.slokv_paged_decode_int4_workspace_bytes(0, 34, 2, 128) == 0


def test_logits_and_scores_arguments(pkg):
    lib = pkg._lib.lib()

    def logits(lg=P, lse=P, ls=64, dt=0):
        return lib.slokv_paged_decode_logits(P, 1024, 128, P, 1024, 128, P, P, 32768, 32768, 3, 64, 8, 2,
                                             128, P, 4, 4, P, 3, 0.1, dt, lg, ls, lse, None, 0, None, None)
    assert logits(lg=None) == -1 and logits(lse=None) == -1 and logits(ls=0) == -1
    assert logits(ls=66) == -2 and logits(lg=ctypes.c_void_p(264)) == -2
    assert logits(dt=2) == -3                              # fp32 pools are not scored
    assert logits(dt=3) == -3

    def acc(batch=2, hq=8, hkv=2, width=64, scores=P, rows=2, cap=256, ls=64):
        return lib.slokv_kv_scores_accumulate(scores, 128, 64, width, rows, None, P, ls, 0, P, P, batch,
                                              hq, hkv, cap, 1.0, None, None)
    assert acc(batch=0) == 0 and acc(width=0) == 0 and acc(cap=0) == 0
    assert acc(batch=-1) == -1 and acc(hq=7) == -1 and acc(scores=None) == -1 and acc(ls=0) == -1
    assert acc(batch=65536) == -3 and acc(scores=ctypes.c_void_p(258)) == -2


def test_evict_arguments(pkg):
    lib = pkg._lib.lib()

    def call(dt=0, keep=10, recent=4, batch=2, d=128, bs=64, cache=P, scores=P, new=P, ws=None, wsb=0,
             stride=32768, w=4):
        return lib.slokv_kv_evict(cache, cache, stride, stride, 3, bs, 2, d, dt, P, 4, w, P, batch, scores,
                                  128, 64, 64, 2, None, keep, recent, new, None, ws, wsb, None, None)
    assert call(batch=0) == 0
    assert call(keep=0) == -1 and call(recent=-1) == -1 and call(recent=11) == -1 and call(batch=-1) == -1
    assert call(dt=3) == -3                                # FP8: the scale is shared by a block
    assert call(d=64) == -3 and call(dt=4, bs=96) == -3
    assert call(cache=None) == -1 and call(scores=None) == -1 and call(new=None) == -1 and call(w=0) == -1
    assert call(cache=ctypes.c_void_p(264)) == -2 and call(stride=32760) == -2
    need = lib.slokv_kv_evict_workspace_bytes(2, 2, 10, 64)
    assert need == 2 * 2 * (1 + 2 * 10) * 4
    assert lib.slokv_kv_evict_workspace_bytes(2, 2, 60, 64) == 2 * 2 * (1 + 2 * 4) * 4
    assert call() == -5 and call(ws=P, wsb=need - 1) == -5


def test_python_refusals(pkg):
    E = pkg.SlokvError
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    pool = torch.zeros(pkg.int4_pool_shape(2, 64, 2), dtype=torch.uint8)
    slots = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(E, match="CUDA"):
        pkg.store_kvcache_int4(k, k, pool, pool, slots)    # no CPU fallback
    with pytest.raises(E, match="multiple"):
        pkg.int4_pool_shape(2, 48, 2)
    for args in ((k[..., :64], k[..., :64], pool, pool, slots), (k, k[:2], pool, pool, slots),
                 (k, k.half(), pool, pool, slots), (k.int(), k.int(), pool, pool, slots),
                 (k, k, pool.view(2, 2, 64, 72), pool, slots), (k, k, pool[:, :1], pool[:, :1], slots),
                 (k, k, pool[..., :100], pool[..., :100], slots), (k, k, pool, pool[:1], slots),
                 (k.transpose(0, 2), k.transpose(0, 2), pool, pool, slots)):
        with pytest.raises(E):
            pkg.store_kvcache_int4(*args)
    q = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16)
    ln, bt = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(E, match="CUDA"):
        pkg.flash_attn_with_kvcache_int4(q, pool, pool, ln, bt)
    with pytest.raises(E, match="block_table is required"):
        pkg.flash_attn_varlen_func_int4(q[:, 0], pool, pool, ln, ln, 1, 1)
    with pytest.raises(E, match="causal"):
        pkg.flash_attn_varlen_func_int4(q[:, 0], pool, pool, ln, ln, 1, 1, causal=False, block_table=bt)
    fp8 = torch.zeros(2, 64, 2, 128, dtype=torch.uint8)
    with pytest.raises(E):
        pkg.flash_attn_with_kvcache_scored(q, fp8, fp8, torch.zeros(2, 2, 8), ln, bt)
    with pytest.raises(E):
        pkg.kv_evict(fp8, fp8, torch.zeros(2, 2, 8), ln, bt, 4, 1)
    for keep, recent in ((0, 0), (4, 5), (4, -1), (2 ** 31, 0), (2 ** 32 + 4, 1)):
        with pytest.raises(E, match="keep"):
            pkg.kv_evict(pool, pool, torch.zeros(2, 2, 8), ln, bt, keep, recent)


def test_sizes_past_32_bits_are_refused(pkg):
    """A table's reach whose tiles, or a score row whose positions, pass 32 bits."""
    lib = pkg._lib.lib()

    def int4(batch, hkv, w):
        stride = hkv * 64 * 72
        return lib.slokv_paged_decode_int4(P, 1024, 128, P, 1024, 128, P, P, stride, stride, 3, 64, hkv,
                                           hkv, 128, P, w, w, None, P, batch, 0.1, 0, None, 0, None,
                                           None, 0, None, None)
    assert int4(8192, 64, 4096) == -3 and int4(1, 2, 2 ** 30) == -3 and int4(8192, 2 ** 18, 1) == -3

    def logits(batch, w):
        return lib.slokv_paged_decode_logits(P, 1024, 128, P, 1024, 128, P, P, 32768, 32768, 3, 64, 8, 2,
                                             128, P, w, w, P, batch, 0.1, 0, P, 64, P, None, 0, None, None)
    assert logits(8192, 2 ** 16) == -3 and logits(1, 2 ** 29) == -3

    assert lib.slokv_kv_scores_accumulate(P, 2 ** 31, 2 ** 31, 2 ** 31 - 1, 2, None, P, 2 ** 31, 0, P, P, 2,
                                          8, 2, 2 ** 40, 1.0, None, None) == -3
    assert lib.slokv_kv_evict(P, P, 32768, 32768, 3, 64, 2, 128, 0, P, 2 ** 26, 2 ** 26, P, 2, P, 2 ** 31,
                              2 ** 31, 2 ** 31 - 1, 2, None, 10, 4, P, None, P, 2 ** 40, None, None) == -3
