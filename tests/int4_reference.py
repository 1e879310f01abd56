"""Plain 64-bit restatements of the 4-bit pool, its attention and the eviction rule.

Test infrastructure.  Everything works on CPU tensors and follows the definitions in
include/slokv.h step by step: the format byte by byte, attention as an explicit
softmax, eviction by sorted lists.
"""
import math

import numpy as np
import torch

D = 128


def row_offsets(off):
    """(first code byte, first parameter byte) of token `off` in its (block, head) run."""
    tile, row = divmod(off, 64)
    return tile * 4608 + row * 64, tile * 4608 + 4096 + row * 8


def encode_row(x):
    """(codes [128] 0..15, parameters [4] as bf16 bits, finite) of one row, fp32 arithmetic."""
    x = x.float().numpy().astype(np.float32)
    codes, par, fine = np.zeros(D, np.uint8), np.zeros(4, np.uint16), True
    for g in range(2):
        v = x[64 * g:64 * g + 64]
        ok = bool(np.isfinite(v).all())
        if ok:
            with np.errstate(over="ignore"):
                s = torch.tensor(np.float32(np.float32(v.max() - v.min()) / np.float32(15))).bfloat16()
            m = torch.tensor(v.min()).bfloat16()
            ok = bool(torch.isfinite(s)) and bool(torch.isfinite(m))
        if not ok:
            par[2 * g], fine = 0x7FFF, False
            continue
        sf, mf = np.float32(s.float().item()), np.float32(m.float().item())
        if sf > 0:
            with np.errstate(over="ignore"):
                codes[64 * g:64 * g + 64] = np.clip(np.rint((v - mf) / sf), 0, 15).astype(np.uint8)
        par[2 * g] = s.view(torch.int16).item() & 0xFFFF
        par[2 * g + 1] = m.view(torch.int16).item() & 0xFFFF
    return codes, par, fine


def put_row(pool, block, head, off, codes, par):
    """Write one row into a CPU pool [NB, H, bs * 72] (numpy uint8)."""
    c0, p0 = row_offsets(off)
    for d in range(D):
        g, i = divmod(d, 64)
        word, nib = divmod(i, 8)
        byte = c0 + 4 * (2 * word + g) + nib // 2
        old = int(pool[block, head, byte])
        pool[block, head, byte] = (old & 0x0F) | (int(codes[d]) << 4) if nib % 2 else \
            (old & 0xF0) | int(codes[d])
    for k in range(4):
        pool[block, head, p0 + 2 * k] = int(par[k]) & 0xFF
        pool[block, head, p0 + 2 * k + 1] = int(par[k]) >> 8


def store(key, value, k_pool, v_pool, slots, block):
    """store_kvcache_int4 on CPU tensors; returns whether every group was finite."""
    kp, vp = k_pool.numpy(), v_pool.numpy()
    fine = True
    for t, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        for h in range(key.shape[1]):
            for x, pool in ((key, kp), (value, vp)):
                codes, par, ok = encode_row(x[t, h])
                put_row(pool, slot // block, h, slot % block, codes, par)
                fine &= ok
    return fine


def decode_pool(pool):
    """fp64 values [NB, bs, H, 128] and parameters (scale, minimum) [NB, bs, H, 2] of a pool."""
    nb, h, size = pool.shape
    tiles = pool.numpy().reshape(nb, h, size // 4608, 4608)
    code = tiles[..., :4096].reshape(nb, h, -1, 64, 16, 4)             # 16 words a row
    vals = np.zeros((nb, h, code.shape[2], 64, D))
    for d in range(D):
        g, i = divmod(d, 64)
        word, nib = divmod(i, 8)
        vals[..., d] = (code[..., 2 * word + g, nib // 2] >> (4 * (nib % 2))) & 15
    bits = np.ascontiguousarray(tiles[..., 4096:]).view(np.uint16).reshape(nb, h, -1, 64, 4)
    par = (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    vals[..., :64] = par[..., 1:2] + par[..., 0:1] * vals[..., :64]
    vals[..., 64:] = par[..., 3:4] + par[..., 2:3] * vals[..., 64:]
    v = torch.from_numpy(vals).reshape(nb, h, -1, D).transpose(1, 2)
    scale = torch.from_numpy(np.ascontiguousarray(par[..., 0::2])).reshape(nb, h, -1, 2).transpose(1, 2)
    return v, scale


def gather(values, table, n):
    """Rows 0 .. n - 1 of a sequence, [n, H, 128], through its block table row; a block id
    outside the pool reads as zeros."""
    bs = values.shape[1]
    out = torch.zeros(n, *values.shape[2:], dtype=values.dtype)
    for p in range((n + bs - 1) // bs):
        blk = int(table[p])
        stop = min(n, (p + 1) * bs)
        if 0 <= blk < values.shape[0]:
            out[p * bs:stop] = values[blk, :stop - p * bs]
    return out


def attend(q, k, v, scale):
    """(out [Hq, 128], weights [Hq, n]) of q [Hq, 128] over k, v [n, H, 128], fp64."""
    G = q.shape[0] // k.shape[1]
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("hd,nhd->hn", q.double(), kk) * scale
    w = torch.softmax(s, -1)
    return torch.einsum("hn,nhd->hd", w, vv), w


def kept_index(score, n, keep, recent):
    """Source position of each slot below min(n, keep), for one (sequence, head)."""
    if n <= keep:
        return list(range(n))
    val = [-math.inf if math.isnan(x) else x for x in score[:n]]
    old = sorted(range(n - recent), key=lambda t: (-val[t], t))[:keep - recent]
    kept = set(old) | set(range(n - recent, n))
    holes = [t for t in range(keep) if t not in kept]
    moved = sorted(t for t in kept if t >= keep)
    assert len(holes) == len(moved)
    src = list(range(keep))
    for a, b in zip(holes, moved):
        src[a] = b
    return src
