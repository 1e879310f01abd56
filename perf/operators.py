"""Timed cases of the 4-bit KV cache and of eviction by attention weight.

  store    quantising append of a step's keys and values to a 4-bit pool, read back as values
  decode   one query per sequence over a 4-bit pool
  varlen   prefill chunks over a 4-bit pool's cached pages (causal, ragged)
  scored   decode over a bf16 / f16 / 4-bit pool that also accumulates each key's attention weight
  evict    keeping the recent and the heaviest tokens of each head, in place

`run` computes each in plain torch (32 bits, vectorised) or, where `own` is
set, calls the package.  `exact` follows the definitions in 64 bits.

A 4-bit pool is uint8 [num_blocks, kv_heads, block_size * 72]: per block and
head, tiles of 64 tokens, each 64 rows of 64 code bytes and then 64 rows of
(scale, minimum) x 2 groups in bf16.  A row's sixteen 32-bit words alternate
between the two 64-dim groups; within a group's 32 bytes dim 2i is the low and
2i + 1 the high half of byte i.  value = minimum + scale * code.
"""
import importlib
import math

import torch

own = False

D = 128          # head_dim of every cache here
TILE = 64        # tokens of a 4-bit tile
ROW = 72         # bytes of a token and head in a 4-bit pool


def _pkg():
    return importlib.import_module("slo-aware-llm-serving-engine_b200")


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _store(name, tokens, kv_heads, dtype, block, runs, fused):
    return dict(name=name, kind="store", tokens=tokens, kv_heads=kv_heads, dtype=dtype, block=block,
                runs=runs, fused=fused)


def _decode(name, batch, lo, hi, kv_heads, group, dtype, block):
    return dict(name=name, kind="decode", batch=batch, lo=lo, hi=hi, kv_heads=kv_heads,
                group=group, dtype=dtype, block=block)


def _varlen(name, rows, q_lo, q_hi, p_lo, p_hi, kv_heads, group, dtype, block):
    return dict(name=name, kind="varlen", rows=rows, q_lo=q_lo, q_hi=q_hi, p_lo=p_lo, p_hi=p_hi,
                kv_heads=kv_heads, group=group, dtype=dtype, block=block)


def _scored(name, batch, lo, hi, kv_heads, group, dtype, cache, block, decay):
    return dict(name=name, kind="scored", batch=batch, lo=lo, hi=hi, kv_heads=kv_heads,
                group=group, dtype=dtype, cache=cache, block=block, decay=decay)


def _evict(name, batch, lo, hi, kv_heads, dtype, cache, block, keep, recent):
    return dict(name=name, kind="evict", batch=batch, lo=lo, hi=hi, kv_heads=kv_heads,
                dtype=dtype, cache=cache, block=block, keep=keep, recent=recent)


def listed():
    return [
        # one decode step's new tokens of 256 sequences
        _store("store_decode_step", 256, 8, "bf16", 256, False, True),
        # a prefill step: a ragged 6,000-odd tokens, v a view into the fused qkv rows
        _store("store_prefill", 6211, 8, "bf16", 256, True, True),
        # a lone short request
        _decode("decode_one", 1, 513, 513, 8, 4, "f16", 128),
        # the FP8 decode workload's shape on a 4-bit pool
        _decode("decode_batch", 128, 1024, 8192, 8, 4, "bf16", 256),
        # two long documents, wide groups
        _decode("decode_long", 2, 90001, 98765, 4, 8, "bf16", 256),
        # a follow-up question of a few tokens on a cached conversation
        _varlen("varlen_followup", 1, 17, 17, 700, 700, 8, 4, "bf16", 256),
        # ragged prefill chunks, each with a cached prefix
        _varlen("varlen_chunks", 4, 1200, 2048, 900, 4000, 8, 4, "bf16", 256),
        # a small batch being scored
        _scored("scored_small", 3, 100, 700, 8, 4, "f16", "f16", 128, 0.5),
        # the bf16 decode workload's batch, accumulating weights
        _scored("scored_batch", 256, 512, 4096, 8, 4, "bf16", "bf16", 256, 1.0),
        # the same on a 4-bit pool
        _scored("scored_4bit", 96, 1000, 6000, 8, 4, "bf16", "int4", 256, 1.0),
        # a small batch held to a small budget, 4-bit
        _evict("evict_small", 2, 300, 700, 8, "bf16", "int4", 128, 200, 32),
        # a full batch cut to a quarter of the longest context
        _evict("evict_batch", 128, 512, 4096, 8, "bf16", "bf16", 256, 1024, 128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "decode", "varlen", "scored", "evict"])
    dtype = rng.choice(["bf16", "f16"])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    block = rng.choice([64, 128, 192, 256])
    if kind == "store":
        t = _log(rng, 1, 6000)
        c = _store("", t, kv_heads, dtype, block, t > 300 or rng.random() < 0.5, rng.random() < 0.5)
    elif kind == "varlen":
        q = _log(rng, 1, 1800)
        p = _log(rng, 1, 4000)
        c = _varlen("", rng.randint(1, 4), max(1, q // 2), q, p // 2, p, rng.choice([1, 2, 4, 8]),
                    rng.choice([1, 2, 4]), dtype, rng.choice([128, 256]))
    else:
        hi = _log(rng, 1, 60000 if kind == "decode" else 9000)
        lo = max(1, int(hi * rng.random()))
        # the largest listed batches hold about 600,000 tokens x 8 heads
        batch = _log(rng, 1, max(1.0, min(160.0, 2.5e6 / (hi * kv_heads))))
        cache = rng.choice([dtype, "int4"])
        if kind == "decode":
            c = _decode("", batch, lo, hi, kv_heads, group, dtype, block)
        elif kind == "scored":
            c = _scored("", batch, lo, hi, kv_heads, group, dtype, cache, block,
                        round(rng.choice([0.0, 1.0, rng.random()]), 3))
        else:
            keep = _log(rng, 1, max(1, hi))
            c = _evict("", batch, lo, hi, kv_heads, dtype, cache, block, keep,
                       rng.randint(0, keep))
    c.pop("name")
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float16


def _quantise(x):
    """Codes (uint8, 0..15) and (scale, minimum) of rows x [..., 128]: 32-bit
    arithmetic is the format's definition (subtraction, division and rounding to
    an even code each once)."""
    g = x.float().unflatten(-1, (2, 64))
    mn, mx = g.amin(-1), g.amax(-1)
    fifteen = torch.full((), 15.0, device=x.device).expand_as(mx)  # a true division, not x (1 / 15)
    scale = ((mx - mn) / fifteen).bfloat16()
    low = mn.bfloat16()
    s = scale.float().unsqueeze(-1)
    c = ((g - low.float().unsqueeze(-1)) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15)
    c = torch.where(s > 0, c, 0.0)
    return c.flatten(-2).to(torch.uint8), torch.stack((scale, low), -1)


def _pack(codes, params):
    """Rows' 64 code bytes and 8 parameter bytes as they lie in a pool."""
    b = codes.unflatten(-1, (64, 2))
    b = b[..., 0] | (b[..., 1] << 4)                                  # [..., 64]: two groups of 32
    b = b.unflatten(-1, (2, 8, 4)).transpose(-3, -2).flatten(-3)      # words alternate
    return b.contiguous(), params.flatten(-2).contiguous().view(torch.uint8)


def _tiles(cache):
    """(code bytes, parameter bytes) views of a pool [NB, H, bs * 72]: [NB, H, bs / 64, 64, 64 | 8]."""
    t = cache.unflatten(-1, (-1, TILE * ROW))
    return (t[..., :TILE * 64].unflatten(-1, (TILE, 64)),
            t[..., TILE * 64:].unflatten(-1, (TILE, 8)))


def _put(cache, rows, slots, block):
    """Store rows [T, H, 128] at `slots` of a 4-bit pool; -1 is skipped."""
    code, par = _pack(*_quantise(rows))
    keep = slots >= 0
    s = torch.where(keep, slots, 0).long()
    blk, off = s // block, s % block
    c, p = _tiles(cache)
    blk, tile, row = blk[keep], (off // TILE)[keep], (off % TILE)[keep]
    c[blk, :, tile, row] = code[keep]
    p[blk, :, tile, row] = par[keep]


def _values(pages):
    """fp32 values [n, bs, H, 128] of pages [n, H, bs * 72]."""
    c, p = _tiles(pages)
    b = c.unflatten(-1, (8, 2, 4)).transpose(-3, -2).flatten(-3)
    code = torch.stack((b & 15, b >> 4), -1).flatten(-2).unflatten(-1, (2, 64))
    par = p.contiguous().view(torch.bfloat16).unflatten(-1, (2, 2)).float()
    v = par[..., 1:] + par[..., :1] * code
    return v.flatten(-2).flatten(2, 3).transpose(1, 2)


def _pool(case, blocks, g, fill=True):
    """A pool of one side with random content (0.5 N(0, 1), one value in a hundred
    four times as large); every slot holds a row."""
    h, bs = case["kv_heads"], case["block"]
    if case.get("cache", "int4") == "int4":
        pool = torch.zeros(blocks, h, bs * ROW, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 25) // (h * bs * D))
        for i in range(0, blocks if fill else 0, step):
            n = min(step, blocks - i)
            slots = torch.arange(i * bs, (i + n) * bs, device="cuda")
            _put(pool, _rows((n * bs, h, D), _dtype(case["dtype"]), g), slots, bs)
        return pool
    pool = torch.empty(blocks, bs, h, D, dtype=_dtype(case["cache"]), device="cuda")
    step = max(1, (1 << 27) // (h * bs * D))
    for i in range(0, blocks, step):
        pool[i:i + step] = _rows(pool[i:i + step].shape, pool.dtype, g)
    return pool


def _rows(shape, dtype, g):
    x = torch.randn(shape, device="cuda", generator=g) * 0.5
    big = torch.rand(shape, device="cuda", generator=g) < 0.01
    return torch.where(big, 4 * x, x).to(dtype)


def _lens(n, lo, hi, g):
    return torch.randint(lo, hi + 1, (n,), device="cuda", generator=g, dtype=torch.int32)


def _spread(n, lo, hi):
    """n lengths from lo to hi, the longest first (the outputs' shape hangs on them, so no seed does)."""
    return torch.tensor([hi - (hi - lo) * i // max(1, n - 1) for i in range(n)], dtype=torch.int32,
                        device="cuda")


def _tables(lens, longest, block, g):
    """(block_table [B, W] of a shuffled pool, -1 past each row's last block; blocks)."""
    need = (lens.long() + block - 1) // block
    w = (longest + block - 1) // block
    total = lens.shape[0] * w + 2                                     # some blocks no row owns
    perm = torch.randperm(total, device="cuda", generator=g)
    first = torch.cumsum(need, 0) - need
    col = torch.arange(w, device="cuda")
    at = first.unsqueeze(1) + col
    t = torch.where(col < need.unsqueeze(1), perm[at.clamp(max=total - 1)], -1)
    return t.int().contiguous(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    dt = _dtype(case["dtype"])
    h, bs = case["kv_heads"], case["block"]
    st = {"case": case}
    if case["kind"] == "store":
        t = case["tokens"]
        i = torch.arange(t, device="cuda")
        if case["runs"]:                          # a prompt's tokens fill shuffled blocks in order
            blocks = (t + bs - 1) // bs + 3
            st["slots"] = torch.randperm(blocks, device="cuda", generator=g)[i // bs] * bs + i % bs
        else:                                     # each sequence's next token, in its own last block
            blocks = t + 3
            off = torch.randint(0, bs, (t,), device="cuda", generator=g)
            st["slots"] = torch.randperm(blocks, device="cuda", generator=g)[:t] * bs + off
        if t > 1:
            st["slots"][t // 2] = -1              # a padding row
        st["slots"] = st["slots"].int()
        if case["fused"]:
            qkv = _rows((t, 6 * h, D), dt, g)                         # q | k | v rows of one projection
            st["k"], st["v"] = qkv[:, 4 * h:5 * h], qkv[:, 5 * h:]
        else:
            st["k"], st["v"] = _rows((t, h, D), dt, g), _rows((t, h, D), dt, g)
        st["k_cache"] = _pool(case, blocks, g, fill=False)
        st["v_cache"] = _pool(case, blocks, g, fill=False)
        return st
    if case["kind"] == "varlen":
        n = case["rows"]
        ql = _spread(n, case["q_lo"], case["q_hi"])
        kl = ql + _lens(n, case["p_lo"], case["p_hi"], g)
        st["cu_q"] = torch.nn.functional.pad(ql.cumsum(0), (1, 0)).int()
        st["cu_k"] = torch.nn.functional.pad(kl.cumsum(0), (1, 0)).int()
        st["max_q"], st["max_k"] = case["q_hi"], case["q_hi"] + case["p_hi"]
        st["tables"], blocks = _tables(kl, st["max_k"], bs, g)
        st["q"] = torch.randn(int(ql.sum()), h * case["group"], D, device="cuda", generator=g).to(dt)
    else:
        b = case["batch"]
        st["lens"] = _lens(b, case["lo"], case["hi"], g)
        st["max_k"] = case["hi"]
        st["tables"], blocks = _tables(st["lens"], case["hi"], bs, g)
        if case["kind"] != "evict":
            st["q"] = torch.randn(b, 1, h * case["group"], D, device="cuda", generator=g).to(dt)
        if case["kind"] != "decode":
            # accumulated weights: a heavy tail, some keys never looked at, equal values
            s = torch.rand(b, h, st["max_k"], device="cuda", generator=g) ** 6
            s = torch.where(s < 1e-4, 0.0, (s * 4096).round() / 1024)
            live = torch.arange(st["max_k"], device="cuda") < st["lens"].view(-1, 1, 1)
            st["scores"] = torch.where(live, s, 0.0).contiguous()
    st["k_cache"] = _pool(case, blocks, g)
    st["v_cache"] = _pool(case, blocks, g)
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _gathered(cache, tables):
    """fp32 rows [B, H, W * bs, 128] of a pool through a block table (-1 reads block 0)."""
    pages = cache[tables.clamp(min=0).long()]
    if cache.dtype == torch.uint8:
        v = _values(pages.flatten(0, 1)).unflatten(0, pages.shape[:2])
    else:
        v = pages.float()
    return v.flatten(1, 2).transpose(1, 2)


def _attend(q, k, v, live):
    """(out, weights) of q [B, H, G, D] over k, v [B, H, L, D]; live: [B, 1, 1 | G, L]."""
    s = torch.matmul(q * D ** -0.5, k.transpose(-1, -2))
    s = torch.where(live, s, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    return torch.matmul(w, v), w


def _plain_step(st):
    case = st["case"]
    q = st["q"]
    qh = q.float().view(q.shape[0], case["kv_heads"], case["group"], D)
    k, v = _gathered(st["k_cache"], st["tables"]), _gathered(st["v_cache"], st["tables"])
    live = torch.arange(k.shape[2], device="cuda") < st["lens"].view(-1, 1, 1, 1)
    o, w = _attend(qh, k, v, live)
    return o.reshape(q.shape).to(q.dtype), w


def _plain_varlen(st):
    case, q = st["case"], st["q"]
    n, h, grp = case["rows"], case["kv_heads"], case["group"]
    ql, kl = st["cu_q"].diff().long(), st["cu_k"].diff().long()
    col = torch.arange(st["max_q"], device="cuda")
    at = st["cu_q"][:-1].long().unsqueeze(1) + col
    there = col < ql.unsqueeze(1)
    rows = q.float()[at.clamp(max=q.shape[0] - 1)]                    # [n, max_q, Hq, D]
    rows = rows.view(n, st["max_q"], h, grp, D).permute(0, 2, 3, 1, 4).reshape(n, h, -1, D)
    k, v = _gathered(st["k_cache"], st["tables"]), _gathered(st["v_cache"], st["tables"])
    key = torch.arange(k.shape[2], device="cuda")
    last = (kl - ql).unsqueeze(1) + col                               # the last key that a query sees
    live = key <= last.unsqueeze(-1)
    live = live.unsqueeze(1).expand(n, grp, -1, -1).reshape(n, 1, -1, k.shape[2])
    o, _ = _attend(rows, k, v, live)
    o = o.view(n, h, grp, st["max_q"], D).permute(0, 3, 1, 2, 4).reshape(n, st["max_q"], h * grp, D)
    return o[there].to(q.dtype)


def _kept(scores, lens, keep, recent):
    """(new lengths [B], source position of each slot below the new length [B, H, keep], -1 past it)."""
    t = torch.arange(scores.shape[-1], device="cuda")
    n = lens.long().view(-1, 1, 1)
    live = t < n
    safe = live & (t >= n - recent)
    key = torch.where(live & ~safe, scores.nan_to_num(-math.inf, math.inf, -math.inf), -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    # a protected token sorts as -inf: drop it from the order before the best are taken
    free = torch.gather((live & ~safe).expand_as(key), -1, order)
    take = free & (free.cumsum(-1) <= keep - recent)
    kept = torch.zeros_like(take).scatter(-1, order, take) | safe
    kept = torch.where(n <= keep, live, kept)
    new = lens.clamp(max=keep)
    m = new.long().view(-1, 1, 1)
    hole, mover = (t < m) & ~kept, (t >= m) & kept
    movers = torch.sort((~mover).byte(), dim=-1, stable=True).indices  # movers first, in order
    src = torch.where(hole, torch.gather(movers, -1, (hole.cumsum(-1) - 1).clamp(min=0)), t)
    src = torch.where(t < m, src, -1)
    return new, torch.nn.functional.pad(src, (0, keep), value=-1)[..., :keep].int()


def _plain_evict(st):
    case = st["case"]
    lens, scores, bs = st["lens"], st["scores"].clone(), case["block"]
    new, src = _kept(scores, lens, case["keep"], case["recent"])
    slot = torch.arange(src.shape[-1], device="cuda")
    b, h, to = torch.nonzero((src >= 0) & (src != slot), as_tuple=True)
    frm = src[b, h, to].long()
    tb, fb = st["tables"][b, to // bs].long(), st["tables"][b, frm // bs].long()
    to, frm = to % bs, frm % bs
    for cache in (st["k_cache"], st["v_cache"]):
        if cache.dtype == torch.uint8:
            for part in _tiles(cache):
                part[tb, h, to // TILE, to % TILE] = part[fb, h, frm // TILE, frm % TILE]
        else:
            cache[tb, to, h] = cache[fb, frm, h]
    moved = torch.gather(scores, -1, src[..., :scores.shape[-1]].clamp(min=0).long())
    moved = torch.where(src[..., :scores.shape[-1]] >= 0, moved, 0.0)
    scores.zero_()
    scores[..., :moved.shape[-1]] = moved
    return new, src, scores


def run(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "store":
        if own:
            p = _pkg()
            p.store_kvcache_int4(st["k"], st["v"], st["k_cache"], st["v_cache"], st["slots"])
            return (p.int4_decode(st["k_cache"], st["slots"]), p.int4_decode(st["v_cache"], st["slots"]))
        out = []
        for x, cache in ((st["k"], st["k_cache"]), (st["v"], st["v_cache"])):
            _put(cache, x, st["slots"], case["block"])
            s = st["slots"].long()
            c, p = _tiles(cache)
            blk, off = s.clamp(min=0) // case["block"], s.clamp(min=0) % case["block"]
            at = (blk, slice(None), off // TILE, off % TILE)
            # each stored row read back as a block of a single token
            b = c[at].unflatten(-1, (8, 2, 4)).transpose(-3, -2).flatten(-3)
            code = torch.stack((b & 15, b >> 4), -1).flatten(-2).unflatten(-1, (2, 64))
            par = p[at].contiguous().view(torch.bfloat16).unflatten(-1, (2, 2)).float()
            v = (par[..., 1:] + par[..., :1] * code).flatten(-2)
            out.append(torch.where(s.view(-1, 1, 1) >= 0, v, 0.0))
        return tuple(out)
    if kind == "decode":
        if own:
            return _pkg().flash_attn_with_kvcache_int4(st["q"], st["k_cache"], st["v_cache"],
                                                       st["lens"], st["tables"])
        return _plain_step(st)[0]
    if kind == "varlen":
        if own:
            return _pkg().flash_attn_varlen_func_int4(st["q"], st["k_cache"], st["v_cache"],
                                                      st["cu_q"], st["cu_k"], st["max_q"],
                                                      st["max_k"], block_table=st["tables"])
        return _plain_varlen(st)
    if kind == "scored":
        scores = st["scores"].clone()             # the call adds in place: a pass can be repeated
        if own:
            o = _pkg().flash_attn_with_kvcache_scored(st["q"], st["k_cache"], st["v_cache"], scores,
                                                      st["lens"], st["tables"], st["max_k"],
                                                      decay=case["decay"])
            return o, scores
        o, w = _plain_step(st)
        w = w.sum(2)[..., :scores.shape[-1]]
        live = torch.arange(scores.shape[-1], device="cuda") < st["lens"].view(-1, 1, 1)
        return o, torch.where(live, case["decay"] * scores + w, scores)
    if own:
        scores = st["scores"].clone()
        new, src = _pkg().kv_evict(st["k_cache"], st["v_cache"], scores, st["lens"], st["tables"],
                                   case["keep"], case["recent"], return_index=True)
    else:
        new, src, scores = _plain_evict(st)
    return new, src, scores, st["k_cache"], st["v_cache"]


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------

def work(case):
    h = case["kv_heads"]
    row = 2 * (ROW if case.get("cache", "int4") == "int4" else 2 * D)  # K and V bytes of a token and head
    if case["kind"] == "store":
        t = case["tokens"]
        # rows in, 4-bit rows out, and read back as fp32 values
        return {"bytes": t * h * 2 * (2 * D + 2 * ROW + 4 * D), "flops": t * h * 2 * D * 6}
    if case["kind"] == "varlen":
        q = case["rows"] * (case["q_lo"] + case["q_hi"]) / 2
        pre = (case["p_lo"] + case["p_hi"]) / 2
        per = (case["q_lo"] + case["q_hi"]) / 2
        pairs = q * (pre + (per + 1) / 2)
        return {"bytes": 2 * q * h * case["group"] * D * 2 + case["rows"] * (pre + per) * h * row,
                "flops": 4 * D * h * case["group"] * pairs}
    tokens = case["batch"] * (case["lo"] + case["hi"]) / 2
    if case["kind"] == "evict":
        # scores in and out; of the kept tokens the share that lies past `keep` moves
        span = case["hi"] - case["lo"] + 1
        lens = [case["lo"] + span * (i + 0.5) / 64 for i in range(64)]
        moved = sum(case["keep"] * (1 - case["keep"] / n) for n in lens if n > case["keep"]) / 64
        return {"bytes": tokens * h * 8 + case["batch"] * h * (moved * 2 * row + 4 * case["keep"]),
                "flops": tokens * h}
    qo = 2 * case["batch"] * h * case["group"] * D * 2
    scores = 8 if case["kind"] == "scored" else 0
    return {"bytes": tokens * h * (row + scores) + qo,
            "flops": tokens * h * case["group"] * (4 * D + 4)}


# ---------------------------------------------------------------------------
# definitions in 64 bits
# ---------------------------------------------------------------------------

def _value64(cache, blk, off):
    """Rows [n, H, 128] in 64 bits at (block, offset) of a pool, bit by bit from the format."""
    if cache.dtype != torch.uint8:
        return cache[blk, off].double()
    n, h = blk.shape[0], cache.shape[1]
    raw = cache[blk]                                                   # [n, H, bs * 72]
    base = (off // 64) * 4608
    d = torch.arange(128, device="cuda")
    word = 2 * ((d % 64) // 8) + d // 64                               # alternating words
    byte = 4 * word + (d % 8) // 2
    at = (base + (off % 64) * 64).view(n, 1, 1) + byte
    nib = torch.gather(raw, 2, at.expand(n, h, 128))
    code = torch.where(d % 2 == 1, nib // 16, nib % 16).double()
    lo = (base + 4096 + (off % 64) * 8).view(n, 1, 1) + 4 * (d // 64)

    def bf16(first):
        a = torch.gather(raw, 2, (first).expand(n, h, 128)).int()
        b = torch.gather(raw, 2, (first + 1).expand(n, h, 128)).int()
        return ((a | (b << 8)) << 16).view(torch.float32).double()

    return bf16(lo + 2) + bf16(lo) * code


def _row64(st, cache, b, n):
    """Keys 0 .. n - 1 of row b in 64 bits, [H, n, 128]."""
    bs = st["case"]["block"]
    t = torch.arange(n, device="cuda")
    blk = st["tables"][b].long()[t // bs]
    step = 16384
    rows = [_value64(cache, blk[i:i + step], (t % bs)[i:i + step]) for i in range(0, n, step)]
    return torch.cat(rows).transpose(0, 1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "store":
        out = []
        for x in (st["k"], st["v"]):
            x = x.double().reshape(-1, 64)
            lo, hi = x.min(1).values, x.max(1).values
            s = ((hi - lo) / 15).float().bfloat16().double()           # stored as bf16
            m = lo.float().bfloat16().double()
            r = torch.where(s > 0, s, 1.0).unsqueeze(1)
            c = torch.clamp(torch.round((x - m.unsqueeze(1)) / r), 0, 15)
            v = m.unsqueeze(1) + s.unsqueeze(1) * c
            v = v.reshape(case["tokens"], case["kv_heads"], D)
            out.append(v * (st["slots"] >= 0).view(-1, 1, 1))
        return tuple(out)
    if case["kind"] in ("decode", "scored"):
        q = st["q"].double()
        out = torch.zeros_like(q)
        scores = st["scores"].double() if case["kind"] == "scored" else None
        for b, n in enumerate(st["lens"].tolist()):
            k, v = _row64(st, st["k_cache"], b, n), _row64(st, st["v_cache"], b, n)
            qb = q[b, 0].view(case["kv_heads"], case["group"], D)
            w = torch.softmax(torch.einsum("hgd,hnd->hgn", qb, k) / math.sqrt(D), -1)
            out[b, 0] = torch.einsum("hgn,hnd->hgd", w, v).reshape(-1, D)
            if scores is not None:
                scores[b, :, :n] = case["decay"] * scores[b, :, :n] + w.sum(1)
        return out if scores is None else (out, scores)
    if case["kind"] == "varlen":
        q = st["q"].double()
        out = torch.zeros_like(q)
        cq, ck = st["cu_q"].tolist(), st["cu_k"].tolist()
        for b in range(case["rows"]):
            lq, lk = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
            k, v = _row64(st, st["k_cache"], b, lk), _row64(st, st["v_cache"], b, lk)
            qb = q[cq[b]:cq[b + 1]].view(lq, case["kv_heads"], case["group"], D)
            s = torch.einsum("qhgd,hnd->hgqn", qb, k) / math.sqrt(D)
            see = torch.ones(lq, lk, device="cuda", dtype=torch.bool).tril(lk - lq)
            w = torch.softmax(s.masked_fill(~see, -math.inf), -1)
            out[cq[b]:cq[b + 1]] = torch.einsum("hgqn,hnd->qhgd", w, v).reshape(lq, -1, D)
        return out
    # eviction moves values: its scores and bf16 / f16 rows, by lists on the host
    if case["batch"] * case["kv_heads"] * st["max_k"] > 400_000:
        return None
    bs, keep, recent = case["block"], case["keep"], case["recent"]
    host = st["scores"].double().cpu()
    scores = torch.zeros_like(host)
    tables = st["tables"].tolist()
    caches = [None if c.dtype == torch.uint8 else c.double().cpu() for c in (st["k_cache"], st["v_cache"])]
    for b, n in enumerate(st["lens"].tolist()):
        for h in range(case["kv_heads"]):
            row = host[b, h].tolist()
            if n <= keep:
                scores[b, h] = host[b, h]
                continue
            old = sorted(range(n - recent), key=lambda t: (-row[t], t))[:keep - recent]
            kept = set(old) | set(range(n - recent, n))
            holes = [t for t in range(keep) if t not in kept]
            moved = sorted(t for t in kept if t >= keep)
            src = dict(zip(holes, moved))
            for t in range(keep):
                scores[b, h, t] = row[src.get(t, t)]
            for t, f in src.items():
                for c in caches:
                    if c is not None:
                        c[tables[b][t // bs], t % bs, h] = c[tables[b][f // bs], f % bs, h]
    return None, None, scores, caches[0], caches[1]
