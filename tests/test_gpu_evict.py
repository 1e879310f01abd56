"""Scored decode and eviction on the GPU against 64-bit restatements
(tests/int4_reference.py).

Tolerance of the scores: a weight is 2^(x - lse) with x an fp32 score.  Its error e is at
most 400 u times the absolute sum of the score's products (u = 2^-24; see
test_gpu_int4.py), the subtraction and the exponential add u |x - lse| and 2^-21, the
denominator moves by the same and by 2 u sqrt-free per added key (n u at most), so a weight is
off by (2 e + 2^-20 + (n + 200) u) of itself; accumulating adds u of the score.  Eviction only
moves bytes: everything about it is compared exactly.
"""
import math

import numpy as np
import pytest
import torch

from tests import int4_reference as R
from tests.golden.detgen import det_ints, det_normal, det_perm
from tests.test_gpu_int4 import make_pool, make_tables

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dense_pool(seed, nb, bs, h, dtype):
    return (torch.from_numpy(det_normal(seed, (nb, bs, h, 128))).float() * 0.5).to(dtype).cuda()


def pool_values(pool):
    return R.decode_pool(pool.cpu())[0] if pool.dim() == 3 else pool.cpu().double()


def any_pool(pkg, kind, seed, nb, bs, h, dtype):
    return make_pool(pkg, seed, nb, bs, h) if kind == "int4" else dense_pool(seed, nb, bs, h, dtype)


@pytest.mark.parametrize("kind", ["dense", "int4"])
@pytest.mark.parametrize("lens,H,G,bs,dtype,decay", [
    ([1], 1, 1, 64, torch.bfloat16, 1.0),
    ([65, 0, 300, 1], 2, 4, 64, torch.float16, 0.75),
    ([2500, 31], 3, 5, 128, torch.bfloat16, 0.0),
    ([700], 1, 16, 192, torch.bfloat16, 1.0),
])
def test_scored_decode(pkg, kind, lens, H, G, bs, dtype, decay):
    B = len(lens)
    nb = sum((n + bs - 1) // bs for n in lens) + 1
    kp, vp = (any_pool(pkg, kind, 5 + i, nb, bs, H, dtype) for i in range(2))
    tables = make_tables(7, lens, bs, nb).cuda()
    q = torch.from_numpy(det_normal(8, (B, 1, H * G, 128))).float().to(dtype)
    width = max(lens) + 3
    old = torch.from_numpy(det_normal(9, (B, H, width))).float().abs()
    scores = old.cuda()
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    pkg.read_device_errors()
    out = pkg.flash_attn_with_kvcache_scored(q.cuda(), kp, vp, scores, ln, tables, max(lens), decay=decay)
    assert pkg.read_device_errors() == 0
    plain = (pkg.flash_attn_with_kvcache_int4 if kind == "int4" else pkg.flash_attn_with_kvcache)(
        q.cuda(), kp, vp, ln, tables)
    assert torch.equal(out, plain)                     # scoring does not change the attention
    kv, vv = pool_values(kp), pool_values(vp)
    got = scores.cpu().double()
    assert torch.equal(scores.cpu()[:, :, max(lens):], old[:, :, max(lens):])
    for b, n in enumerate(lens):
        assert torch.equal(scores.cpu()[b, :, n:], old[b, :, n:])     # past the context: untouched
        if not n:
            continue
        k, v = R.gather(kv, tables[b].cpu(), n), R.gather(vv, tables[b].cpu(), n)
        _, w = R.attend(q[b, 0], k, v, 128 ** -0.5)
        span = k.abs().max() * 3                       # 15 s + |m| against max |k| of a group
        e = 400 * U * 128 ** -0.5 * q[b, 0].double().abs().sum(-1).max() * span
        w = w.view(H, G, n).sum(1)
        want = decay * old[b, :, :n].double() + w
        tol = (2 * e + 2.0 ** -20 + (n + 200) * U) * w + 2 * U * want
        assert ((got[b, :, :n] - want).abs() <= tol).all()


def test_scored_rows_width_and_views(pkg):
    """score_rows maps and skips, a narrow table is flagged and left alone past its width,
    strided score tables work, and rows that are not named stay as they were."""
    lens, H, G, bs = [100, 50, 200], 2, 2, 64
    nb = 9
    kp, vp = dense_pool(11, nb, bs, H, torch.bfloat16), dense_pool(12, nb, bs, H, torch.bfloat16)
    tables = make_tables(13, lens, bs, nb).cuda()
    q = torch.from_numpy(det_normal(14, (3, 1, H * G, 128))).float().bfloat16().cuda()
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    full = torch.zeros(3, H, 200, device="cuda")
    pkg.flash_attn_with_kvcache_scored(q, kp, vp, full, ln, tables)
    pkg.read_device_errors()
    store = torch.full((5, H, 2, 210), 3.0, device="cuda")
    scores = store[:, :, 1, 1:202]                     # unaligned view: 4-byte accesses
    rows = torch.tensor([4, -1, 0], dtype=torch.int32, device="cuda")
    pkg.flash_attn_with_kvcache_scored(q, kp, vp, scores, ln, tables, score_rows=rows, decay=0.0)
    assert pkg.read_device_errors() == 0
    assert torch.equal(scores[4, :, :100], full[0, :, :100])
    assert torch.equal(scores[0, :, :200], full[2, :, :200])
    assert (scores[1:4] == 3).all() and (store[:, :, 0] == 3).all() and (scores[4, :, 100:] == 3).all()
    bad = torch.tensor([5, 1, -3], dtype=torch.int32, device="cuda")
    pkg.flash_attn_with_kvcache_scored(q, kp, vp, scores, ln, tables, score_rows=bad)
    assert pkg.read_device_errors() == 0x1
    narrow = torch.zeros(3, H, 64, device="cuda")
    pkg.flash_attn_with_kvcache_scored(q, kp, vp, narrow, ln, tables)
    assert pkg.read_device_errors() == 0x4
    assert torch.equal(narrow[2], full[2, :, :64]) and torch.equal(narrow[1, :, :50], full[1, :, :50])


def test_scored_shared_prefix_block(pkg):
    """Two sequences that share their first block are scored apart."""
    bs, H, G = 64, 1, 4
    kp, vp = make_pool(pkg, 21, 4, bs, H), make_pool(pkg, 22, 4, bs, H)
    tables = torch.tensor([[2, 0], [2, 1]], dtype=torch.int32, device="cuda")
    q = torch.from_numpy(det_normal(23, (2, 1, 4, 128))).float().bfloat16().cuda()
    ln = torch.tensor([90, 100], dtype=torch.int32, device="cuda")
    both = torch.zeros(2, H, 100, device="cuda")
    pkg.flash_attn_with_kvcache_scored(q, kp, vp, both, ln, tables)
    for b in range(2):
        one = torch.zeros(1, H, 100, device="cuda")
        pkg.flash_attn_with_kvcache_scored(q[b:b + 1], kp, vp, one, ln[b:b + 1], tables[b:b + 1])
        assert torch.equal(one[0], both[b])


def test_scored_graph_replays_accumulate(pkg):
    bs, H, G = 64, 2, 4
    kp, vp = make_pool(pkg, 31, 6, bs, H), make_pool(pkg, 32, 6, bs, H)
    tables = make_tables(33, [300], bs, 6).cuda()
    q = torch.from_numpy(det_normal(34, (1, 1, 8, 128))).float().bfloat16().cuda()
    ln = torch.tensor([300], dtype=torch.int32, device="cuda")
    once = torch.zeros(1, H, 300, device="cuda")
    pkg.flash_attn_with_kvcache_scored(q, kp, vp, once, ln, tables)
    scores = torch.zeros(1, H, 300, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pkg.flash_attn_with_kvcache_scored(q, kp, vp, scores, ln, tables)
    assert (scores == 0).all()
    for _ in range(3):
        g.replay()
    assert torch.equal(scores, once + once + once)


# ---- eviction ---------------------------------------------------------------------

def scores_for(seed, B, H, width, lens, kind):
    x = det_normal(seed, (B, H, width)).astype(np.float32)
    if kind == "ties":
        x = np.round(np.abs(x) * 2) / 2
    if kind == "odd":                                  # every kind of float
        x[..., ::7] = np.nan
        x[..., 1::7] = np.inf
        x[..., 2::11] = -np.inf
        x[..., 3::5] = 0.0
        x[..., 4::5] = -0.0
    if kind == "zeros":
        x[:] = 0
    for b, n in enumerate(lens):
        x[b, :, n:] = 0
    return torch.from_numpy(x)


EVICT = [
    # lens, keep, recent, H, bs
    ([1, 2, 3], 1, 0, 1, 64),
    ([1, 2, 3], 1, 1, 1, 64),
    ([0, 64, 65, 130], 64, 10, 2, 64),
    ([700, 33, 1023], 200, 0, 3, 128),
    ([700, 33, 1023], 200, 200, 2, 128),
    ([513, 400], 400, 32, 2, 192),
    ([900], 899, 5, 1, 64),
    ([9500, 8300], 4000, 100, 2, 256),                 # more keys than shared memory holds
    ([50], 1000, 10, 2, 64),
]


@pytest.mark.parametrize("lens,keep,recent,H,bs", EVICT, ids=[str(i) for i in range(len(EVICT))])
@pytest.mark.parametrize("kind", ["normal", "ties", "odd", "zeros"])
@pytest.mark.parametrize("cache", ["bf16", "int4"])
def test_evict(pkg, lens, keep, recent, H, bs, kind, cache):
    B = len(lens)
    nb = sum((n + bs - 1) // bs for n in lens) + 2
    width = max(lens) + 5
    if cache == "int4":                                # random bytes: only moved, never read
        shape = pkg.int4_pool_shape(nb, bs, H)
        kp, vp = (torch.from_numpy(det_ints(40 + i, int(np.prod(shape)), 0, 256).astype(np.uint8)
                                   .reshape(shape)).cuda() for i in range(2))
    else:
        kp, vp = dense_pool(41, nb, bs, H, torch.bfloat16), dense_pool(42, nb, bs, H, torch.bfloat16)
    tables = make_tables(43, lens, bs, nb)
    scores = scores_for(44, B, H, width, lens, kind)
    want_k, want_v, want_s = kp.cpu().clone(), vp.cpu().clone(), scores.clone()
    want_i = torch.full((B, H, keep), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(H):
            src = R.kept_index(scores[b, h].tolist(), n, keep, recent)
            want_i[b, h, :len(src)] = torch.tensor(src, dtype=torch.int32)
            if n > keep:
                want_s[b, h, :keep] = scores[b, h, src]
                want_s[b, h, keep:n] = 0
            for t, f in enumerate(src):
                if t == f:
                    continue
                tb, fb = int(tables[b, t // bs]), int(tables[b, f // bs])
                for want, have in ((want_k, kp), (want_v, vp)):
                    if cache == "int4":
                        tc, tp = R.row_offsets(t % bs)
                        fc, fp = R.row_offsets(f % bs)
                        want[tb, h, tc:tc + 64] = want[fb, h, fc:fc + 64]
                        want[tb, h, tp:tp + 8] = want[fb, h, fp:fp + 8]
                    else:
                        want[tb, t % bs, h] = want[fb, f % bs, h]
    gs = scores.cuda()
    pkg.read_device_errors()
    new, index = pkg.kv_evict(kp, vp, gs, torch.tensor(lens, dtype=torch.int32).cuda(), tables.cuda(),
                              keep, recent, return_index=True)
    assert pkg.read_device_errors() == 0
    assert new.tolist() == [min(n, keep) for n in lens]
    assert torch.equal(index.cpu(), want_i)
    assert torch.equal(gs.cpu().view(torch.int32), want_s.view(torch.int32))
    same = (lambda a, b: torch.equal(a, b)) if cache == "int4" else \
        (lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16)))
    assert same(kp.cpu(), want_k) and same(vp.cpu(), want_v)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_evict_other_pools_and_rows(pkg, dtype):
    """f16 and fp32 pools with strided blocks, score rows by index, one of them skipped."""
    bs, H, nb, lens, keep, recent = 16, 2, 8, [40, 60], 20, 4
    kp = dense_pool(51, 2 * nb, bs, H, dtype)[::2]
    vp = dense_pool(52, nb, bs, H, dtype)
    tables = make_tables(53, lens, bs, nb)
    scores = scores_for(54, 6, H, 60, [60] * 6, "normal")
    rows = torch.tensor([-1, 3], dtype=torch.int32, device="cuda")
    want_k, want_v = kp.cpu().clone(), vp.cpu().clone()
    for h in range(H):
        for t, f in enumerate(R.kept_index(scores[3, h].tolist(), 60, keep, recent)):
            tb, fb = int(tables[1, t // bs]), int(tables[1, f // bs])
            want_k[tb, t % bs, h], want_v[tb, t % bs, h] = want_k[fb, f % bs, h].clone(), want_v[fb, f % bs, h].clone()
    gs = scores.cuda()
    new = pkg.kv_evict(kp, vp, gs, torch.tensor(lens, dtype=torch.int32).cuda(), tables.cuda(), keep,
                       recent, score_rows=rows)
    assert new.tolist() == [40, 20]
    assert torch.equal(kp.cpu(), want_k) and torch.equal(vp.cpu(), want_v)
    assert torch.equal(gs.cpu()[[0, 1, 2, 4, 5]], scores[[0, 1, 2, 4, 5]])


def test_evict_bad_metadata_is_flagged(pkg):
    """Rows whose context outruns the table or the scores, or whose score row does not
    exist, are left as they are; a move through a bad block id is dropped."""
    bs, H = 64, 1
    kp, vp = make_pool(pkg, 61, 4, bs, H), make_pool(pkg, 62, 4, bs, H)
    k0, v0 = kp.clone(), vp.clone()
    ln = torch.tensor([300, 100], dtype=torch.int32, device="cuda")
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    scores = torch.zeros(2, H, 128, device="cuda")
    pkg.read_device_errors()
    new = pkg.kv_evict(kp, vp, scores, ln, tables, 200, 0)
    assert pkg.read_device_errors() == 0x4 and new.tolist() == [300, 100]
    new = pkg.kv_evict(kp, vp, scores[:, :, :90], ln[1:], tables[1:], 10, 10)
    assert pkg.read_device_errors() == 0x4 and new.tolist() == [100]
    new = pkg.kv_evict(kp, vp, scores, ln[1:], tables[1:], 10, 10,
                       score_rows=torch.tensor([2], dtype=torch.int32, device="cuda"))
    assert pkg.read_device_errors() == 0x1 and new.tolist() == [100]
    new = pkg.kv_evict(kp, vp, scores, ln[1:], torch.tensor([[2, 9]], dtype=torch.int32, device="cuda"),
                       10, 10)
    assert pkg.read_device_errors() == 0x2 and new.tolist() == [10]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


def test_evict_captured_and_on_two_streams(pkg):
    """Two captured evictions replayed side by side, three times on restored inputs, equal the
    eager ones."""
    bs, H, keep, recent = 64, 2, 100, 10
    cases = []
    for i, lens in enumerate(([300, 90], [700, 101])):
        nb = sum((n + bs - 1) // bs for n in lens)
        kp, vp = make_pool(pkg, 81 + i, nb, bs, H), dense_pool(83 + i, nb, bs, H, torch.bfloat16)
        kp, vp = (kp, kp.clone()) if i else (vp, vp.clone())
        cases.append([kp, vp, scores_for(85 + i, 2, H, 700, lens, "ties").cuda(),
                      torch.tensor(lens, dtype=torch.int32).cuda(), make_tables(87 + i, lens, bs, nb).cuda()])
    start = [[t.clone() for t in c[:3]] for c in cases]

    def restore():
        for c, s in zip(cases, start):
            for t, u in zip(c, s):
                t.copy_(u)
        torch.cuda.synchronize()

    want = []
    for c in cases:
        new, index = pkg.kv_evict(*c, keep, recent, return_index=True)
        want.append([t.clone() for t in c[:3]] + [new, index])
    graphs, got = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(pkg.kv_evict(*c, keep, recent, return_index=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        restore()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, w, (new, index) in zip(cases, want, got):
            for t, u in zip(c[:3] + [new, index], w):
                assert torch.equal(t, u)


def test_evict_then_attend(pkg):
    """A scored run as it is used: score, evict, decode on.  What remains attends as fp64
    attention over exactly the kept tokens."""
    bs, H, G, n, keep, recent = 64, 2, 4, 500, 120, 16
    kp, vp = make_pool(pkg, 71, 10, bs, H), make_pool(pkg, 72, 10, bs, H)
    tables = make_tables(73, [n], bs, 10)
    kv, vv = pool_values(kp), pool_values(vp)
    k, v = R.gather(kv, tables[0], n), R.gather(vv, tables[0], n)
    scores = torch.zeros(1, H, 512, device="cuda")
    ln = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.from_numpy(det_normal(74, (6, 1, 1, H * G, 128))).float().bfloat16()
    for i in range(5):
        pkg.flash_attn_with_kvcache_scored(q[i].cuda(), kp, vp, scores, ln, tables.cuda(), n)
    new, index = pkg.kv_evict(kp, vp, scores, ln, tables.cuda(), keep, recent, return_index=True)
    out = pkg.flash_attn_with_kvcache_int4(q[5].cuda(), kp, vp, new, tables.cuda()).cpu().double()
    for h in range(H):
        src = index[0, h].tolist()
        assert sorted(src)[-recent:] == list(range(n - recent, n)) and len(set(src)) == keep
        ref, _ = R.attend(q[5, 0, 0, h * G:(h + 1) * G], k[src, h:h + 1], v[src, h:h + 1], 128 ** -0.5)
        # 2^-8 for the bf16 output, 2^-11 for the rounded probabilities of values up to 4
        assert ((out[0, 0, h * G:(h + 1) * G] - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -11 * 4).all()
    assert (scores[0, :, keep:] == 0).all()


def test_evict_index_up_to_the_largest_keep(pkg):
    """keep 2^31 - 1 (keep everything, 8 GiB of index): the index fill ends with the buffer."""
    bs, keep, lens = 64, 2 ** 31 - 1, [100, 0]
    kp, vp = make_pool(pkg, 91, 2, bs, 1), make_pool(pkg, 92, 2, bs, 1)
    k0 = kp.clone()
    scores = torch.ones(2, 1, 128, device="cuda")
    tables = torch.tensor([[0, 1], [1, 0]], dtype=torch.int32, device="cuda")
    for b in range(2):
        new, index = pkg.kv_evict(kp, vp, scores[b:b + 1], torch.tensor(lens[b:b + 1], dtype=torch.int32).cuda(),
                                  tables[b:b + 1], keep, 0, return_index=True)
        torch.cuda.synchronize()
        assert new.tolist() == lens[b:b + 1]
        assert torch.equal(index[0, 0, :lens[b]].cpu(), torch.arange(lens[b], dtype=torch.int32))
        for at in range(lens[b], keep, 2 ** 29):
            assert (index[0, 0, at:at + 2 ** 29] == -1).all()
        del index
    assert torch.equal(kp, k0) and pkg.read_device_errors() == 0


@pytest.mark.parametrize("kind", ["normal", "ties", "odd", "zeros"])
def test_evict_past_one_group_of_words_a_warp(pkg, kind):
    """Rows of more than 32,768 tokens, where a warp ranks several groups of 32 words and
    carries its ties from one to the next; bytes compared exactly."""
    bs, H, lens, keep, recent = 256, 2, [41007, 70003, 32769], 9001, 130
    nb = sum((n + bs - 1) // bs for n in lens)
    width = max(lens)
    kp, vp = dense_pool(93, nb, bs, H, torch.bfloat16), dense_pool(94, nb, bs, H, torch.bfloat16)
    tables = make_tables(95, lens, bs, nb)
    scores = scores_for(96, 3, H, width, lens, kind)
    want_s, want_i = scores.clone(), torch.empty(3, H, keep, dtype=torch.int64)
    for b, n in enumerate(lens):
        for h in range(H):
            want_i[b, h] = torch.tensor(R.kept_index(scores[b, h].tolist(), n, keep, recent))
            want_s[b, h, :keep] = scores[b, h, want_i[b, h]]
            want_s[b, h, keep:n] = 0
    want = []
    for pool in (kp, vp):
        w, flat = pool.clone(), pool.flatten(0, 1)
        for b in range(3):
            t = tables[b].long().cuda()
            slot = lambda x: t[x // bs] * bs + x % bs
            for h in range(H):
                w.flatten(0, 1)[slot(torch.arange(keep).cuda()), h] = flat[slot(want_i[b, h].cuda()), h]
        want.append(w)
    gs = scores.cuda()
    new, index = pkg.kv_evict(kp, vp, gs, torch.tensor(lens, dtype=torch.int32).cuda(), tables.cuda(),
                              keep, recent, return_index=True)
    assert new.tolist() == [keep] * 3 and pkg.read_device_errors() == 0
    assert torch.equal(index.cpu().long(), want_i)
    assert torch.equal(gs.cpu().view(torch.int32), want_s.view(torch.int32))
    for pool, w in zip((kp, vp), want):
        assert torch.equal(pool.view(torch.int16), w.view(torch.int16))


@pytest.mark.parametrize("kind", ["dense", "int4"])
def test_scored_scratch_is_bounded_by_the_tables(pkg, kind):
    """The scratch goes by what the block tables reach, not by the score table's width (here
    1 GiB of it); the scores are those of a narrow table."""
    lens, H, G, bs = [200, 130, 1, 256], 1, 16, 64
    nb = sum((n + bs - 1) // bs for n in lens)
    kp, vp = (any_pool(pkg, kind, 15 + i, nb, bs, H, torch.bfloat16) for i in range(2))
    tables = make_tables(17, lens, bs, nb).cuda()
    q = torch.from_numpy(det_normal(18, (4, 1, H * G, 128))).float().bfloat16().cuda()
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    narrow = torch.zeros(4, H, 256, device="cuda")
    want = pkg.flash_attn_with_kvcache_scored(q, kp, vp, narrow, ln, tables)
    wide = torch.zeros(4, H, 2 ** 22, device="cuda")
    pkg.read_device_errors()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = pkg.flash_attn_with_kvcache_scored(q, kp, vp, wide, ln, tables)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 2 ** 26      # the decode's workspace, mostly
    assert torch.equal(out, want) and torch.equal(wide[:, :, :256], narrow)
    assert not wide[:, :, 256:].any() and pkg.read_device_errors() == 0
    # a context past the tables' reach is cut and flagged (and so is the padding of its table
    # row, which it runs over), as on a narrow table
    ln[2] = 300
    pkg.flash_attn_with_kvcache_scored(q, kp, vp, wide, ln, tables, decay=0.0)
    assert pkg.read_device_errors() == 0x6 and not wide[:, :, 256:].any()
    pkg.flash_attn_with_kvcache_scored(q, kp, vp, narrow, ln, tables, decay=0.0)
    assert pkg.read_device_errors() == 0x6 and torch.equal(wide[:, :, :256], narrow)
