"""The 4-bit pool and eviction as the layers and the runner use them: Attention and
forward_mixed over a 4-bit pool, KVPool, and a scored run with evictions in between.
Each attention call is checked against 64-bit attention on what its pool holds, with
the bounds of test_gpu_int4.py."""
import pytest
import torch

from tests import int4_reference as R
from tests.golden.detgen import det_normal
from tests.test_gpu_int4 import check_decode, make_pool, make_tables

pytestmark = pytest.mark.gpu


def attention(pkg, H, G, bs, nb, seed=0):
    attn = pkg.Attention(H * G, 128, 128 ** -0.5, H)
    attn.k_cache, attn.v_cache = make_pool(pkg, seed, nb, bs, H, 0.5), make_pool(pkg, seed + 1, nb, bs, H)
    return attn


def rows(seed, T, H, G):
    x = torch.from_numpy(det_normal(seed, (T, H * (G + 2), 128))).float().bfloat16().cuda()
    return x[:, :H * G], x[:, H * G:H * G + H], x[:, H * G + H:]


def check_varlen(out, q, k, v, tables, qlens, klens, half=2.0 ** -8):
    """Bound as in test_gpu_int4.test_varlen; k, v: fp64 values [NB, bs, H, 128] or lists of rows."""
    at, G = 0, q.shape[1] // (k[0].shape[1] if isinstance(k, list) else k.shape[2])
    out, q = out.cpu().double(), q.cpu()
    for b, (nq, nk) in enumerate(zip(qlens, klens)):
        kk = k[b] if isinstance(k, list) else R.gather(k, tables[b], nk).bfloat16().double()
        vv = v[b] if isinstance(v, list) else R.gather(v, tables[b], nk).bfloat16().double()
        for i in range(nq):
            n = nk - nq + i + 1
            ref, w = R.attend(q[at + i], kk[:n], vv[:n], 128 ** -0.5)
            wv = torch.einsum("hn,nhd->hd", w, vv[:n].repeat_interleave(G, 1).abs())
            assert ((out[at + i] - ref).abs() <= (2 * half + 2.0 ** -13) * wv + 2.0 ** -25).all()
        at += nq


def test_attention_prefill_decode_mixed(pkg):
    H, G, bs, nb = 2, 4, 128, 12
    attn = attention(pkg, H, G, bs, nb)
    tables = make_tables(3, [400, 300], bs, nb)
    slot = lambda b, t: int(tables[b, t // bs]) * bs + t % bs
    cu = lambda x: torch.tensor([0] + torch.tensor(x).cumsum(0).tolist(), dtype=torch.int32).cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    values = lambda: (R.decode_pool(attn.k_cache.cpu())[0], R.decode_pool(attn.v_cache.cpu())[0])

    # cold prompts attend on their own rows and are stored quantised
    q, k, v = rows(10, 150, H, G)
    slots = [slot(0, t) for t in range(100)] + [slot(1, t) for t in range(50)]
    pkg.set_context(True, cu([100, 50]), cu([100, 50]), 100, 100, i32(slots), None, None)
    out = attn(q, k, v)
    pkg.reset_context()
    own = [x.cpu().double() for x in (k[:100], k[100:])], [x.cpu().double() for x in (v[:100], v[100:])]
    check_varlen(out, q, own[0], own[1], None, [100, 50], [100, 50])
    want = torch.zeros_like(attn.k_cache.cpu()), torch.zeros_like(attn.v_cache.cpu())
    R.store(k.cpu(), v.cpu(), want[0], want[1], torch.tensor(slots), bs)
    kv, vv = values()
    wk, wv = R.decode_pool(want[0])[0], R.decode_pool(want[1])[0]
    for s in slots:
        assert torch.equal(kv[s // bs, s % bs], wk[s // bs, s % bs])
        assert torch.equal(vv[s // bs, s % bs], wv[s // bs, s % bs])

    # a chunk with cached history
    q, k, v = rows(11, 70, H, G)
    slots = [slot(0, 90 + t) for t in range(50)] + [slot(1, 50 + t) for t in range(20)]
    pkg.set_context(True, cu([50, 20]), cu([140, 70]), 50, 140, i32(slots), None, tables.cuda())
    out = attn(q, k, v)
    pkg.reset_context()
    check_varlen(out, q, *values(), tables, [50, 20], [140, 70])

    # a decode step, not scored and scored: the same outputs
    q, k, v = rows(12, 2, H, G)
    pkg.set_context(False, None, None, 0, 0, i32([slot(0, 140), slot(1, 70)]), i32([141, 71]), tables.cuda())
    out = attn(q, k, v)
    attn.scores = torch.zeros(3, H, 200, device="cuda")
    attn.score_rows = i32([2, 0])
    assert torch.equal(attn(q, k, v), out)
    pkg.reset_context()
    check_decode(out, q.unsqueeze(1).cpu(), attn.k_cache, attn.v_cache, [141, 71], tables, 128 ** -0.5)
    # every head's weights sum to 1: G a KV head (150 keys, each within 2^-20 or so of itself)
    total = attn.scores.sum(-1).cpu()
    assert ((total[[2, 0]] - G).abs() < G * 2.0 ** -16).all() and (total[1] == 0).all()

    # one decode row and a prefill row with history in one step
    q, k, v = rows(13, 31, H, G)
    slots = [slot(0, 141)] + [slot(1, 71 + t) for t in range(30)]
    attn.score_rows = i32([1])
    meta = pkg.MixedAttentionContext(1, 30, i32([142]), tables[:1].cuda(), cu([30]), cu([101]),
                                     tables[1:].cuda(), 30, 101, True)
    pkg.set_context(False, None, None, 0, 0, i32(slots), None, None)
    pkg.get_context().mixed = meta
    out = attn(q, k, v)
    pkg.reset_context()
    check_decode(out[:1].unsqueeze(1), q[:1].unsqueeze(1).cpu(), attn.k_cache, attn.v_cache, [142], tables,
                 128 ** -0.5)
    check_decode(out[1:].unsqueeze(1), q[1:].unsqueeze(1).cpu(), attn.k_cache, attn.v_cache,
                 list(range(72, 102)), tables[1:].expand(30, -1), 128 ** -0.5)
    assert ((attn.scores[1].sum(-1).cpu() - G).abs() < G * 2.0 ** -16).all()
    assert pkg.read_device_errors() == 0


def test_pool_copies_and_swaps_int4_pages(pkg):
    pool = pkg.KVPool(2, 6, 64, 2, 128, kv_dtype="int4")
    assert pool.kv_cache.shape == (2, 2, 6, 2, 64 * 72)
    assert pool.kv_cache.numel() == 6 * pkg.block_bytes(2, 64, 2, 128, "int4")
    mods = [pkg.Attention(8, 128, 0.1, 2) for _ in range(2)]
    assert pool.bind(mods) == 2
    x = torch.from_numpy(det_normal(1, (64, 2, 128))).float().bfloat16().cuda()
    for m in mods:
        pkg.store_kvcache_int4(x, -x, m.k_cache, m.v_cache,
                               torch.arange(64, 128, dtype=torch.int32, device="cuda"))
    ids = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    pool.copy_blocks(ids(1), ids(4))
    saved = pool.swap_out(ids(4))
    pool.swap_in(saved, ids(0))
    for m in mods:
        for c, want in ((m.k_cache, x), (m.v_cache, -x)):
            near = pkg.int4_decode(c, torch.arange(64, dtype=torch.int32, device="cuda"))
            same = pkg.int4_decode(c, torch.arange(64, 128, dtype=torch.int32, device="cuda"))
            assert torch.equal(near, same)
            # half a step: the range of 64 normals below 8, in 15 steps, and the scale's rounding
            assert (near - want.float()).abs().max() < 8 / 15 * (0.5 + 15 * 2.0 ** -8)


def tiny(pkg):
    from importlib import import_module
    H = import_module("slo-aware-llm-serving-engine_b200.qwen3_harness")
    cfg = H.Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_layers=2, num_heads=4,
                        num_kv_heads=2, head_dim=128, max_position=512)
    return H, H.Qwen3Model(cfg, seed=5)


@pytest.mark.parametrize("kv_dtype", ["bf16", "int4"])
def test_runner_scores_and_evicts(pkg, kv_dtype):
    """Two runs of the same steps, eager and replayed from a graph, with an eviction in the
    middle: equal tokens, scores and cache lengths, and positions that go on counting."""
    H, model = tiny(pkg)
    prompts = [[3, 7, 11] * 20, [5] * 33, [9, 1]]
    got = []
    for use_graph in (False, True):
        run = H.GreedyRunner(model, [60, 33, 2], 40, block_size=64, kv_dtype=kv_dtype, score=True)
        tok = run.prefill(prompts)
        seq = [tok.tolist()]
        for step in range(12):
            tok = run.decode(tok, use_graph=use_graph)
            seq.append(tok.tolist())
            if step == 5:
                assert run.evict(40, 8).tolist() == [40, 39, 8]
                assert run.cached.tolist() == [40, 39, 8] and run.pos.tolist() == [66, 39, 8]
        assert run.cached.tolist() == [46, 45, 14] and run.pos.tolist() == [72, 45, 14]
        assert (run.scores[:, 0, :, 46:] == 0).all()
        got.append((seq, run.scores.clone()))
        run.release()
    assert got[0][0] == got[1][0] and torch.equal(got[0][1], got[1][1])
    # each head spreads a weight of 1 a step over the cached tokens: 12 steps x 2 heads a KV
    # head, less what was evicted with the tokens that held it
    total = got[0][1].sum(-1)
    assert (total <= 24 * (1 + 2.0 ** -16)).all() and (total[:, 1:] >= 24 * (1 - 2.0 ** -16)).all()
    assert (total[:, 0] >= 12).all()


def test_runner_int4_attention_is_its_pools(pkg):
    """Every decode of an int4 run is 64-bit attention on the 4-bit values in its pool."""
    H, model = tiny(pkg)
    run = H.GreedyRunner(model, [70, 5], 8, block_size=64, kv_dtype="int4")
    tok = run.prefill([list(range(70)), [1, 2, 3, 4, 5]])
    seen = []

    class Spy(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner, self.k_cache, self.k_scale = inner, inner.k_cache, None

        def forward(self, q, k, v):
            out = self.inner(q, k, v)
            seen.append((q.clone(), out.clone(), self.inner.k_cache.clone(), self.inner.v_cache.clone()))
            return out

    for lw in model.layers:
        lw.attn = Spy(lw.attn)
    run.decode(tok, use_graph=False)
    assert len(seen) == 2
    for q, out, kp, vp in seen:
        check_decode(out.view(2, 1, 4, 128), q.unsqueeze(1).cpu(), kp, vp, [71, 6], run.tables.cpu(), 128 ** -0.5)


def test_fp8_pools_are_not_scored(pkg):
    attn = pkg.Attention(4, 128, 0.1, 2)
    attn.k_cache = attn.v_cache = torch.zeros(2, 64, 2, 128, dtype=torch.uint8, device="cuda")
    attn.k_scale = attn.v_scale = torch.zeros(2, 2, device="cuda")
    attn.scores = torch.zeros(1, 2, 64, device="cuda")
    q, k, v = rows(1, 1, 2, 2)
    with pytest.raises(RuntimeError, match="FP8"):
        attn(q, k, v)
