"""Binding another pool, or making another runner, leaves nothing of the one before on the
attention modules (CPU: no kernel runs)."""
import importlib

import pytest
import torch

@pytest.mark.parametrize("order", [("fp8", "int4", "bf16"), ("int4", "fp8", "f16"), ("fp8", "bf16", "fp8")])
def test_bind_replaces_the_scales(pkg, order):
    mods = [pkg.Attention(4, 128, 0.1, 2) for _ in range(3)]
    for kind in order:
        pool = pkg.KVPool(3, 2, 64, 2, 128, kv_dtype=kind, device="cpu")
        pool.bind(mods)
        for i, m in enumerate(mods):
            assert m.k_cache.data_ptr() == pool.kv_cache[0, i].data_ptr()
            assert m.v_cache.data_ptr() == pool.kv_cache[1, i].data_ptr()
            if kind == "fp8":
                assert m.k_scale.data_ptr() == pool.k_scale[i].data_ptr()
                assert m.v_scale.data_ptr() == pool.v_scale[i].data_ptr()
            else:
                assert m.k_scale is None and m.v_scale is None


@pytest.mark.parametrize("score", [False, True])
def test_runner_takes_over_the_score_table(pkg, score):
    """A runner scores its batch row by row and without decay, whatever the modules' score
    table was mapped by before."""
    h = importlib.import_module("slo-aware-llm-serving-engine_b200.qwen3_harness")
    cfg = h.Qwen3Config(vocab_size=97, hidden_size=64, intermediate_size=96, num_layers=2, num_heads=4,
                        num_kv_heads=2, head_dim=16, max_position=256)
    model = h.Qwen3Model(cfg, seed=3, device="cpu", dtype=torch.float32)
    for attn in model.attention_modules():
        attn.scores = torch.zeros(7, 2, 9)
        attn.score_rows = torch.tensor([6, 1, 0], dtype=torch.int32)
        attn.score_decay = 0.5
    run = h.GreedyRunner(model, [5, 11, 1], 4, block_size=64, score=score)
    for i, attn in enumerate(model.attention_modules()):
        assert attn.score_rows is None and attn.score_decay == 1.0
        if score:
            assert attn.scores.data_ptr() == run.scores[i].data_ptr()
        else:
            assert attn.scores is None
