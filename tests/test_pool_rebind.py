"""Binding another pool leaves nothing of the one before on the attention modules (CPU: no
kernel runs)."""
import pytest

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
