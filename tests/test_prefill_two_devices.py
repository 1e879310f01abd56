"""The prefill entry points on a second device of one process.  The limit of dynamic shared
memory is an attribute of a function on one device; the host code runs here against a fake
runtime with two devices (tests/fake_cudart.cpp), without a GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "slo-aware-llm-serving-engine_b200", "csrc")
P = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def fake(pkg, tmp_path_factory):
    from importlib import import_module
    nvcc = import_module("slo-aware-llm-serving-engine_b200.build").nvcc_path()
    tmp = tmp_path_factory.mktemp("prefill")
    obj, lib = str(tmp / "paged_prefill.o"), str(tmp / "fake.so")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=compute_100a", "-std=c++17",
                    "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC", "-c",
                    os.path.join(CSRC, "paged_prefill.cu"), "-o", obj], check=True)
    include = os.path.join(os.path.dirname(os.path.dirname(nvcc)), "include")
    # -Bsymbolic: its calls meet the fake, not the runtime that torch has loaded
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I", include, "-o", lib,
                    os.path.join(ROOT, "tests", "fake_cudart.cpp"), obj, "-lpthread"], check=True)
    h = ctypes.CDLL(lib)
    sig = pkg._lib.SIGNATURES
    for name in ("slokv_paged_prefill", "slokv_paged_prefill_fp8"):
        getattr(h, name).restype, getattr(h, name).argtypes = sig[name]
    return h


def prefill(h, dtype, group):
    return h.slokv_paged_prefill(P, 128 * group, 128, P, 128 * group, 128, 200, P, P, 0, 0, 0, 16384, 16384,
                                 P, P, 1, 200, P, 2, 2, 2, 128, group, 1, 128, 0.1, dtype, None, None, 0,
                                 None, None)


def prefill_fp8(h, dtype, group):
    return h.slokv_paged_prefill_fp8(P, 128 * group, 128, P, 128 * group, 128, 200, P, P, 16384, 16384, P, P,
                                     P, P, 1, 200, P, 2, 2, 2, 128, group, 1, 128, 0.1, dtype, None, 0,
                                     None, None)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("call,group,regs", [   # the registers that the two-head kernels are built for
    (prefill, 1, 168), (prefill, 4, 168), (prefill_fp8, 4, 128)])
def test_each_device_gets_its_limit(fake, call, group, regs, dtype):
    for device in (0, 1, 0, 1):
        fake.fake_reset(device, regs, 0)
        before = fake.fake_launches()
        assert call(fake, dtype, group) == 0, device
        assert fake.fake_launches() > before
    sets = fake.fake_sets()
    for device in (0, 1):                                  # once a device and no more
        fake.fake_reset(device, regs, 0)
        assert call(fake, dtype, group) == 0
    assert fake.fake_sets() == sets


def test_a_failed_attribute_is_tried_again(fake):
    fake.fake_reset(3, 168, 1)
    assert prefill(fake, 0, 4) == -4
    fake.fake_reset(3, 168, 0)
    assert prefill(fake, 0, 4) == 0
    fake.fake_reset(70, 168, 0)                            # past the ids that are kept track of
    assert prefill(fake, 0, 4) == 0


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_int4_prefill_on_the_second_device(pkg):
    outs = []
    for d in range(2):
        dev = torch.device("cuda", d)
        g = torch.Generator().manual_seed(1)
        x = torch.randn(300, 2, 128, generator=g).bfloat16().to(dev)
        q = torch.randn(200, 8, 128, generator=g).bfloat16().to(dev)
        kp = torch.zeros(pkg.int4_pool_shape(5, 64, 2), dtype=torch.uint8, device=dev)
        vp = torch.zeros_like(kp)
        pkg.store_kvcache_int4(x, x + 1, kp, vp, torch.arange(300, dtype=torch.int32, device=dev))
        i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)
        outs.append(pkg.flash_attn_varlen_func_int4(q, kp, vp, i32(0, 200), i32(0, 300), 200, 300,
                                                    block_table=torch.arange(5, dtype=torch.int32,
                                                                             device=dev).view(1, 5)).cpu())
    assert torch.equal(*outs)
