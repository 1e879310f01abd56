"""4-bit KV pool on the GPU: store, read-back, decode and prefill attention against 64-bit
restatements (tests/int4_reference.py).

Tolerances.  Stored bytes are compared exactly.  Decode (derived from the kernel's
arithmetic, u = 2^-24, half a step of fp32):
  * p s is rounded to f16, to two f16 for f16 outputs: 2^-11 or 2^-22 of sum_t w_t s_t c_t
    (plus nothing below 2^-29 of the largest value, which the cases do not reach; the second
    f16's own smallest step is 2^-25 against a largest p s of 2^14 at least, so another
    2^-38 of the largest value a token);
  * an error e in a score changes its weight by a factor within 1 +- 2 e: e <= (128 + 16)
    products and sums in fp32, each within u of their absolute sum, so e <= 400 u
    scale sum_d |q_d| (15 s + |m|) with the tensor core's truncation counted double;
    the exponential adds 2^-21;  out moves by at most (2 e + 2^-20) sum_t w_t |v_t|;
  * accumulating sum r c over n tokens: one rounding (2 u, the MMA truncates) per 16 tokens
    and per tile of a running sum that is moved out every 512 tokens, and so at most 15 times
    these tokens' sum w s (odd dims: the difference of sums of at most 255 and 15, divided
    by 16, so 17); the moves add u of the whole each: ((512 / 16 + 40) 2 u 32 + (n / 512 +
    2) u 17) sum_t w_t s_t; and (n / 8 + 40) 2 u for a lane's sum p |m|;
  * the output's own rounding: 2^-8 (bf16) or 2^-11 (f16) of the value, and f16's
    smallest step 2^-25.
"""
import numpy as np
import pytest
import torch

from tests import int4_reference as R
from tests.golden.detgen import det_ints, det_normal, det_perm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def make_pool(pkg, seed, nb, bs, h, amp=1.0, bias=0.0):
    """Random pool content (K or V side) on the CPU through the reference encoder's rules,
    vectorised: every slot holds an encoded row."""
    x = torch.from_numpy(det_normal(seed, (nb * bs, h, 128))).float() * amp + bias
    x = x.bfloat16()
    pool = torch.zeros(pkg.int4_pool_shape(nb, bs, h), dtype=torch.uint8, device="cuda")
    other = torch.zeros_like(pool)
    slots = torch.arange(nb * bs, dtype=torch.int32, device="cuda")
    pkg.store_kvcache_int4(x.cuda(), x.cuda(), pool, other, slots)
    torch.cuda.synchronize()
    assert torch.equal(pool, other)
    return pool


def make_tables(seed, lens, bs, nb, width=None):
    pages = [(max(0, n) + bs - 1) // bs for n in lens]
    w = width or max(1, max(pages))
    perm = det_perm(seed, nb).tolist()
    assert sum(pages) <= nb
    t, cur = [], 0
    for n in pages:
        t.append(perm[cur:cur + n] + [-1] * (w - n))
        cur += n
    return torch.tensor(t, dtype=torch.int32)


def decode_bound(q, k, v, ks, vs, kmin_abs, w, out, scale, dtype):
    """The bound of the module docstring for one sequence; everything fp64.
    q [Hq,128], k/v [n,H,128], ks/vs scales [n,H,2], w [Hq,n], out [Hq,128]."""
    Hq, n = w.shape
    G = Hq // k.shape[1]
    rep = lambda x: x.repeat_interleave(G, 1)
    s_dim = rep(vs).repeat_interleave(64, -1)                       # [n, Hq, 128]
    vv = rep(v)
    vmin = rep(kmin_abs[1]).repeat_interleave(64, -1)
    above = (vv - vmin).abs()                                       # s c
    k_abs = rep(kmin_abs[0].abs() + 15 * ks).repeat_interleave(64, -1)
    e = 400 * U * abs(scale) * torch.einsum("hd,nhd->hn", q.double().abs(), k_abs).max(-1).values
    wv = torch.einsum("hn,nhd->hd", w, vv.abs())
    ws = torch.einsum("hn,nhd->hd", w, s_dim)
    wz = torch.einsum("hn,nhd->hd", w, vmin.abs())
    wc = torch.einsum("hn,nhd->hd", w, above)
    if dtype == torch.float16:
        b = 2.0 ** -22 * wc + n * 2.0 ** -38 * 15 * torch.maximum(s_dim, vmin.abs()).amax((0, 2)).unsqueeze(-1)
    else:
        b = 2.0 ** -11 * wc
    b = b + (2 * e + 2.0 ** -20).unsqueeze(-1) * wv
    b = b + ((512 / 16 + 40) * 2 * U * 32 + (n / 512 + 2) * U * 17) * ws + (n / 8 + 40) * 2 * U * wz
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    return b + half * (out.abs() + b) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)


def mins_of(pool):
    """minimum parameters [NB, bs, H, 2] of a CPU pool, fp64."""
    nb, h, size = pool.shape
    t = pool.numpy().reshape(nb, h, size // 4608, 4608)[..., 4096:]
    bits = np.ascontiguousarray(t).view(np.uint16).reshape(nb, h, -1, 64, 4)[..., 1::2]
    f = (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return torch.from_numpy(f).reshape(nb, h, -1, 2).transpose(1, 2)


def check_decode(out, q, kp, vp, lens, tables, scale):
    kp, vp = kp.cpu(), vp.cpu()
    kv, ks = R.decode_pool(kp)
    vv, vs = R.decode_pool(vp)
    km, vm = mins_of(kp), mins_of(vp)
    out = out.cpu().double()
    assert out.shape == q.shape
    for b, n in enumerate(lens):
        if n <= 0:
            assert (out[b] == 0).all()
            continue
        g = lambda x: R.gather(x, tables[b], n)
        k, v = g(kv), g(vv)
        ref, w = R.attend(q[b, 0], k, v, scale)
        bound = decode_bound(q[b, 0], k, v, g(ks), g(vs), (g(km), g(vm)), w, ref, scale, q.dtype)
        err = (out[b, 0] - ref).abs()
        bad = ~(err <= bound)
        assert not bad.any(), (b, n, err[bad].max().item(), bound[bad].min().item())


# ---- store and read-back --------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,bs", [(1, 1, 64), (5, 3, 64), (17, 8, 192), (33, 2, 128)])
def test_store_bytes(pkg, dtype, T, H, bs):
    nb = 3
    k = (torch.from_numpy(det_normal(T * 7 + H, (T, H, 128))).float() * 3).to(dtype)
    v = (torch.from_numpy(det_normal(T * 7 + H + 1, (T, H, 128))).float() + 5).to(dtype)
    slots = torch.from_numpy(det_perm(T + bs, nb * bs)[:T].astype(np.int32))
    if T > 4:
        slots[2] = -1
    shape = pkg.int4_pool_shape(nb, bs, H)
    kp = torch.full(shape, 0xA5, dtype=torch.uint8)
    vp = torch.full(shape, 0x5A, dtype=torch.uint8)
    gk, gv = kp.cuda(), vp.cuda()
    pkg.store_kvcache_int4(k.cuda(), v.cuda(), gk, gv, slots.cuda())
    assert R.store(k, v, kp, vp, slots, bs)
    assert torch.equal(gk.cpu(), kp) and torch.equal(gv.cpu(), vp)   # all else is left as it was
    got = pkg.int4_decode(gk, slots.cuda()).cpu()
    vals, _ = R.decode_pool(kp)
    for t, s in enumerate(slots.tolist()):
        want = vals[s // bs, s % bs].float() if s >= 0 else torch.zeros(H, 128)
        assert torch.equal(got[t], want)
    assert pkg.read_device_errors() == 0


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_store_strided_and_unaligned(pkg, shift, dtype):
    T, H, bs = 9, 2, 64
    raw = torch.from_numpy(det_normal(5, (T * 6 * H * 128 + 64,))).float().to(dtype).cuda()
    rows = raw[shift:shift + T * 6 * H * 128].view(T, 6 * H, 128)
    k, v = rows[:, 4 * H:5 * H], rows[:, 1:1 + 2 * H:2]              # heads apart by 256 too
    kp = torch.zeros(pkg.int4_pool_shape(2, bs, H), dtype=torch.uint8)
    vp = torch.zeros_like(kp)
    gk, gv = kp.cuda(), vp.cuda()
    slots = torch.tensor([3, 70, 64, 127, 0, -1, 9, 8, 63], dtype=torch.int32)
    pkg.store_kvcache_int4(k, v, gk, gv, slots.cuda())
    R.store(k.cpu(), v.cpu(), kp, vp, slots, bs)
    assert torch.equal(gk.cpu(), kp) and torch.equal(gv.cpu(), vp)


def test_store_special_groups(pkg):
    """Constant, zero, denormal, huge and non-finite groups; a NaN stays within its group."""
    x = torch.zeros(10, 1, 128)
    x[0] = 2.5                                        # constant: scale 0
    x[2] = torch.linspace(-3e38, 3e38, 128)           # torch's own step overflows: not finite
    x[3, 0, :64] = torch.linspace(-3e38, 3.3e38, 64)  # the range overflows fp32
    x[4, 0, 70] = float("nan")
    x[5, 0, 3] = float("inf")
    x[6] = torch.linspace(0, 1e-38, 128)
    x[7, 0, :64] = -0.0
    x[7, 0, 64:] = torch.arange(64) * 0.5             # 31.5 / 15: ties included
    x[8, 0, ::2] = 1e-30
    x[9] = torch.linspace(-3e38, 3e38, 128, dtype=torch.float64).float()  # a group's range is 3e38
    x = x.bfloat16()
    kp = torch.zeros(pkg.int4_pool_shape(1, 64, 1), dtype=torch.uint8)
    vp = torch.zeros_like(kp)
    gk, gv = kp.cuda(), vp.cuda()
    slots = torch.arange(10, dtype=torch.int32)
    pkg.read_device_errors()
    pkg.store_kvcache_int4(x.cuda(), x.cuda(), gk, gv, slots.cuda())
    assert not R.store(x, x, kp, vp, slots, 64)
    got, want = pkg.int4_decode(gk, slots.cuda()).cpu(), R.decode_pool(kp)[0][0, :10].float()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    assert got[4, 0, 64:].isnan().all() and torch.equal(got[4, 0, :64], torch.zeros(64))
    assert got[3, 0, :64].isnan().all() and got[5, 0, :64].isnan().all()
    assert torch.equal(got[0], torch.full((1, 128), 2.5)) and torch.equal(got[1], torch.zeros(1, 128))
    assert pkg.read_device_errors() == 0x10
    # half a step from the value everywhere (a step is the scale; the scale and the minimum are rounded)
    for r in (6, 7, 9):
        for g in range(2):
            v = x[r, 0, 64 * g:64 * g + 64].double()
            step = (v.max() - v.min()) / 15
            err = (got[r, 0, 64 * g:64 * g + 64].double() - v).abs().max()
            # half a step of the rounded scale, 15 times its rounding, and a denormal step of bf16
            assert err <= step * (0.5 + 15 * 2.0 ** -8) * (1 + 2.0 ** -8) + 2.0 ** -133 * 8


def test_store_slot_out_of_range(pkg):
    k = torch.ones(4, 2, 128, dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros(pkg.int4_pool_shape(2, 64, 2), dtype=torch.uint8, device="cuda")
    slots = torch.tensor([128, -2, 2 ** 31 - 1, 5], dtype=torch.int32, device="cuda")
    pkg.read_device_errors()
    pkg.store_kvcache_int4(k, k, pool, pool.clone(), slots)
    assert pkg.read_device_errors() == 0x1
    want = torch.zeros(2, 2, 64 * 72, dtype=torch.uint8)
    R.store(k.cpu()[3:], k.cpu()[3:], want, want.clone(), slots.cpu()[3:], 64)
    assert torch.equal(pool.cpu(), want)
    got = pkg.int4_decode(pool, slots)
    assert pkg.read_device_errors() == 0x1
    assert (got[:3] == 0).all() and (got[3] == 1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("amp,bias", [(0.5, 0), (0.5, 4), (0.5, 16), (0.5, 64), (0.5, -64), (3.0, 1000),
                                      (1e-3, -1000), (200.0, 100)])
def test_store_offset_rows(pkg, dtype, amp, bias):
    """How far a stored value lies from its input, with R the group's range and s its scale.  A code
    that is not clamped is half a step s off.  The minimum may be 2^-8 |min| off (bf16 rows: not
    at all) and 15 s below R by 2^-8 R, so a clamped one is 2^-8 (|min| + R) off at most, which is
    less than half a step while |min| <= 7 R: s / 2 >= R / 30 (1 - 2^-8) > 0.033 R and 2^-8 8 R
    < 0.0313 R.  The quotient is 2^-20 of a step off its border, the fp32 value 2^-24 of itself."""
    T, H, bs = 24, 2, 64
    x = (torch.from_numpy(det_normal(int(abs(bias)) + 3, (T, H, 128))).float() * amp + bias).to(dtype)
    kp = torch.zeros(pkg.int4_pool_shape(1, bs, H), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    pkg.store_kvcache_int4(x.cuda(), x.cuda(), kp, vp, slots)
    got = pkg.int4_decode(kp, slots).cpu().double().view(T, H, 2, 64)
    scale = R.decode_pool(kp.cpu())[1][0, :T].unsqueeze(-1)               # [T, H, 2, 1]
    v = x.double().view(T, H, 2, 64)
    low = v.amin(-1, keepdim=True)
    span, low = v.amax(-1, keepdim=True) - low, low.abs()
    clamped = 2.0 ** -8 * ((low if dtype != torch.bfloat16 else 0) + span)
    half = 0.5 * scale * (1 + 2.0 ** -19)
    bound = torch.where(low <= 7 * span, half, torch.maximum(half, clamped))
    if dtype == torch.bfloat16:
        bound = half.expand_as(span)
    assert ((got - v).abs() <= bound + 2.0 ** -23 * v.abs()).all()


# ---- decode ----------------------------------------------------------------------

LENS = [[1], [64, 65, 63, 0, 1, 128], [0, 0], [700, 5, 1023, 0, 129], [4500]]


@pytest.mark.parametrize("lens", LENS, ids=[str(i) for i in range(len(LENS))])
@pytest.mark.parametrize("H,G,bs,dtype", [(1, 1, 64, torch.bfloat16), (2, 4, 256, torch.bfloat16),
                                          (3, 5, 192, torch.float16), (2, 8, 128, torch.float16),
                                          (1, 16, 64, torch.bfloat16), (2, 9, 128, torch.float16)])
def test_decode(pkg, lens, H, G, bs, dtype):
    nb = sum((n + bs - 1) // bs for n in lens) + 3
    kp, vp = make_pool(pkg, 11, nb, bs, H, 0.7), make_pool(pkg, 12, nb, bs, H, 1.0, 0.3)
    tables = make_tables(13, lens, bs, nb)
    q = torch.from_numpy(det_normal(14, (len(lens), 1, H * G, 128))).float().to(dtype)
    pkg.read_device_errors()
    out = pkg.flash_attn_with_kvcache_int4(q.cuda(), kp, vp, torch.tensor(lens, dtype=torch.int32).cuda(),
                                           tables.cuda())
    check_decode(out, q, kp, vp, lens, tables, 128 ** -0.5)
    assert pkg.read_device_errors() == 0


def test_decode_many_rows_and_batch_prefix(pkg):
    """More rows than warps, empty ones among them, and a scale that is not the default."""
    lens = [int(x) for x in det_ints(3, 301, 0, 90)]
    lens[0] = lens[7] = lens[8] = lens[9] = lens[10] = lens[300] = 0
    bs, H, G = 64, 1, 2
    nb = sum((n + bs - 1) // bs for n in lens)
    kp, vp = make_pool(pkg, 21, nb, bs, H), make_pool(pkg, 22, nb, bs, H)
    tables = make_tables(23, lens, bs, nb)
    q = torch.from_numpy(det_normal(24, (301, 1, 2, 128))).float().bfloat16()
    for scale in (0.3, -0.05, 0.0):
        out = pkg.flash_attn_with_kvcache_int4(q.cuda(), kp, vp,
                                               torch.tensor(lens, dtype=torch.int32).cuda(),
                                               tables.cuda(), softmax_scale=scale)
        check_decode(out, q, kp, vp, lens, tables, scale)


def test_decode_batch_limit_and_long_gaps(pkg):
    """8,192 rows, all but three without tokens, one of them long: ranges cross the gaps."""
    bs, H, G, B = 64, 1, 1, 8192
    lens = [0] * B
    lens[5], lens[4000], lens[8191] = 130, 20000, 65
    nb = sum((n + bs - 1) // bs for n in lens)
    kp, vp = make_pool(pkg, 25, nb, bs, H), make_pool(pkg, 26, nb, bs, H)
    short = make_tables(27, [130, 20000, 65], bs, nb)
    tables = torch.full((B, short.shape[1]), -1, dtype=torch.int32)
    tables[[5, 4000, 8191]] = short
    q = torch.from_numpy(det_normal(28, (B, 1, 1, 128))).float().bfloat16()
    out = pkg.flash_attn_with_kvcache_int4(q.cuda(), kp, vp, torch.tensor(lens, dtype=torch.int32).cuda(),
                                           tables.cuda())
    check_decode(out, q, kp, vp, lens, tables, 128 ** -0.5)
    assert pkg.read_device_errors() == 0


def test_decode_stale_and_foreign_bytes(pkg):
    """0xFF bytes (NaN parameters) in every slot that no sequence reaches change nothing."""
    lens, bs, H, G = [65, 130, 1], 128, 2, 4
    nb = 6
    kp, vp = make_pool(pkg, 31, nb, bs, H), make_pool(pkg, 32, nb, bs, H)
    tables = make_tables(33, lens, bs, nb)
    live = torch.zeros(nb, bs, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            live[tables[b, t // bs], t % bs] = True
    for pool in (kp, vp):
        for blk in range(nb):
            for off in range(bs):
                if not live[blk, off]:
                    c0, p0 = R.row_offsets(off)
                    pool[blk, :, c0:c0 + 64] = 0xFF
                    pool[blk, :, p0:p0 + 8] = 0xFF
    q = torch.from_numpy(det_normal(34, (3, 1, 8, 128))).float().bfloat16()
    out = pkg.flash_attn_with_kvcache_int4(q.cuda(), kp, vp, torch.tensor(lens, dtype=torch.int32).cuda(),
                                           tables.cuda())
    assert torch.isfinite(out).all()
    check_decode(out, q, kp, vp, lens, tables, 128 ** -0.5)


def test_decode_strides_out_and_wide_tables(pkg):
    lens, bs, H, G = [100, 300], 128, 2, 4
    nb = 5
    big_k = make_pool(pkg, 41, 2 * nb, bs, H)
    big_v = make_pool(pkg, 42, 3 * nb, bs, H)
    kp, vp = big_k[::2], big_v[1::3]                                  # strided blocks
    tables = torch.full((4, 9), 77, dtype=torch.int32)
    tables[:2, :3] = make_tables(43, lens, bs, nb, 3)
    tables = tables[:, :7]                                            # rows apart by 9
    q = torch.from_numpy(det_normal(44, (2, 1, 20, 128))).float().half()[:, :, 4:20:2]
    store = torch.full((2, 1, 10, 128), 9.0, dtype=torch.float16, device="cuda")
    out = store[:, :, 1:9]
    gq = q.cuda().as_strided(q.shape, q.stride()) if q.is_contiguous() else \
        torch.from_numpy(det_normal(44, (2, 1, 20, 128))).float().half().cuda()[:, :, 4:20:2]
    res = pkg.flash_attn_with_kvcache_int4(gq, kp, vp, torch.tensor(lens, dtype=torch.int32).cuda(),
                                           tables.cuda(), out=out)
    assert res.data_ptr() == out.data_ptr()
    check_decode(out, q, kp.contiguous(), vp.contiguous(), lens, tables, 128 ** -0.5)
    assert (store[:, :, 0] == 9).all() and (store[:, :, 9] == 9).all()


def test_decode_bad_metadata_is_flagged(pkg):
    """A block id outside the pool reads as zeros; a context past the table is cut."""
    lens, bs, H, G = [200, 100], 64, 1, 4
    nb = 8
    kp, vp = make_pool(pkg, 51, nb, bs, H), make_pool(pkg, 52, nb, bs, H)
    tables = torch.tensor([[1, 99, 3, 4], [-7, 5, 0, 0]], dtype=torch.int32)
    q = torch.from_numpy(det_normal(54, (2, 1, 4, 128))).float().bfloat16()
    pkg.read_device_errors()
    out = pkg.flash_attn_with_kvcache_int4(q.cuda(), kp, vp, torch.tensor(lens, dtype=torch.int32).cuda(),
                                           tables.cuda())
    assert pkg.read_device_errors() == 0x2
    check_decode(out, q, kp, vp, lens, tables, 128 ** -0.5)
    out = pkg.flash_attn_with_kvcache_int4(q.cuda()[:1], kp, vp,
                                           torch.tensor([10 ** 9], dtype=torch.int32).cuda(),
                                           torch.tensor([[1, 2]], dtype=torch.int32).cuda())
    assert pkg.read_device_errors() == 0x4
    check_decode(out, q[:1], kp, vp, [128], torch.tensor([[1, 2]]), 128 ** -0.5)


def test_decode_value_range(pkg):
    """V rows whose scales differ by 2^20 between tokens, large and tiny q, a group without
    spread and a large bias: no value is lost to f16's range."""
    bs, H, n = 64, 1, 64
    k = torch.from_numpy(det_normal(61, (n, H, 128))).float()
    v = torch.from_numpy(det_normal(62, (n, H, 128))).float()
    v[:8] *= 2.0 ** 20
    v[9] = 1000.0
    k[:8] -= 3.0                                       # the large values are looked at least
    k, v = k.bfloat16(), v.bfloat16()
    kp = torch.zeros(pkg.int4_pool_shape(1, bs, H), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    pkg.store_kvcache_int4(k.cuda(), v.cuda(), kp, vp, torch.arange(n, dtype=torch.int32, device="cuda"))
    tables = torch.zeros(4, 1, dtype=torch.int32)
    q = torch.full((4, 1, 2, 128), 1.0)
    q[1] = 2.0 ** 100
    q[2] = 2.0 ** -100
    q[3] = 0.0
    q = (q * torch.from_numpy(det_normal(63, (4, 1, 2, 128))).float().abs()).bfloat16()
    for i, scale in ((0, 0.05), (1, 2.0 ** -104), (2, 2.0 ** 96), (3, 1.0)):
        out = pkg.flash_attn_with_kvcache_int4(q[i:i + 1].cuda(), kp, vp,
                                               torch.tensor([n], dtype=torch.int32).cuda(),
                                               tables[:1].cuda(), softmax_scale=scale)
        check_decode(out, q[i:i + 1], kp, vp, [n], tables[:1], scale)


def test_decode_values_all_zero(pkg):
    """Thousands of tokens whose V rows are all zero (the reference that the scores are taken
    against then lies far above the others'), alone and before rows that are not."""
    bs, n = 256, 9000
    nb = (n + bs - 1) // bs
    kp = make_pool(pkg, 65, nb, bs, 1)
    vp = torch.zeros_like(kp)
    tables = torch.arange(nb, dtype=torch.int32).view(1, -1)
    q = torch.from_numpy(det_normal(66, (1, 1, 2, 128))).float().bfloat16()
    ln = torch.tensor([n], dtype=torch.int32).cuda()
    scores = torch.zeros(1, 1, n, device="cuda")
    out = pkg.flash_attn_with_kvcache_scored(q.cuda(), kp, vp, scores, ln, tables.cuda())
    assert (out == 0).all() and abs(scores.sum().item() - 2) < 2 * 2.0 ** -16
    one = make_pool(pkg, 67, 1, bs, 1)
    vp[nb - 1] = one[0]
    out = pkg.flash_attn_with_kvcache_int4(q.cuda(), kp, vp, ln, tables.cuda())
    check_decode(out, q, kp, vp, [n], tables, 128 ** -0.5)


def test_decode_long_uniform_attention(pkg):
    """The mean of 19,000 random V rows, each head's in one warp's long run: the result is a
    hundredth of a value, the sums of codes behind it are not.  Root mean square error of it: the
    output's rounding (2^-8 / sqrt 3), the rounding of p s against codes of 2.5 times a value
    (2^-11 2.5 / sqrt 3) and a tenth of that for the sums: 2.4e-3 in all, at most 3e-3."""
    bs, H, G, n, B = 256, 8, 4, 19000, 128
    nb = (n + bs - 1) // bs
    kp, vp = make_pool(pkg, 68, nb, bs, H), make_pool(pkg, 69, nb, bs, H)
    tables = torch.arange(nb, dtype=torch.int32).repeat(B, 1)          # all rows read the same pages
    q = torch.zeros(B, 1, H * G, 128, dtype=torch.bfloat16)
    out = pkg.flash_attn_with_kvcache_int4(q.cuda(), kp, vp, torch.full((B,), n, dtype=torch.int32).cuda(),
                                           tables.cuda()).cpu().double()
    ref = R.decode_pool(vp.cpu())[0].reshape(-1, H, 128)[:n].mean(0).repeat_interleave(G, 0)
    err = (out[:, 0] - ref).square().mean().sqrt() / ref.square().mean().sqrt()
    assert err <= 3e-3, err


def test_decode_nan_stays_in_its_group(pkg):
    n, bs = 70, 128
    k = torch.from_numpy(det_normal(71, (n, 1, 128))).float().bfloat16()
    v = torch.from_numpy(det_normal(72, (n, 1, 128))).float().bfloat16()
    v[66, 0, 100] = float("nan")
    kp = torch.zeros(pkg.int4_pool_shape(1, bs, 1), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    pkg.store_kvcache_int4(k.cuda(), v.cuda(), kp, vp, torch.arange(n, dtype=torch.int32, device="cuda"))
    pkg.read_device_errors()
    q = torch.from_numpy(det_normal(73, (1, 1, 2, 128))).float().bfloat16()
    out = pkg.flash_attn_with_kvcache_int4(q.cuda(), kp, vp, torch.tensor([n], dtype=torch.int32).cuda(),
                                           torch.zeros(1, 1, dtype=torch.int32).cuda()).cpu()
    ref, _ = R.attend(q[0, 0], R.gather(R.decode_pool(kp.cpu())[0], [0], n),
                      R.gather(R.decode_pool(vp.cpu())[0], [0], n), 128 ** -0.5)
    assert out[0, 0, :, 64:].isnan().all()
    assert ((out[0, 0, :, :64].double() - ref[:, :64]).abs() <= 2.0 ** -7 * ref[:, :64].abs() + 2e-3).all()


def test_decode_captured_twice_and_other_stream(pkg):
    """Two captured graphs replayed side by side on two streams, and an eager call on a third:
    no scratch is shared, every result equals the eager one."""
    bs, H, G = 64, 2, 4
    cases = []
    for i, lens in enumerate(([900, 30, 0], [64, 2000, 5])):
        nb = sum((n + bs - 1) // bs for n in lens) + 1
        kp, vp = make_pool(pkg, 81 + i, nb, bs, H), make_pool(pkg, 84 + i, nb, bs, H)
        q = torch.from_numpy(det_normal(87 + i, (3, 1, 8, 128))).float().bfloat16().cuda()
        cases.append((q, kp, vp, torch.tensor(lens, dtype=torch.int32).cuda(),
                      make_tables(89, lens, bs, nb).cuda()))
    eager = [pkg.flash_attn_with_kvcache_int4(*c) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pkg.flash_attn_with_kvcache_int4(*c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = pkg.flash_attn_with_kvcache_int4(*cases[0])
    torch.cuda.synchronize()
    for o, e in zip(outs, eager):
        assert torch.equal(o, e)
    assert torch.equal(third, eager[0])


# ---- prefill over cached pages ---------------------------------------------------

@pytest.mark.parametrize("qlens,hist,H,G,bs,dtype", [
    ([1], [0], 1, 2, 64, torch.bfloat16),
    ([5, 130, 1], [700, 0, 64], 2, 4, 192, torch.bfloat16),
    ([33, 257], [1000, 127], 2, 2, 256, torch.float16),
    ([64], [2049], 8, 4, 128, torch.bfloat16),
    ([7, 0, 12], [9, 100, 500], 1, 1, 64, torch.float16),
    ([16] * 5, [0, 0, 300, 63, 64], 2, 8, 64, torch.bfloat16),
    ([17] * 5, [0, 0, 300, 63, 64], 2, 8, 64, torch.bfloat16),
    ([4], [200], 1, 24, 64, torch.bfloat16),            # a wider group than the decode takes
])
def test_varlen(pkg, qlens, hist, H, G, bs, dtype):
    """Short calls (SHORT_CHUNK, SHORT_CALL) run as decode rows and have their bound.  Longer
    ones: against fp64 attention on the pool's values rounded to q's type (the documented
    rounding).  Bound: a rounded probability (half a step of the type, relative) and a
    rounded output, 2 half-steps of sum w |v|, plus the fp32 scores' 400 u of their absolute
    sum as above and the exponential, in all below 2^-13 of sum w |v|."""
    klens = [a + b for a, b in zip(qlens, hist)]
    nb = sum((n + bs - 1) // bs for n in klens) + 2
    kp, vp = make_pool(pkg, 91, nb, bs, H, 0.5), make_pool(pkg, 92, nb, bs, H, 0.5)
    tables = make_tables(93, klens, bs, nb)
    # every byte that no row reaches is NaN
    live = torch.zeros(nb, bs, dtype=torch.bool)
    for b, n in enumerate(klens):
        for t in range(n):
            live[tables[b, t // bs], t % bs] = True
    for pool in (kp, vp):
        host = pool.cpu()
        for blk, off in (~live).nonzero().tolist():
            _, p0 = R.row_offsets(off)
            host[blk, :, p0:p0 + 8] = 0xFF
        pool.copy_(host)
    q = torch.from_numpy(det_normal(94, (sum(qlens), H * G, 128))).float().to(dtype)
    cu = lambda x: torch.tensor([0] + list(np.cumsum(x)), dtype=torch.int32)
    pkg.read_device_errors()
    out = pkg.flash_attn_varlen_func_int4(q.cuda(), kp, vp, cu(qlens).cuda(), cu(klens).cuda(),
                                          max(qlens), max(klens), block_table=tables.cuda()).cpu()
    assert pkg.read_device_errors() == 0
    from importlib import import_module
    K = import_module("slo-aware-llm-serving-engine_b200.kvcache_int4")
    if (max(qlens) <= K.SHORT_CHUNK or sum(qlens) <= K.SHORT_CALL) and G <= 16:
        seen = [nk - nq + i + 1 for nq, nk in zip(qlens, klens) for i in range(nq)]
        per = torch.cat([tables[b:b + 1].expand(nq, -1) for b, nq in enumerate(qlens)])
        check_decode(out.unsqueeze(1), q.unsqueeze(1), kp, vp, seen, per, 128 ** -0.5)
        return
    kv, vv = R.decode_pool(kp.cpu())[0], R.decode_pool(vp.cpu())[0]
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    at = 0
    for b, (nq, nk) in enumerate(zip(qlens, klens)):
        k, v = R.gather(kv, tables[b], nk).to(dtype).double(), R.gather(vv, tables[b], nk).to(dtype).double()
        for i in range(nq):
            seen = nk - nq + i + 1
            ref, w = R.attend(q[at + i], k[:seen], v[:seen], 128 ** -0.5)
            wv = torch.einsum("hn,nhd->hd", w, v[:seen].repeat_interleave(G, 1).abs())
            err = (out[at + i].double() - ref).abs()
            assert (err <= (2 * half + 2.0 ** -13) * wv + 2.0 ** -25).all(), (b, i)
        at += nq


def test_varlen_in_groups_and_on_streams(pkg, monkeypatch):
    """Rows that do not fit the scratch together run in groups; two such calls on two streams
    at once share nothing."""
    from importlib import import_module
    K = import_module("slo-aware-llm-serving-engine_b200.kvcache_int4")
    H, G, bs, qlens, klens = 2, 4, 64, [70, 5, 0, 90, 33], [300, 5, 10, 700, 40]
    cases = []
    for i in range(2):
        nb = sum((n + bs - 1) // bs for n in klens) + 1
        kp, vp = make_pool(pkg, 100 + i, nb, bs, H), make_pool(pkg, 102 + i, nb, bs, H)
        q = torch.from_numpy(det_normal(104 + i, (sum(qlens), H * G, 128))).float().bfloat16().cuda()
        cu = lambda x: torch.tensor([0] + list(np.cumsum(x)), dtype=torch.int32).cuda()
        cases.append(((q, kp, vp, cu(qlens), cu(klens), 90, 700),
                      dict(block_table=make_tables(106 + i, klens, bs, nb).cuda())))
    whole = [pkg.flash_attn_varlen_func_int4(*a, **k) for a, k in cases]
    monkeypatch.setattr(K, "_WIDE_BYTES", 2 * 2 * 768 * H * 128 * 2 + 1)      # two rows
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = []
    for _ in range(10):
        for (a, k), s in zip(cases, streams):
            with torch.cuda.stream(s):
                outs.append(pkg.flash_attn_varlen_func_int4(*a, **k))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, whole[i % 2])
    assert pkg.read_device_errors() == 0


@pytest.mark.parametrize("nq", [2, 70])
def test_varlen_bad_metadata_is_flagged(pkg, nq):
    kp, vp = make_pool(pkg, 95, 4, 64, 1), make_pool(pkg, 96, 4, 64, 1)
    q = torch.zeros(nq, 2, 128, dtype=torch.bfloat16, device="cuda")
    cu_q = torch.tensor([0, nq], dtype=torch.int32, device="cuda")
    cu_k = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    pkg.read_device_errors()
    out = pkg.flash_attn_varlen_func_int4(q, kp, vp, cu_q, cu_k, nq, 100, block_table=torch.tensor(
        [[1, 9]], dtype=torch.int32, device="cuda"))
    assert pkg.read_device_errors() & 0x2 and torch.isfinite(out).all()
    # more keys than the table reaches, by more than one widened page
    cu_k = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    out = pkg.flash_attn_varlen_func_int4(q, kp, vp, cu_q, cu_k, nq, 300, block_table=torch.tensor(
        [[1]], dtype=torch.int32, device="cuda"))
    assert pkg.read_device_errors() & 0x4 and torch.isfinite(out).all()


@pytest.mark.parametrize("nq", [3, 66])
def test_varlen_rows_behind_and_without_keys(pkg, nq):
    """Query tokens before the first and behind the last row keep what `out` held; a query that
    sees no key (more queries than keys) gives zeros."""
    H, G, bs = 1, 2, 64
    kp, vp = make_pool(pkg, 97, 4, bs, H), make_pool(pkg, 98, 4, bs, H)
    q = torch.from_numpy(det_normal(99, (nq + 7, 2, 128))).float().bfloat16()
    out = torch.full((nq + 7, 2, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    pkg.read_device_errors()
    pkg.flash_attn_varlen_func_int4(q.cuda(), kp, vp, torch.tensor([0, nq], dtype=torch.int32).cuda(),
                                    torch.tensor([0, nq - 2], dtype=torch.int32).cuda(), nq, nq - 2,
                                    block_table=torch.tensor([[3]], dtype=torch.int32).cuda(), out=out)
    assert pkg.read_device_errors() == 0
    assert (out[nq:] == 5).all() and (out[:2] == 0).all()
    check_decode(out[2:nq].unsqueeze(1), q[2:nq].unsqueeze(1), kp, vp, list(range(1, nq - 1)),
                 torch.full((nq, 1), 3), 128 ** -0.5) if nq <= 32 else None
