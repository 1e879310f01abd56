"""Prefill over a 4-bit pool at the edges of its contract.  Calls of 64 query tokens run as
decode rows, of 65 in one chunk through widened pages; both are checked with the bounds of
test_gpu_int4.py."""
import pytest
import torch

from tests import int4_reference as R
from tests.golden.detgen import det_normal
from tests.test_gpu_int4 import check_decode, make_pool, make_tables

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_long(out, q, k, v, seen, dtype):
    """Bound of test_gpu_int4.test_varlen's longer calls: out and q [T, Hq, 128], k and v the fp64
    values of one row in q's type, query i sees the first seen[i]."""
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    G = q.shape[1] // k.shape[1]
    for i, n in enumerate(seen):
        ref, w = R.attend(q[i], k[:n], v[:n], SCALE)
        wv = torch.einsum("hn,nhd->hd", w, v[:n].repeat_interleave(G, 1).abs())
        err = (out[i].double() - ref).abs()
        assert (err <= (2 * half + 2.0 ** -13) * wv + 2.0 ** -25).all(), (i, (err - 2 * half * wv).max())


def place(raw, at, shape, strides):
    """A view of the flat tensor `raw` that starts at element `at`."""
    return torch.as_strided(raw, shape, strides, raw.storage_offset() + at)


@pytest.mark.parametrize("T", [61, 64, 65])           # 64 query tokens in all; 67; 68
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at,row,head", [
    (0, 1024, 128),                  # contiguous
    (4, 1024, 128),                  # 8 bytes off
    (1, 1024, 128),                  # an odd element
    (0, 1540, 128),                  # rows of a fused projection, 8 bytes off a multiple of 16
    (8, 1600, 130),                  # heads 4 bytes off
    (2, 1601, 131),                  # neither rows nor heads on 4 bytes
    (0, 1024, 0),                    # one head's query for all (q only)
])
def test_varlen_any_view(pkg, T, dtype, at, row, head):
    """q and out at any address and stride give what contiguous ones do; rows behind the last
    sequence and the elements between out's rows keep what they held."""
    H, G, bs, klen, more = 2, 4, 64, 150, 3
    kp, vp = make_pool(pkg, 1, 4, bs, H), make_pool(pkg, 2, 4, bs, H)
    tables = make_tables(3, [klen], bs, 4).cuda()
    n = T + more
    raw = torch.from_numpy(det_normal(4, (at + n * max(row, 1024) + 2048,))).float().to(dtype).cuda()
    q = place(raw, at, (n, H * G, 128), (row, head, 1))
    if head:
        held = torch.full_like(raw, 7.0)
        out = place(held, at, (n, H * G, 128), (row, head, 1))
    else:
        held, out = None, torch.full((n, H * G, 128), 7.0, dtype=dtype, device="cuda")
    args = (kp, vp, i32(0, T), i32(0, klen), T, klen)
    pkg.read_device_errors()
    want = torch.full((n, H * G, 128), 7.0, dtype=dtype, device="cuda")
    pkg.flash_attn_varlen_func_int4(q.clone(memory_format=torch.contiguous_format), *args,
                                    block_table=tables, out=want)
    res = pkg.flash_attn_varlen_func_int4(q, *args, block_table=tables, out=out)
    assert res.data_ptr() == out.data_ptr() and pkg.read_device_errors() == 0
    assert torch.equal(out, want) and (out[T:] == 7).all()
    if held is not None:
        out.fill_(7.0)
        assert (held == 7).all()
    fresh = pkg.flash_attn_varlen_func_int4(q, *args, block_table=tables)
    assert torch.equal(fresh[:T], want[:T])


@pytest.mark.parametrize("nq", [3, 66])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_varlen_rows_around_and_values(pkg, nq, dtype):
    """Query tokens before the first and behind the last row keep what `out` held, those without
    keys give zeros, the others their attention."""
    H, G, bs, first = 1, 2, 64, 3
    kp, vp = make_pool(pkg, 5, 4, bs, H), make_pool(pkg, 6, 4, bs, H)
    n = first + nq + 4
    q = torch.from_numpy(det_normal(7, (n, H * G, 128))).float().to(dtype)
    out = torch.full((n, H * G, 128), 5.0, dtype=dtype, device="cuda")
    pkg.read_device_errors()
    pkg.flash_attn_varlen_func_int4(q.cuda(), kp, vp, i32(first, first + nq), i32(0, nq - 2), nq, nq - 2,
                                    block_table=i32(3).view(1, 1), out=out)
    assert pkg.read_device_errors() == 0
    out = out.cpu()
    last = first + nq
    assert (out[:first] == 5).all() and (out[last:] == 5).all() and (out[first:first + 2] == 0).all()
    seen = list(range(1, nq - 1))
    mine, mq = out[first + 2:last], q[first + 2:last]
    if nq <= 64:
        check_decode(mine.unsqueeze(1), mq.unsqueeze(1), kp, vp, seen, torch.full((nq, 1), 3), SCALE)
    else:
        k, v = (R.gather(R.decode_pool(p.cpu())[0], [3], nq - 2).to(dtype).double() for p in (kp, vp))
        check_long(mine, mq, k, v, seen, dtype)


@pytest.mark.parametrize("T", [64, 70])
def test_varlen_values_at_the_end_of_f16(pkg, T):
    """f16 rows whose values read back past f16's largest (the minimum -65,504 is stored as
    -65,536; a scale rounded up takes code 15 to 65,714) stay finite on either path."""
    H, G, bs, klen, dtype = 1, 2, 64, 200, torch.float16
    nb = 4
    k = torch.from_numpy(det_normal(11, (klen, H, 128))).float() * 0.5
    v = torch.from_numpy(det_normal(12, (klen, H, 128))).float() * 100
    v[5, 0, :64] = torch.linspace(-65504, -60000, 64)
    v[9, 0, 64:] = torch.linspace(-46, 65504, 64)
    k[11, 0, :64] = torch.linspace(-65504, -65000, 64)
    k, v = k.half(), v.half()
    kp = torch.zeros(pkg.int4_pool_shape(nb, bs, H), dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    tables = make_tables(13, [klen], bs, nb)
    slots = [int(tables[0, t // bs]) * bs + t % bs for t in range(klen)]
    pkg.read_device_errors()
    pkg.store_kvcache_int4(k.cuda(), v.cuda(), kp, vp, i32(*slots))
    got = pkg.int4_decode(vp, i32(slots[5], slots[9])).cpu()
    assert got[0].min() == -65536 and got[1].max() > 65520       # past what f16 rounds to its largest
    q = torch.from_numpy(det_normal(14, (T, H * G, 128))).float().half()
    q[:, :, :64] = 0                                 # the large keys weigh as the others do
    out = pkg.flash_attn_varlen_func_int4(q.cuda(), kp, vp, i32(0, T), i32(0, klen), T, klen,
                                          block_table=tables.cuda()).cpu()
    assert pkg.read_device_errors() == 0 and torch.isfinite(out).all()
    seen = [klen - T + i + 1 for i in range(T)]
    if T <= 64:
        check_decode(out.unsqueeze(1), q.unsqueeze(1), kp, vp, seen, tables.expand(T, -1), SCALE)
        return
    # -65,536 and 65,714 read as -65,504 and 65,504: half a step of f16 and less than 2^-8
    kk, vv = (R.gather(R.decode_pool(p.cpu())[0], tables[0], klen).clamp(-65504, 65504).half().double()
              for p in (kp, vp))
    check_long(out, q, kk, vv, seen, dtype)


@pytest.mark.parametrize("T", [64, 70])
def test_varlen_values_past_f16_are_flagged(pkg, T):
    """A pool of larger values than any f16 row leaves in it, read with f16 queries: decode rows
    compute on, widened pages cannot hold the values and say so."""
    H, G, bs, klen = 1, 2, 64, 100
    kp = make_pool(pkg, 15, 2, bs, H)
    vp = make_pool(pkg, 16, 2, bs, H, 1000.0, 70000.0)
    tables = torch.tensor([[1, 0]], dtype=torch.int32)
    q = torch.from_numpy(det_normal(17, (T, H * G, 128))).float().half()
    pkg.read_device_errors()
    pkg.flash_attn_varlen_func_int4(q.cuda(), kp, vp, i32(0, T), i32(0, klen), T, klen,
                                    block_table=tables.cuda())
    assert pkg.read_device_errors() == (0 if T <= 64 else 0x10)
