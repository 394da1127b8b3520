"""CPU: what the operators over a base refuse, before any device is asked for (rg_softmax_*, rg_q4_*), and the sizes of their scratch."""
import ctypes as C

import pytest

from roargraph_amd import softmax
from roargraph_amd._lib import RG_ERR_ARG, RG_ERR_DEVICE, RG_OK, RgError, lib

P = 0x10000          # a pointer that is never followed: every call here ends before the device
u32, u64, vp, f32 = C.c_uint32, C.c_uint64, C.c_void_p, C.c_float


def shard(base=P, nb=100, bstride=32, q=P, nq=10, qstride=32, dim=32, dtype=0, scale=1.0, targets=P, id_base=0, rest=P, own=P, lse=P, loss=P, mean=P, work=P, bytes_=1 << 40, device=0):
    return lib().rg_softmax_shard_dev(vp(base), u32(nb), u64(bstride), vp(q), u32(nq), u64(qstride), u32(dim), C.c_int(dtype), f32(scale), vp(targets), u32(id_base), vp(rest), vp(own), vp(lse),
                                      vp(loss), vp(mean), vp(work), u64(bytes_), C.c_int(device), vp(0))


def grad(base=P, nb=100, bstride=32, q=P, nq=10, qstride=32, dim=32, dtype=0, scale=1.0, targets=P, id_base=0, lse=P, loss=P, rest=P, mean=P, w=P, dq=P, dqs=32, db=P, dbs=32, work=P,
         bytes_=1 << 40):
    return lib().rg_softmax_grad_dev(vp(base), u32(nb), u64(bstride), vp(q), u32(nq), u64(qstride), u32(dim), C.c_int(dtype), f32(scale), vp(targets), u32(id_base), vp(lse), vp(loss), vp(rest),
                                     vp(mean), vp(w), vp(dq), u64(dqs), vp(db), u64(dbs), vp(work), u64(bytes_), C.c_int(0), vp(0))


def score(codes=P, cs=16, scales=P, mins=0, ss=1, nb=100, dim=32, group=32, q=P, nq=2, qs=32, dtype=0, out=P, os=100):
    return lib().rg_q4_score_dev(vp(codes), u64(cs), vp(scales), vp(mins), u64(ss), u32(nb), u32(dim), u32(group), vp(q), u32(nq), u64(qs), C.c_int(dtype), vp(out), u64(os), C.c_int(0), vp(0))


def pack(rows=P, nb=100, stride=32, dim=32, dtype=0, group=32, codes=P, cs=16, scales=P, mins=0, ss=1):
    return lib().rg_q4_pack_dev(vp(rows), u32(nb), u64(stride), u32(dim), C.c_int(dtype), u32(group), vp(codes), u64(cs), vp(scales), vp(mins), u64(ss), C.c_int(0), vp(0))


def unpack(codes=P, cs=16, scales=P, mins=0, ss=1, nb=100, dim=32, group=32, ids=0, n=100, out=P, os=32):
    return lib().rg_q4_unpack_dev(vp(codes), u64(cs), vp(scales), vp(mins), u64(ss), u32(nb), u32(dim), u32(group), vp(ids), u32(n), vp(out), u64(os), C.c_int(0), vp(0))


@pytest.mark.parametrize("call", [
    lambda: shard(base=0), lambda: shard(q=0), lambda: shard(targets=0), lambda: shard(rest=0), lambda: shard(own=0), lambda: shard(work=0), lambda: shard(dim=0), lambda: shard(dim=1025, bstride=1025, qstride=1025),
    lambda: shard(bstride=31), lambda: shard(qstride=31), lambda: shard(dtype=3), lambda: shard(dtype=-1), lambda: shard(scale=float("nan")), lambda: shard(scale=float("inf")), lambda: shard(scale=3e38),
    lambda: shard(base=P + 2), lambda: shard(q=P + 1, dtype=1), lambda: shard(work=P + 128), lambda: shard(bytes_=64), lambda: shard(nb=1 << 31), lambda: shard(nq=1 << 31),
    lambda: shard(id_base=0xffffffff - 50),
    lambda: grad(lse=0), lambda: grad(loss=0), lambda: grad(w=0), lambda: grad(mean=0), lambda: grad(rest=0), lambda: grad(targets=0), lambda: grad(dqs=31), lambda: grad(dbs=31), lambda: grad(db=P + 2),
    lambda: grad(work=0), lambda: grad(bytes_=64), lambda: grad(dtype=7), lambda: grad(dim=0),
    lambda: score(codes=0), lambda: score(scales=0), lambda: score(q=0), lambda: score(out=0), lambda: score(group=16), lambda: score(group=48), lambda: score(group=0), lambda: score(dim=0),
    lambda: score(dim=4097, cs=2064, qs=4097, ss=200), lambda: score(cs=12), lambda: score(cs=18), lambda: score(codes=P + 2), lambda: score(ss=0), lambda: score(qs=31), lambda: score(os=99),
    lambda: score(dtype=9), lambda: score(out=P + 2), lambda: score(nb=1 << 31, os=1 << 31), lambda: score(mins=P + 1),
    lambda: pack(rows=0), lambda: pack(codes=0), lambda: pack(scales=0), lambda: pack(group=31), lambda: pack(stride=31), lambda: pack(cs=15), lambda: pack(dtype=5), lambda: pack(mins=P + 1),
    lambda: shard(nq=1 << 24), lambda: grad(nq=1 << 24), lambda: score(cs=(1 << 26) + 4), lambda: score(ss=(1 << 25) + 1), lambda: score(nq=1 << 31), lambda: unpack(ids=P, n=1 << 31),
    lambda: unpack(codes=0), lambda: unpack(out=0), lambda: unpack(os=31), lambda: unpack(n=101), lambda: unpack(group=8),
])
def test_refused(call):
    assert call() == RG_ERR_ARG
    assert lib().rg_last_error()


def test_merge_refused():
    m = lib().rg_softmax_merge_dev
    for args in ((0, P, 1, 5, P, P, P), (P, 0, 1, 5, P, P, P), (P, P, 0, 5, P, P, P), (P, P, 1, 5, 0, P, P), (P, P, 1, 5, P, 0, P), (P, P, 1, 5, P, P, 0), (P, P, 1, 1 << 24, P, P, P)):
        a = args
        assert m(vp(a[0]), vp(a[1]), u32(a[2]), u32(a[3]), vp(a[4]), vp(a[5]), vp(a[6]), C.c_int(0), vp(0)) == RG_ERR_ARG


def test_nothing_to_do_needs_no_device():
    assert shard(nq=0) == RG_OK and score(nq=0) == RG_OK and score(nb=0, os=0) == RG_OK and pack(nb=0) == RG_OK and unpack(n=0) == RG_OK


def test_without_a_device_good_calls_say_so():
    if lib().rg_device_count() > 0:
        pytest.skip("a GPU is visible here")
    for call in (shard, grad, score, pack, unpack):
        assert call() == RG_ERR_DEVICE
        assert b"no CPU fallback" in lib().rg_last_error()


def test_scratch_sizes():
    for what in (softmax.STATS, softmax.MEAN, softmax.GRAD):
        for nb, nq, dim in ((1, 1, 1), (1000, 64, 24), (10_000_000, 1, 200), (10_000_000, 4096, 200), (0, 10, 8), (10, 0, 8), (2 ** 31 - 1, 1, 1024), (100, 2 ** 20, 512)):
            for code in (0, 1, 2):
                n = softmax.workspace(what, nb, nq, dim, code)
                # partial sums of at most a few thousand pieces, or of the rows themselves where they are many: never the logits
                assert 0 <= n and n % 256 == 0
                if nb * nq > 10 ** 9:
                    assert n < nb * nq
    with pytest.raises(RgError):
        softmax.workspace(3, 10, 10, 8, 0)
    with pytest.raises(RgError):
        softmax.workspace(0, 10, 10, 0, 0)
    assert lib().rg_softmax_workspace(C.c_int(0), u32(1), u32(1), u32(8), C.c_int(0), None) == RG_ERR_ARG


def test_a_scale_that_requires_grad():
    import torch
    s = torch.tensor(2.0, requires_grad=True)
    x, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    for scale in (s, s.exp()):
        with pytest.raises(TypeError, match="queries"):
            softmax.softmax_loss(x, x, t, scale)


def test_sizes_beyond_32_bits():
    """(ctypes takes the lowest 32 bits of a number: 2^32 + 5 rows would be 5)"""
    import torch
    from roargraph_amd import q4
    t = torch.zeros(3, dtype=torch.int32)
    x = torch.zeros(3, 32)
    for shape in ((2 ** 31, 1), (2 ** 32 + 5, 1), (1, 2 ** 32 + 8)):
        far = torch.empty(shape, device="meta")
        for call in (lambda: softmax.softmax_shard_dev(far, x, t, 1.0), lambda: softmax.softmax_grad_dev(x, far, t, 1.0, x, x, x), lambda: q4.q4_pack(far)):
            with pytest.raises(ValueError, match="2\\^31"):
                call()
    for id_base in (-1, 2 ** 32):
        for call in (lambda: softmax.softmax_shard_dev(x, x, t, 1.0, id_base=id_base), lambda: softmax.softmax_grad_dev(x, x, t, 1.0, x, x, x, id_base=id_base)):
            with pytest.raises(ValueError, match="id_base"):
                call()
    for sizes in ((2 ** 32, 1, 8), (1, 2 ** 32 + 1, 8), (1, 1, 2 ** 32 + 8), (-1, 1, 8)):
        with pytest.raises(ValueError, match="32 bits"):
            softmax.workspace(softmax.STATS, *sizes, 0)


def test_tensors_of_the_host_and_unknown_groups():
    import torch
    from roargraph_amd import q4
    x, t = torch.zeros(3, 32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        q4.q4_pack(x)
    with pytest.raises(ValueError, match="GPU"):
        softmax.softmax_merge_dev(torch.zeros(1, 3), torch.zeros(1, 3), t)
    with pytest.raises(ValueError, match="groups"):
        q4.q4_score(x, q4.Q4Base(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1).half(), None, 32, 0))
