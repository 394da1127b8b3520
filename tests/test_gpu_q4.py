"""-m gpu: a base in 4 bits (rg_q4_*) against its definition.

Codes, scales, minima and unpacked values are compared exactly (the level is the nearest one, ties to the even code; the values are one fp32
product and sum).  Scores: fp32 sums of dim products of exact factors, |dy| <= (dim + 8) 2^-24 sum |q||v|; a query enters as two halves, 22 bits
of its elements relative to the largest: 2^-22 max|q| sum |v|; with minima the sum over the codes and the sum over the minima are rounded
apart, each up to 16 scales and the minimum in size."""
import numpy as np
import pytest
import torch

from roargraph_amd import q4

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def plain_pack(x, group, mins):
    """codes, scales, mins, values as the header defines them (numpy, 64 bits where a level is decided)"""
    x = x.float().numpy()
    nb, dim = x.shape
    groups = -(-dim // group)
    codes, scales, lows, values = np.zeros((nb, dim), np.int64), np.zeros((nb, groups), np.float16), np.zeros((nb, groups), np.float16), np.zeros((nb, dim), np.float32)
    for g in range(groups):
        p = x[:, g * group:(g + 1) * group]
        if mins:
            s = ((p.max(1) - p.min(1)) * (np.float32(1) / np.float32(15))).astype(np.float16)
            m = p.min(1).astype(np.float16)
        else:
            s = (np.abs(p).max(1) * (np.float32(1) / np.float32(7))).astype(np.float16)
            m = np.zeros(nb, np.float16)
        sd = s.astype(np.float64)[:, None]
        lo, hi = (0, 15) if mins else (-8, 7)
        c = np.where(sd > 0, np.clip(np.rint((p.astype(np.float64) - m.astype(np.float64)[:, None]) / np.where(sd > 0, sd, 1)), lo, hi), 0)
        codes[:, g * group:(g + 1) * group] = c - lo
        values[:, g * group:(g + 1) * group] = c.astype(np.float32) * s.astype(np.float32)[:, None] + (m.astype(np.float32)[:, None] if mins else 0)
        scales[:, g], lows[:, g] = s, m
    return codes, scales, lows, values


def nibbles(codes, dim):
    c = codes.cpu().numpy()
    return np.stack((c & 15, c >> 4), -1).reshape(c.shape[0], -1)


SHAPES = [(1, 1), (3, 7), (17, 8), (100, 24), (65, 32), (129, 33), (40, 64), (50, 93), (64, 128), (333, 200), (70, 301), (31, 512), (18, 1000), (9, 1024), (5, 4096), (3, 4095)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group,mins", [(32, False), (64, True), (128, False), (32, True)])
@pytest.mark.parametrize("nb,dim", SHAPES)
def test_pack_and_unpack(nb, dim, group, mins, dtype):
    g = torch.Generator().manual_seed(nb + dim)
    x = (torch.randn(nb, dim, generator=g) + (0.5 if mins else 0)).to(DT[dtype])
    x[0] = 0                                                       # a group of zeros
    if nb > 2:
        x[1] = 0.75                                                # all equal
        x[2, : min(dim, 8)] = torch.tensor([7.0, 0.5, 1.5, 2.5, -0.5, -1.5, -7.0, 3.5])[: min(dim, 8)].to(DT[dtype])   # ties where the scale comes out as 1
    codes, scales, lows, values = plain_pack(x, group, mins)
    p = q4.q4_pack(x.cuda(), group=group, mins=mins)
    got = nibbles(p.codes, dim)
    assert (p.scales.cpu().numpy().view(np.uint16) == scales.view(np.uint16)).all()
    if mins:
        assert (p.mins.cpu().numpy() == lows).all()
    assert (got[:, :dim] == codes).all()
    assert (got[:, dim:] == 0).all()
    assert (q4.q4_unpack(p).cpu().numpy() == values).all()
    ids = torch.tensor([nb - 1, 0, nb - 1, nb // 2])
    assert (q4.q4_unpack(p, ids.cuda()).cpu().numpy() == values[ids.numpy()]).all()
    assert q4.q4_unpack(p, torch.tensor([nb, -1]).cuda()).isnan().all()


def random_form(nb, dim, group, mins, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    groups = -(-dim // group)
    codes = torch.randint(256, (nb, -(-dim // 8) * 4 + pad), generator=g, dtype=torch.uint8)
    scales = ((torch.rand(nb, groups, generator=g) + 0.5) * 0.05).half()
    low = (scales.float() * -(torch.rand(nb, groups, generator=g) * 16)).half() if mins else None
    return codes, scales, low


def values_of(codes, scales, low, dim, group):
    at = torch.arange(dim)
    c = (codes[:, at // 2].long() >> (4 * (at % 2))) & 15
    s = scales.double()[:, at // group]
    return (c - 8) * s if low is None else c * s + low.double()[:, at // group]


def score_tolerance(q, v, scales, low, dim, group):
    u = 2.0 ** -24
    size = v.abs()
    if low is not None:
        at = torch.arange(dim)
        size = 16 * scales.double()[:, at // group] + low.double()[:, at // group].abs()
    x = q.double().abs()
    return (dim + 8) * u * (x @ size.T) + 2.0 ** -22 * x.amax(1, keepdim=True) * size.sum(1)[None] + 1e-30


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group,mins", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("nq,nb,dim", [(1, 1, 1), (1, 17, 7), (1, 2000, 200), (2, 333, 24), (3, 129, 93), (4, 1000, 128), (5, 70, 33), (8, 515, 512), (9, 260, 301), (13, 64, 1000), (16, 333, 1024),
                                       (17, 100, 96), (33, 50, 40), (1, 31, 4096), (70, 21, 2056), (1, 70001, 8)])
def test_scores(nq, nb, dim, group, mins, dtype):
    codes, scales, low = random_form(nb, dim, group, mins, seed=nq + nb + dim)
    q = torch.randn(nq, dim, generator=torch.Generator().manual_seed(3)).to(DT[dtype])
    v = values_of(codes, scales, low, dim, group)
    p = q4.Q4Base(codes.cuda(), scales.cuda(), low.cuda() if mins else None, dim, group)
    got = q4.q4_score(q.cuda(), p)
    off = (got.double().cpu() - q.double() @ v.T).abs() / score_tolerance(q, v, scales, low, dim, group)
    assert off.max() <= 1.0, off.max()
    assert torch.equal(got, q4.q4_score(q.cuda(), p))


def test_score_strides_and_surroundings():
    """rows inside wider buffers, queries at an odd offset, scores into a wider buffer: the same bits, and nothing around them written"""
    for dim, group, mins in ((200, 32, True), (93, 64, False), (512, 128, True)):
        nb, nq = 301, 5
        codes, scales, low = random_form(nb, dim, group, mins, seed=dim)
        q = torch.randn(nq, dim)
        groups = scales.shape[1]
        want = q4.q4_score(q.cuda(), q4.Q4Base(codes.cuda(), scales.cuda(), low.cuda() if mins else None, dim, group))
        wide = torch.randint(256, (nb + 2, codes.shape[1] + 12), dtype=torch.uint8, device="cuda")
        wide[1:-1, 4:4 + codes.shape[1]] = codes.cuda()
        sc = torch.full((2, nb, groups + 3), float("nan"), dtype=torch.float16, device="cuda")
        sc[0, :, 1:1 + groups] = scales.cuda()
        if mins:
            sc[1, :, 1:1 + groups] = low.cuda()
        qq = torch.full((nq + 1, dim + 3), float("nan"), device="cuda")
        qq[1:, 1:1 + dim] = q.cuda()
        out = torch.full((nq, nb + 9), 77.0, device="cuda")
        form = q4.Q4Base(wide[1:-1, 4:4 + codes.shape[1]], sc[0, :, 1:1 + groups], sc[1, :, 1:1 + groups] if mins else None, dim, group)
        q4.q4_score(qq[1:, 1:1 + dim], form, out=out[:, 3:3 + nb])
        assert torch.equal(out[:, 3:3 + nb], want) and (out[:, :3] == 77).all() and (out[:, 3 + nb:] == 77).all()
        assert torch.equal(q4.q4_unpack(form), q4.q4_unpack(q4.Q4Base(codes.cuda(), scales.cuda(), low.cuda() if mins else None, dim, group)))


def test_pack_strides_and_surroundings():
    import ctypes as C
    from roargraph_amd._lib import check, lib
    nb, dim, group = 77, 93, 32
    x = torch.randn(nb, dim)
    want = q4.q4_pack(x.cuda(), group=group, mins=True)
    buf = torch.full((nb + 1, dim + 5), float("nan"), device="cuda")
    buf[1:, 2:2 + dim] = x.cuda()
    codes = torch.full((nb + 1, 60), 0x5a, dtype=torch.uint8, device="cuda")
    sc = torch.full((2, nb + 1, 5), 77.0, dtype=torch.float16, device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    check(lib().rg_q4_pack_dev(p(buf[1:, 2:]), C.c_uint32(nb), C.c_uint64(dim + 5), C.c_uint32(dim), C.c_int(0), C.c_uint32(group), p(codes), C.c_uint64(60), p(sc[0]), p(sc[1]), C.c_uint64(5),
                               C.c_int(0), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert torch.equal(codes[:nb, :48], want.codes) and (codes[:nb, 48:] == 0x5a).all() and (codes[nb:] == 0x5a).all()
    assert torch.equal(sc[0, :nb, :3], want.scales) and torch.equal(sc[1, :nb, :3], want.mins) and (sc[:, :, 3:] == 77).all() and (sc[:, nb:] == 77).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_queries_of_any_size(dtype):
    """queries far from 1 keep their digits; one that is not finite shows in its own scores only"""
    codes, scales, low = random_form(200, 96, 32, True, seed=4)
    v = values_of(codes, scales, low, 96, 32)
    p = q4.Q4Base(codes.cuda(), scales.cuda(), low.cuda(), 96, 32)
    q = torch.randn(6, 96) * torch.tensor([1e-30, 1e-12, 1.0, 1e12, 1e30, 0.0])[:, None]
    q = q.to(DT[dtype])
    got = q4.q4_score(q.cuda(), p).double().cpu()
    assert ((got - q.double() @ v.T).abs() <= score_tolerance(q, v, scales, low, 96, 32)).all()
    q[2, 5] = float("nan")
    q[3, 5] = float("inf")
    bad = q4.q4_score(q.cuda(), p).double().cpu()
    ok = [0, 1, 4, 5]
    assert torch.equal(bad[ok], got[ok]) and bad[2].isnan().all() and not torch.isfinite(bad[3]).any()


def test_empty_and_refused():
    form = q4.Q4Base(torch.zeros(0, 12, dtype=torch.uint8, device="cuda"), torch.zeros(0, 1, dtype=torch.float16, device="cuda"), None, 24, 32)
    assert q4.q4_score(torch.zeros(3, 24, device="cuda"), form).shape == (3, 0) and q4.q4_unpack(form).shape == (0, 24)
    p = q4.q4_pack(torch.randn(10, 24, device="cuda"))
    assert q4.q4_score(torch.zeros(0, 24, device="cuda"), p).shape == (0, 10)
    assert q4.q4_unpack(p, torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 24)
    assert q4.q4_pack(torch.zeros(0, 24, device="cuda")).codes.shape == (0, 12)
    for bad in (lambda: q4.q4_pack(torch.randn(10, 24, device="cuda"), group=16), lambda: q4.q4_score(torch.zeros(1, 23, device="cuda"), p),
                lambda: q4.q4_score(torch.zeros(1, 24, device="cuda"), p._replace(scales=p.scales[:5])), lambda: q4.q4_score(torch.zeros(1, 24, device="cuda"), p._replace(codes=p.codes[:, :8])),
                lambda: q4.q4_score(torch.zeros(1, 24, device="cuda"), p, out=torch.zeros(1, 9, device="cuda")), lambda: q4.q4_unpack(p, torch.zeros(3, device="cuda"))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("mins", [False, True])
def test_a_scale_of_zero_has_one_level(mins):
    """groups whose values are all alike, beside values between two levels: codes of the first level, whatever the neighbours"""
    x = torch.zeros(40, 65)
    x[:, :32] = torch.tensor([0.0, 15.0, 0.5, 1.5, 2.5, 3.5, 7.0, 4.0] * 4)      # (with minima: a scale of 1)
    x[:, 32:64] = torch.linspace(0.1, 3.0, 40)[:, None]
    x[:, 64] = torch.linspace(-1.0, 1.0, 40) + 1e-5
    for rows in (x, x * 1e-9):
        codes, scales, low, values = plain_pack(rows, 32, mins)
        p = q4.q4_pack(rows.cuda(), group=32, mins=mins)
        assert (nibbles(p.codes, 65)[:, :65] == codes).all() and (p.scales.cpu().numpy() == scales).all() and (q4.q4_unpack(p).cpu().numpy() == values).all()


def test_rows_that_overlap_are_refused():
    """(an expanded matrix has no row stride: reading it as rows would leave the tensor)"""
    p = q4.q4_pack(torch.randn(100, 24, device="cuda"), mins=True)
    q = torch.zeros(1, 24, device="cuda")
    for bad in (p._replace(scales=p.scales[:1].expand(100, 1), mins=p.mins[:1].expand(100, 1)), p._replace(codes=p.codes[:1].expand(100, 12)),
                p._replace(mins=None, scales=p.scales[:1].expand(100, 1))):
        for call in (lambda: q4.q4_score(q, bad), lambda: q4.q4_unpack(bad)):
            with pytest.raises(ValueError, match="overlap"):
                call()


def test_ids_beyond_32_bits_are_no_rows():
    p = q4.q4_pack(torch.randn(100, 24, device="cuda"))
    got = q4.q4_unpack(p, torch.tensor([5, 2 ** 32 + 5, -2 ** 32, -1, 2 ** 31, 2 ** 40, 99, 100], device="cuda"))
    want = q4.q4_unpack(p)
    assert torch.equal(got[0], want[5]) and torch.equal(got[6], want[99]) and got[[1, 2, 3, 4, 5, 7]].isnan().all()


def test_rows_and_scores_beyond_4_gigabytes():
    nb, dim = 5_000_000, 40
    gen = torch.Generator(device="cuda").manual_seed(1)
    p = q4.q4_pack(torch.randn(nb, dim, device="cuda", generator=gen), mins=True)
    far = p._replace(codes=torch.empty(nb, 1024, dtype=torch.uint8, device="cuda")[:, 900:900 + p.codes.shape[1]],
                     scales=torch.empty(nb, 512, dtype=torch.float16, device="cuda")[:, 300:300 + p.scales.shape[1]], mins=torch.empty(nb, 512, dtype=torch.float16, device="cuda")[:, 7:7 + p.scales.shape[1]])
    far.codes.copy_(p.codes), far.scales.copy_(p.scales), far.mins.copy_(p.mins)
    q = torch.randn(3, dim, device="cuda", generator=gen)
    out = torch.empty(3, 700_000_000, device="cuda")[:, 5:5 + nb]
    want = q4.q4_score(q, p)
    assert torch.equal(q4.q4_score(q, far, out=out), want) and torch.equal(out, want)
    ids = torch.tensor([nb - 1, 0, nb // 2], device="cuda")
    assert torch.equal(q4.q4_unpack(far, ids), q4.q4_unpack(p)[ids])


def test_streams_and_graphs():
    p = q4.q4_pack(torch.randn(5000, 200, device="cuda"), mins=True)
    sets = [torch.randn(3, 200, device="cuda") for _ in range(3)]
    want = [q4.q4_score(s, p) for s in sets]
    torch.cuda.synchronize()
    side, held, graph = torch.cuda.Stream(), sets[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        q4.q4_score(held, p)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            again = q4.q4_pack(q4.q4_unpack(p), mins=True)
            out = q4.q4_score(held, p)
    values = q4.q4_unpack(p)
    for k in (1, 2, 0, 1):
        held.copy_(sets[k])
        torch.cuda.synchronize()
        graph.replay()
        eager = q4.q4_score(sets[k], p)
        torch.cuda.synchronize()
        assert torch.equal(out, want[k]) and torch.equal(eager, want[k])
        assert torch.equal(again.codes, q4.q4_pack(values, mins=True).codes)
