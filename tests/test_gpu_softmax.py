"""-m gpu: softmax cross entropy over a base (rg_softmax_*) against the definition in 64 bits.

Tolerances, derived from the number formats (u = 2^-24, half a step of fp32 relative to the value):
  logits     fp32 sums of dim products: |dz| <= scale |q||b| (dim + 8) u; fp32 rows are pairs of halves, 22 bits of every element relative to
             the largest of its row, which is at most the row's norm: another 3 2^-22 sqrt(dim) scale |q||b|
  loss       both log sums move by at most |dz|: 2 |dz|, and a few roundings of values of the size of loss and own
  weights p  relative 2 |dz| plus the type a weight is multiplied in: half a step of bf16 (2^-8) or fp16 (2^-11; as pairs of halves 2^-22 for
             fp32 rows), and below 2^-32 of the largest weight of the row the fixed step of fp16
  gradients  the weights' error times the terms' absolute values, sums of fp32, and half a step of the output's type"""
import numpy as np
import pytest
import torch

from roargraph_amd import softmax

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def make(nq, nb, dim, dtype, seed=0, scale=8.0, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(nb, dim, generator=g)
    base /= base.norm(dim=1, keepdim=True).clamp(min=1e-6)
    if spread:
        base *= 10 ** (spread * (torch.rand(nb, 1, generator=g) - 0.5))
    targets = torch.randint(max(nb, 1), (nq,), generator=g, dtype=torch.int32)
    q = torch.randn(nq, dim, generator=g)
    q = 0.7 * q / q.norm(dim=1, keepdim=True).clamp(min=1e-6)
    if nb:
        near = base[targets.long()]
        q += 0.6 * near / near.norm(dim=1, keepdim=True).clamp(min=1e-6)
    w = (torch.rand(nq, generator=g) + 0.5) / max(nq, 1)
    return base.to(DT[dtype]), q.to(DT[dtype]), targets, w, scale


def exact(base, q, targets, w, scale):
    """loss, dq, db and the sums of the absolute values of their terms, in 64 bits on the CPU"""
    b, x, t = base.double(), q.double(), targets.long()
    z = scale * (x @ b.T)
    lse = torch.logsumexp(z, 1)
    rows = torch.arange(x.shape[0])
    has = t >= 0
    tt = t.clamp(min=0)
    z_others = z.clone()
    z_others[rows[has], tt[has]] = -np.inf
    rest = torch.logsumexp(z_others, 1)
    own = z[rows, tt]
    loss = torch.where(has, torch.where(rest == -np.inf, 0.0, torch.nn.functional.softplus(rest - own, threshold=1e9)), 0.0)
    ww = torch.where(has, w.double(), 0.0)
    p = torch.exp(z - lse[:, None])
    miss = -torch.expm1(-loss)
    g = p * ww[:, None]
    g[rows[has], tt[has]] = -(miss * ww)[has]
    return dict(z=z, lse=lse, rest=rest, own=own, loss=loss, g=g, dq=scale * g @ b, db=scale * g.T @ x, aq=abs(scale) * g.abs() @ b.abs(), ab=abs(scale) * g.abs().T @ x.abs())


def tolerances(base, q, targets, w, scale, e, dtype):
    dim = base.shape[1]
    top = base.double().norm(dim=1).max() * q.double().norm(dim=1).max() * abs(scale)
    dz = top * (dim + 8) * U + (3 * 2.0 ** -22 * dim ** 0.5 * top if dtype == "f32" else 0)
    tol_loss = 2 * dz + 4 * U * (e["loss"].abs() + e["own"].abs().clamp(max=1e30)) + 16 * U
    half = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    out = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    tiny = {"f32": 1e-38, "f16": 2.0 ** -25, "bf16": 1e-38}[dtype]
    n, m = q.shape[0], base.shape[0]
    rel = 2 * dz + half
    floor = 0.0 if dtype == "bf16" else 2.0 ** -32
    gq = e["g"].abs().amax(1, keepdim=True) * floor                     # per query: fixed step below its largest weight
    gb = e["g"].abs().amax(0)[:, None] * floor                          # per row alike
    tol_dq = e["aq"] * (rel + (m + 8) * U) + abs(scale) * gq * base.double().abs().sum(0)[None] + out * e["dq"].abs() + tiny
    tol_db = e["ab"] * (rel + (n + 8) * U) + abs(scale) * gb * q.double().abs().sum(0)[None] + out * e["db"].abs() + tiny
    return tol_loss, tol_dq, tol_db


def step(base, q, targets, w, scale, grads="qb"):
    b, x = base.cuda().requires_grad_("b" in grads), q.cuda().requires_grad_("q" in grads)
    loss = softmax.softmax_loss(x, b, targets.cuda(), scale)
    leaves = [t for t, n in ((x, "q"), (b, "b")) if n in grads]
    got = torch.autograd.grad(loss, leaves, w.cuda()) if leaves else ()
    return loss.detach(), got


def within(got, want, tol, what):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert worst <= 1.0, "%s: %.3g times the tolerance" % (what, worst)


SHAPES = [(1, 1, 1), (1, 17, 8), (3, 1000, 24), (64, 1000, 24), (65, 333, 33), (16, 16, 64), (17, 129, 7), (33, 31, 65), (130, 4097, 200), (64, 2048, 208), (40, 700, 209),
          (5, 513, 93), (100, 300, 128), (31, 900, 256), (70, 257, 257), (66, 1025, 384), (129, 515, 512), (20, 260, 513), (9, 400, 768), (19, 130, 1000), (35, 97, 1024),
          (1, 30000, 200), (2000, 40, 96), (300, 20000, 16),
          (70, 2000, 768), (200, 700, 700), (130, 3000, 1024), (64, 6000, 1000), (65, 500, 515), (90, 600, 385),
          (100, 3000, 40), (128, 2000, 64), (129, 2000, 64), (128, 900, 201), (256, 1500, 301), (257, 1500, 301), (200, 5000, 7), (110, 40000, 130)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nb,dim", SHAPES)
def test_loss_and_gradients(nq, nb, dim, dtype):
    data = make(nq, nb, dim, dtype, seed=nq + nb + dim)
    data[2][::7] = -1
    e = exact(*data)
    tl, tq, tb = tolerances(*data, e, dtype)
    loss, (dq, db) = step(*data)
    assert loss.dtype == torch.float32 and dq.dtype == db.dtype == DT[dtype]
    within(loss, e["loss"], tl, "loss")
    within(dq, e["dq"], tq, "dq")
    within(db, e["db"], tb, "db")
    # without gradients, and with one of them, the same bits
    assert torch.equal(step(*data, grads="")[0], loss)
    assert torch.equal(step(*data, grads="q")[1][0], dq)
    assert torch.equal(step(*data, grads="b")[1][0], db)
    assert torch.equal(step(*data)[1][1], db), "the same call gives the same bits"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_targets(dtype):
    """no target, one target for all, the last row, and a target that is no row"""
    base, q, targets, w, scale = make(50, 700, 72, dtype, seed=5)
    for t in (torch.full_like(targets, -1), torch.full_like(targets, 3), torch.full_like(targets, 699)):
        e = exact(base, q, t, w, scale)
        tl, tq, tb = tolerances(base, q, t, w, scale, e, dtype)
        loss, (dq, db) = step(base, q, t, w, scale)
        within(loss, e["loss"], tl, "loss")
        within(dq, e["dq"], tq, "dq")
        within(db, e["db"], tb, "db")
        if t[0] == -1:
            assert not loss.any() and not dq.any() and not db.any()
    t = targets.clone()
    t[4] = 700
    loss, (dq, db) = step(base, q, t, w, scale)
    assert loss[4].item() == np.inf and torch.isfinite(torch.cat((loss[:4], loss[5:]))).all() and torch.isfinite(dq).all() and torch.isfinite(db).all()
    assert torch.equal(step(base, q, targets.long(), w, scale)[0], step(base, q, targets, w, scale)[0]), "int64 ids"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_signs_and_zeros_of_weights(dtype):
    base, q, targets, w, scale = make(90, 500, 100, dtype, seed=6)
    w[::2] *= -1
    w[::5] = 0
    e = exact(base, q, targets, w, scale)
    tl, tq, tb = tolerances(base, q, targets, w, scale, e, dtype)
    _, (dq, db) = step(base, q, targets, w, scale)
    within(dq, e["dq"], tq, "dq")
    within(db, e["db"], tb, "db")
    assert not dq[::5].any()
    _, (dq, db) = step(base, q, targets, torch.zeros_like(w), scale)
    assert not dq.any() and not db.any()


@pytest.mark.parametrize("scale", [300.0, -5.0, 0.0, 1e-3])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scales(dtype, scale):
    base, q, targets, w, _ = make(33, 400, 56, dtype, seed=7)
    e = exact(base, q, targets, w, scale)
    tl, tq, tb = tolerances(base, q, targets, w, scale, e, dtype)
    loss, (dq, db) = step(base, q, targets, w, scale)
    within(loss, e["loss"], tl, "loss")
    within(dq, e["dq"], tq, "dq")
    within(db, e["db"], tb, "db")


@pytest.mark.parametrize("dtype,spread", [("f32", 12.0), ("f32", 3.0), ("bf16", 12.0)])
def test_rows_of_very_different_norms(dtype, spread):
    """rows 10^(+-spread / 2) long: every row keeps its own digits"""
    base, q, targets, w, scale = make(40, 600, 80, dtype, seed=8, scale=1e-6 if spread > 6 else 1.0, spread=spread)
    e = exact(base, q, targets, w, scale)
    tl, tq, tb = tolerances(base, q, targets, w, scale, e, dtype)
    loss, (dq, db) = step(base, q, targets, w, scale)
    within(loss, e["loss"], tl, "loss")
    within(dq, e["dq"], tq, "dq")
    within(db, e["db"], tb, "db")


@pytest.mark.parametrize("scale", [1.0, 0.0, 1e-20])
@pytest.mark.parametrize("dtype,size", [("f32", 1e-22), ("f32", 1e-30), ("bf16", 1e-25), ("f16", 1e-3)])
@pytest.mark.parametrize("nq,dim", [(20, 40), (90, 200)])
def test_products_below_the_normal_range(nq, dim, dtype, size, scale):
    """every logit is next to zero: losses are log(nb), and targets and rows behind the last still take their own way"""
    base, q, targets, w, _ = make(nq, 301, dim, "f32", seed=dim)
    base, q = (base * size).to(DT[dtype]), (q * size).to(DT[dtype])
    e = exact(base, q, targets, w, scale)
    tl, tq, tb = tolerances(base, q, targets, w, scale, e, dtype)
    loss, (dq, db) = step(base, q, targets, w, scale)
    assert loss.sub(np.log(301.0)).abs().max() < 1e-5
    within(loss, e["loss"], tl, "loss")
    within(dq, e["dq"], tq, "dq")
    within(db, e["db"], tb, "db")


@pytest.mark.parametrize("scale", [1.0, 8.0])
@pytest.mark.parametrize("nq,nb,dim", [(1, 300, 40), (2, 1630, 177), (5, 200, 512), (70, 150, 200)])
def test_small_elements_of_fp32_rows_keep_their_digits(nq, nb, dim, scale):
    """Elements of five decades in a row: each gradient is compared with the size of its own terms.  An element x of a row whose largest is t is
    brought to x 2^-e with t 2^-e >= 2^14 and held as two fp16 halves: the second is rounded to 2^-11 of itself, 2^-22 |x|, or, where it is
    subnormal, to half of fp16's smallest step, 2^-25 2^e <= 2^-39 t."""
    base, q, targets, w, _ = make(nq, nb, dim, "f32", seed=nq + dim)
    g = torch.Generator().manual_seed(dim)
    shrink = 10.0 ** (-5 * torch.rand(dim, generator=g))
    base, q = base * shrink, q * shrink
    e = exact(base, q, targets, w, scale)
    tl, tq, tb = tolerances(base, q, targets, w, scale, e, "f32")
    tq = tq + scale * e["g"].abs() @ base.double().abs().amax(1, keepdim=True) * 2.0 ** -39
    tb = tb + scale * e["g"].abs().T @ q.double().abs().amax(1, keepdim=True) * 2.0 ** -39
    loss, (dq, db) = step(base, q, targets, w, scale)
    within(loss, e["loss"], tl, "loss")
    within(dq, e["dq"], tq, "dq")
    within(db, e["db"], tb, "db")


def test_small_losses_keep_their_digits():
    """a query that is answered well: loss = log(1 + what the others weigh), to fp32's digits and not to those of its log sums"""
    dim = 64
    base = torch.eye(dim)
    q = base[:32].clone()
    t = torch.arange(32, dtype=torch.int32)
    for scale in (20.0, 40.0, 80.0):
        loss, (dq, db) = step(base, q, t, torch.ones(32), scale)
        want = torch.log1p((dim - 1) * torch.exp(torch.tensor(-scale, dtype=torch.float64)))
        # z = scale * 1 is exact up to scale's product with log2 e: relative error of e^-scale is scale * 2u, and a few roundings
        assert ((loss.double().cpu() - want).abs() <= want * (2 * scale + 16) * U).all()
        miss = -torch.expm1(-want)
        assert ((dq.double().cpu()[torch.arange(32), t.long()] + scale * miss).abs() <= scale * miss * (4 * scale + 2.0 ** 4) * 4 * U).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [40, 93, 200])
def test_strides_and_what_lies_behind(dtype, dim):
    """rows inside a larger buffer, at an odd offset, NaN all around them: the same bits as from a tight copy"""
    base, q, targets, w, scale = make(37, 300, dim, dtype, seed=9)
    want_loss, (want_q, want_b) = step(base, q, targets, w, scale)
    for off, pad in ((0, 8), (1, 3), (8, 16)):
        def inside(t):
            buf = torch.full((t.shape[0] + 5, dim + off + pad), float("nan"), dtype=t.dtype, device="cuda")
            buf[2:-3, off:off + dim] = t.cuda()
            return buf[2:-3, off:off + dim]
        b, x = inside(base).requires_grad_(), inside(q).requires_grad_()
        loss = softmax.softmax_loss(x, b, targets.cuda(), scale)
        dq, db = torch.autograd.grad(loss, (x, b), w.cuda())
        assert torch.equal(loss, want_loss) and torch.equal(dq, want_q) and torch.equal(db, want_b), (off, pad)


def test_other_layouts_and_broadcasts():
    base, q, targets, w, scale = make(24, 130, 48, "f32", seed=10)
    want_loss, (want_q, want_b) = step(base, q, targets, w, scale)
    bt = base.t().contiguous().cuda().requires_grad_()             # held column by column
    x = q.cuda().requires_grad_()
    loss = softmax.softmax_loss(x, bt.t(), targets.cuda(), scale)
    dq, db = torch.autograd.grad(loss, (x, bt), w.cuda())
    assert torch.equal(loss, want_loss) and torch.equal(dq, want_q) and torch.equal(db.t(), want_b)
    one = q[:1].cuda().requires_grad_()                            # one query asked for every target: gradients add up
    loss = softmax.softmax_loss(one.expand(24, -1), base.cuda(), targets.cuda(), scale)
    (g,) = torch.autograd.grad(loss, one, w.cuda())
    many = q[:1].repeat(24, 1)
    wantl, (each,) = step(base, many, targets, w, scale, grads="q")
    assert torch.equal(loss, wantl)
    assert torch.allclose(g[0].double(), each.double().sum(0), rtol=0, atol=24 * U * each.abs().sum(0).max().item())
    x = q.cuda().requires_grad_()                                  # the gradient of a sum arrives as a broadcast
    (g1,) = torch.autograd.grad(softmax.softmax_loss(x, base.cuda(), targets.cuda(), scale).sum(), x)
    assert torch.equal(g1, step(base, q, targets, torch.ones(24), scale, grads="q")[1][0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cuts", [(0, 900), (0, 300, 900), (0, 0, 17, 17, 600, 899, 900)])
def test_shards_and_merge(dtype, cuts):
    """row shards, empty ones among them, joined: loss, dq (sum of the parts) and db (rows of the shards) of the whole"""
    base, q, targets, w, scale = make(60, 900, 120, dtype, seed=11)
    targets[::9] = -1
    e = exact(base, q, targets, w, scale)
    tl, tq, tb = tolerances(base, q, targets, w, scale, e, dtype)
    b, x, t, ww = base.cuda(), q.cuda(), targets.cuda(), w.cuda()
    base0 = 1000                                                   # ids of this base start here
    t = torch.where(t >= 0, t + base0, t)
    parts = [softmax.softmax_shard_dev(b[lo:hi], x, t, scale, id_base=base0 + lo, want_mean=True) for lo, hi in zip(cuts, cuts[1:])]
    lse, loss = softmax.softmax_merge_dev(torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]), t)
    within(loss, e["loss"], tl * len(parts), "loss")
    within(lse, e["lse"], tl * len(parts), "lse")
    dq, dbs = torch.zeros(60, 120, dtype=torch.float64), []
    for (lo, hi), p in zip(zip(cuts, cuts[1:]), parts):
        a, c = softmax.softmax_grad_dev(b[lo:hi], x, t, scale, lse, loss, ww, rest=p[0], mean=p[4], id_base=base0 + lo)
        dq += a.double().cpu()
        dbs.append(c)
    half = {"f32": U, "bf16": 2.0 ** -8}[dtype]
    assert ((dq - e["dq"]).abs() <= tq + half * e["aq"] * 2).all()       # every part is rounded by itself
    within(torch.cat(dbs), e["db"], tb, "db")


def test_empty_calls():
    b, x, t = torch.zeros(0, 16, device="cuda"), torch.randn(5, 16, device="cuda"), torch.tensor([0, 1, -1, 3, 4], dtype=torch.int32, device="cuda")
    rest, own, lse, loss, mean = softmax.softmax_shard_dev(b, x, t, 1.0, want_mean=True)
    assert (rest == -np.inf).all() and (own == -np.inf).all() and not mean.any()
    assert loss.tolist() == [np.inf, np.inf, 0.0, np.inf, np.inf]
    b = torch.randn(7, 16, device="cuda", requires_grad=True)
    x = torch.randn(0, 16, device="cuda", requires_grad=True)
    loss = softmax.softmax_loss(x, b, t[:0], 1.0)
    dq, db = torch.autograd.grad(loss, (x, b), torch.zeros(0, device="cuda"))
    assert loss.shape == (0,) and dq.shape == (0, 16) and db.shape == (7, 16) and not db.any()
    b = torch.randn(1, 16, device="cuda", requires_grad=True)      # one row: it is the answer for certain
    x = torch.randn(3, 16, device="cuda", requires_grad=True)
    loss = softmax.softmax_loss(x, b, torch.tensor([0, 0, -1], dtype=torch.int32, device="cuda"), 3.0)
    dq, db = torch.autograd.grad(loss, (x, b), torch.ones(3, device="cuda"))
    assert not loss.any() and not dq.any() and not db.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_values_that_are_not_finite(dtype):
    """a row or a query that is not finite shows in what it touches, and nowhere else"""
    base, q, targets, w, scale = make(20, 300, 40, dtype, seed=12)
    bad = q.clone()
    bad[6, 3] = float("nan")
    want = step(base, q, targets, w, scale)
    loss, (dq, db) = step(base, bad, targets, w, scale)
    ok = torch.arange(20) != 6
    assert loss[6].isnan() and torch.equal(loss[ok], want[0][ok]) and dq[6].isnan().all() and torch.equal(dq[ok], want[1][0][ok]) and db.isnan().all()
    worse = base.clone()
    worse[100, 5] = float("inf")
    loss, _ = step(worse, q, targets, w, scale)
    z = scale * q.double() @ worse.double().T
    down = z[:, 100] == -np.inf                                    # e^-inf is 0: such a row takes no part in the loss
    assert down.any() and not down.all()
    keep = [i for i in range(20) if down[i] and targets[i] != 100]
    e = exact(torch.cat((base[:100], base[101:])), q, torch.where(targets > 100, targets - 1, targets), w, scale)
    tl, _, _ = tolerances(base, q, targets, w, scale, e, dtype)
    assert ((loss.double().cpu() - e["loss"]).abs() <= tl)[keep].all()
    assert not torch.isfinite(loss[~down]).any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,dim", [(20, 40), (70, 93), (97, 200), (33, 512), (70, 1024), (40, 771)])
def test_queries_without_a_row_may_hold_anything(nq, dim, dtype):
    base, q, targets, w, scale = make(nq, 300, dim, dtype, seed=nq)
    out = torch.tensor([0, 3, 4, 19, nq - 1])
    targets[out] = -1
    q[out] = 0.0
    want = step(base, q, targets, w, scale)
    q[0], q[3, 1], q[4, dim - 1], q[19, 2], q[nq - 1, 0] = float("nan"), float("inf"), -float("inf"), float("nan"), float("nan")
    loss, (dq, db) = step(base, q, targets, w, scale)
    assert torch.equal(loss, want[0]) and torch.equal(dq, want[1][0]) and torch.equal(db, want[1][1])
    assert not loss[out].any() and not dq[out].any()


def test_targets_beyond_32_bits():
    base, q, targets, w, scale = make(8, 100, 24, "f32", seed=3)
    t = targets.long()
    t[0], t[1], t[2], t[3] = 2 ** 32 + 5, -2 ** 32, 2 ** 40 - 1, -1
    loss = softmax.softmax_loss(q.cuda(), base.cuda(), t.cuda(), scale).cpu()
    assert (loss[:3] == np.inf).all() and loss[3] == 0 and torch.equal(loss[4:], softmax.softmax_loss(q.cuda(), base.cuda(), targets.cuda(), scale).cpu()[4:])


@pytest.mark.parametrize("dtype,nq,nb,dim", [("f32", 70, 4_300_000, 8), ("bf16", 70, 8_500_000, 5), ("f32", 5, 270_000, 1000), ("f32", 300, 4_300_000, 8), ("bf16", 300, 8_500_000, 5)])
def test_a_base_of_more_than_one_piece(dtype, nq, nb, dim):
    """planes of fp32 and unaligned rows are made a gigabyte at a time; the sums go on from piece to piece"""
    gen = torch.Generator(device="cuda").manual_seed(dim)
    base = torch.randn(nb, dim, device="cuda", generator=gen).to(DT[dtype])
    q = torch.randn(nq, dim, device="cuda", generator=gen).to(DT[dtype])
    t = torch.randint(nb, (nq,), device="cuda", generator=gen, dtype=torch.int32)
    t[0], t[1], t[2], t[3] = 0, nb - 1, 4194304 % nb, -1
    w = torch.rand(nq, device="cuda", generator=gen) + 0.5
    scale = 2.0 * dim ** -0.5
    x = q.clone().requires_grad_()
    loss = softmax.softmax_loss(x, base, t, scale)
    dq, = torch.autograd.grad(loss, x, w)
    assert torch.equal(softmax.softmax_loss(q, base, t, scale), loss)
    e, parts = {}, [base[i:i + 200_000].double() for i in range(0, nb, 200_000)]
    has, rows = t >= 0, torch.arange(nq, device="cuda")
    tt = t.long().clamp(min=0)
    own = scale * (q.double() * base[tt].double()).sum(1)
    rest = torch.full((nq,), -np.inf, dtype=torch.float64, device="cuda")
    for pass_ in (0, 1):
        total, size = torch.zeros(nq, dim, dtype=torch.float64, device="cuda"), torch.zeros(nq, dim, dtype=torch.float64, device="cuda")
        for i, b in enumerate(parts):
            z = scale * (q.double() @ b.T.contiguous())
            here = has & (tt >= 200_000 * i) & (tt < 200_000 * i + b.shape[0])
            z[rows[here], tt[here] - 200_000 * i] = -np.inf
            if pass_ == 0:
                rest = torch.logaddexp(rest, torch.logsumexp(z, 1))
            else:
                p = torch.exp(z - e["lse"][:, None])
                total += p @ b
                size += p @ b.abs()
        if pass_ == 0:
            e["own"] = own.cpu()
            e["loss"] = torch.where(has, torch.nn.functional.softplus(rest - own, threshold=1e9), 0.0).cpu()
            e["lse"] = torch.where(has, torch.logaddexp(rest, own), rest)
    ww = torch.where(has, w.double(), 0.0)[:, None]
    miss = -torch.expm1(-e["loss"].cuda())[:, None]
    mine = base[tt].double()
    e["dq"] = (scale * ww * (total - miss * mine)).cpu()
    e["aq"] = (scale * ww * (size + miss * mine.abs())).cpu()
    top = float(base.double().norm(dim=1).max() * q.double().norm(dim=1).max() * scale)
    dz = top * (dim + 8) * U + (3 * 2.0 ** -22 * dim ** 0.5 * top if dtype == "f32" else 0)
    within(loss.detach(), e["loss"], 2 * dz + 4 * U * (e["loss"].abs() + e["own"].abs()) + 16 * U, "loss")
    half, out = {"f32": (2.0 ** -22, U), "bf16": (2.0 ** -8, 2.0 ** -8)}[dtype]
    largest = (ww[:, 0] * torch.maximum(miss[:, 0], torch.exp(top - e["lse"]))).cpu()[:, None]      # (no weight is larger)
    floor = (0.0 if dtype == "bf16" else 2.0 ** -32) * largest * scale * sum(b.abs().sum(0) for b in parts).cpu()[None]
    # sums in fp32: a few thousand terms a lane and slot, the lanes of an MFMA and the slots on top
    within(dq, e["dq"], e["aq"] * (2 * dz + half + (nb / 64 + 4096) * U) + floor + out * e["dq"].abs() + 1e-38, "dq")


@pytest.mark.parametrize("dtype,nq", [("bf16", 3), ("bf16", 70), ("f32", 70)])
def test_rows_beyond_4_gigabytes(dtype, nq):
    width = 2048 if dtype == "bf16" else 1024
    base = torch.empty(1_200_000, width, dtype=DT[dtype], device="cuda")[:, 100 * 8 : 100 * 8 + 40]
    gen = torch.Generator(device="cuda").manual_seed(nq)
    base.copy_(torch.randn(base.shape, device="cuda", generator=gen))
    q = torch.randn(nq, 40, device="cuda", generator=gen).to(DT[dtype])
    t = torch.randint(1_200_000, (nq,), device="cuda", generator=gen, dtype=torch.int32)
    t[-1] = 1_199_999
    got, want = [], []
    for b, to in ((base, got), (base.contiguous(), want)):
        x, b = q.clone().requires_grad_(), b.detach().requires_grad_()
        loss = softmax.softmax_loss(x, b, t, 0.2)
        to += [loss.detach(), *torch.autograd.grad(loss.sum(), (x, b))]
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.isfinite(got[0]).all() and got[2][-1].any()


def test_gradients_are_differences():
    """central differences of the loss the kernels give: h^2 / 6 times the third derivative, and the loss's rounding over h"""
    base, q, targets, _, _ = make(12, 90, 10, "f32", seed=13)
    scale, h = 3.0, 2.0 ** -5
    w = torch.ones(12)
    _, (dq, db) = step(base, q, targets, w, scale)
    e = exact(base, q, targets, w, scale)
    tl, _, _ = tolerances(base, q, targets, w, scale, e, "f32")
    b1 = (base.abs().max() * scale) ** 3
    q1 = (q.abs().max() * scale) ** 3
    for k in range(10):
        for axis in (0, 7):
            d = torch.zeros_like(q)
            d[axis, k] = h
            lp, lm = (step(base, q + s * d, targets, w, scale, "")[0].double().cpu().sum() for s in (1, -1))
            assert abs((lp - lm) / (2 * h) - dq[axis, k].item()) <= h * h / 6 * 8 * b1 + 2 * tl.sum() / h
            d = torch.zeros_like(base)
            d[axis, k] = h
            lp, lm = (step(base + s * d, q, targets, w, scale, "")[0].double().cpu().sum() for s in (1, -1))
            assert abs((lp - lm) / (2 * h) - db[axis, k].item()) <= 12 * h * h / 6 * 8 * q1 + 2 * tl.sum() / h


def raw_grad(base, q, t, scale, lse, loss, rest, mean, w, dq, db, work, n):
    import ctypes as C
    from roargraph_amd._lib import check, lib
    p, code = softmax._ptr, {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[base.dtype]
    check(lib().rg_softmax_grad_dev(p(base), C.c_uint32(base.shape[0]), C.c_uint64(base.stride(0)), p(q), C.c_uint32(q.shape[0]), C.c_uint64(q.stride(0)), C.c_uint32(base.shape[1]), C.c_int(code),
                                    C.c_float(scale), p(t), C.c_uint32(0), p(lse), p(loss), p(rest), p(mean), p(w), p(dq), C.c_uint64(dq.stride(0)), p(db), C.c_uint64(db.stride(0)), p(work),
                                    C.c_uint64(n), C.c_int(0), C.c_void_p(torch.cuda.current_stream().cuda_stream)))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nb,dim", [(33, 200, 24), (70, 1300, 93), (5, 90, 512)])
def test_nothing_else_is_written(dtype, nq, nb, dim):
    """scratch of exactly the bytes asked for, gradients inside wider buffers: what lies around them stays"""
    import ctypes as C
    from roargraph_amd._lib import check, lib
    base, q, targets, w, scale = make(nq, nb, dim, dtype, seed=14)
    want_loss, (want_q, want_b) = step(base, q, targets, w, scale)
    b, x, t, ww = base.cuda(), q.cuda(), targets.cuda(), w.cuda()
    code = {"f32": 0, "f16": 1, "bf16": 2}[dtype]
    p = softmax._ptr
    mark = 0x5a

    def scratch(what, rows):
        n = softmax.workspace(what, rows, nq, dim, code)
        buf = torch.full((n + 512,), mark, dtype=torch.uint8, device="cuda")
        return buf, n

    stats = torch.full((4, nq + 8), 77.0, device="cuda")
    mean = torch.full((nq + 3, dim), 77.0, device="cuda")
    work, n = scratch(softmax.MEAN, nb)
    check(lib().rg_softmax_shard_dev(p(b), C.c_uint32(nb), C.c_uint64(dim), p(x), C.c_uint32(nq), C.c_uint64(dim), C.c_uint32(dim), C.c_int(code), C.c_float(scale), p(t), C.c_uint32(0),
                                     p(stats[0]), p(stats[1]), p(stats[2]), p(stats[3]), p(mean), p(work), C.c_uint64(n), C.c_int(0), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert (work[n:] == mark).all() and (stats[:, nq:] == 77).all() and (mean[nq:] == 77).all()
    assert torch.equal(stats[3, :nq], want_loss)
    rest, _, lse, loss = stats.unbind(0)
    dq = torch.full((nq + 2, dim + 7), 77.0, device="cuda", dtype=b.dtype)
    db = torch.full((nb + 2, dim + 5), 77.0, device="cuda", dtype=b.dtype)
    work, n = scratch(softmax.GRAD, nb)
    raw_grad(b, x, t, scale, lse, loss, rest, mean, ww, dq, db, work, n)
    assert (work[n:] == mark).all()
    assert torch.equal(dq[:nq, :dim], want_q) and torch.equal(db[:nb, :dim], want_b)
    assert (dq[nq:] == 77).all() and (dq[:, dim:] == 77).all() and (db[nb:] == 77).all() and (db[:, dim:] == 77).all()


def test_streams_and_graphs():
    """on another stream, and captured: replayed on new inputs between eager calls, every replay equals the eager result"""
    def all_of(b, x, t, w):
        rest, own, lse, loss, mean = softmax.softmax_shard_dev(b, x, t, 8.0, want_mean=True)
        return (loss,) + softmax.softmax_grad_dev(b, x, t, 8.0, lse, loss, w, rest=rest, mean=mean)

    sets = [[a.cuda() for a in make(50, 3000, 200, "bf16", seed=20 + k)[:4]] for k in range(3)]
    want = [all_of(*s) for s in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = all_of(*sets[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    held = [a.clone() for a in sets[0]]
    with torch.cuda.stream(side):
        all_of(*held)
        side.synchronize()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]        # two graphs, each with scratch of its own
        outs = []
        for g in graphs:
            with torch.cuda.graph(g, stream=side):
                outs.append(all_of(*held))
    torch.cuda.synchronize()
    for k in (1, 2, 0, 1):
        for h, s in zip(held, sets[k]):
            h.copy_(s)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        eager = all_of(*sets[k])
        torch.cuda.synchronize()
        for out in outs + [eager]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k])), k


def test_trained_packed_and_searched():
    """the operators as they are used: ground truth ids train a table, the trained table is packed and scored, and the best rows re-scored"""
    from roargraph_amd import groundtruth, q4, synth
    base, queries = synth.make_synth(21, 4000, 64, 200)
    b, x = torch.from_numpy(base).cuda().requires_grad_(), torch.from_numpy(queries).cuda()
    ids, dists = groundtruth.compute_groundtruth(base, queries, "ip", 10)
    targets = torch.from_numpy(ids[:, 0].astype(np.int32)).cuda()
    scale = 1.0
    loss = softmax.softmax_loss(x, b, targets, scale)
    e = exact(b.detach().cpu(), x.cpu(), targets.cpu(), torch.full((64,), 1 / 64), scale)
    tl, _, tb = tolerances(b.detach().cpu(), x.cpu(), targets.cpu(), None, scale, e, "f32")
    within(loss.detach(), e["loss"], tl, "loss")
    loss.mean().backward()
    within(b.grad, e["db"], tb, "db")
    trained = (b.detach() - 0.1 * b.grad).contiguous()
    packed = q4.q4_pack(trained, group=32)
    scores = q4.q4_score(x, packed)
    top = scores.topk(10, dim=1).indices
    rows = q4.q4_unpack(packed, top.reshape(-1)).reshape(64, 10, 200).double()
    again = (rows * x.double()[:, None]).sum(2)
    # fp32 sums of 200 products, and 22 bits of a query's elements relative to its largest
    tol = (200 + 8) * U * rows.norm(dim=2) * x.double().norm(dim=1, keepdim=True) + 2.0 ** -22 * rows.abs().sum(2) * x.double().abs().amax(1, keepdim=True)
    assert ((scores.gather(1, top).double() - again).abs() <= tol).all()
    # the packed table's own loss: its values are a table like any other
    values = q4.q4_unpack(packed)
    e = exact(values.cpu(), x.cpu(), targets.cpu(), torch.full((64,), 1 / 64), scale)
    tl, _, _ = tolerances(values.cpu(), x.cpu(), targets.cpu(), None, scale, e, "f32")
    within(softmax.softmax_loss(x, values, targets, scale), e["loss"], tl, "loss over the packed table")


def test_python_refusals():
    b, x, t = torch.zeros(8, 16, device="cuda"), torch.zeros(4, 16, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (lambda: softmax.softmax_loss(x.half(), b, t), lambda: softmax.softmax_loss(x.double(), b.double(), t)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: softmax.softmax_loss(x[:, :8], b, t), lambda: softmax.softmax_loss(x, b, t[:3]), lambda: softmax.softmax_loss(x, b, t.float()),
                lambda: softmax.softmax_loss(x, b.cpu(), t.cpu()), lambda: softmax.softmax_loss(x[0], b, t[:1])):
        with pytest.raises(ValueError):
            bad()
    from roargraph_amd._lib import RgError
    with pytest.raises(RgError, match="finite"):
        softmax.softmax_loss(x, b, t, float("nan"))
    with pytest.raises(RgError, match="dim"):
        softmax.softmax_loss(torch.zeros(4, 1025, device="cuda"), torch.zeros(8, 1025, device="cuda"), t)
