"""-m gpu: softmax cross entropy over a base where its digits cancel, and where values are not finite (rg_softmax_*), against the definition in 64 bits.

The formats' roundings are those of test_gpu_softmax: half a step of bf16 is 2^-8 of a value, of fp16 2^-11, of fp32 2^-24 (U)."""
import numpy as np
import pytest
import torch

import test_gpu_softmax
from roargraph_amd import softmax
from test_gpu_softmax import DT, U, exact, make, step, tolerances, within

pytestmark = pytest.mark.gpu

HALF = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def rounded(x, dtype):
    return x.to(DT[dtype]).double()


# ---- digits of the gradients

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nb,dim", [(3, 20000, 200), (20, 20000, 64), (300, 20000, 200), (40, 6000, 1024), (150, 9000, 93)])
@pytest.mark.parametrize("dist", [0.1, 0.03])
def test_a_hard_negative_next_to_the_target(nq, nb, dim, dist, dtype):
    """A query is answered by rows that lie `dist` beside its target t: dq = w scale (part mean - miss b_t) is small beside mean and b_t.  What a rounding
    of the weights may do to it: with W_j = P_j (1 + d_j), |d_j| <= h, and the mean taken over the W,
      mean' - mean = sum p_j d_j (b_j - mean) / (1 + sum p_j d_j),  at most h / (1 - h) sum p_j |b_j - mean|
    -- small where the rows that have it all are alike, whatever their weights are rounded to.  (Divided by the sum of the P, the mean is off by up to h of itself.)"""
    g = torch.Generator().manual_seed(nq + dim)
    base = torch.randn(nb, dim, generator=g)
    base /= base.norm(dim=1, keepdim=True)
    at = torch.randperm(nb // 10, generator=g)[:nq] * 10
    t = at + 9
    off = torch.randn(nq, dim, generator=g)
    n = base[t] + dist * off / off.norm(dim=1, keepdim=True)
    for k in range(8):                                             # (eight of them, a little shorter each: their weights are no powers of two)
        base[at + k] = n * (1 - 0.013 * k)
    q = n + 0.3 * torch.randn(nq, dim, generator=g) / dim ** 0.5
    base, q, w, scale, targets = base.to(DT[dtype]), q.to(DT[dtype]), torch.ones(nq), 16.0, t.int()
    e = exact(base, q, targets, w, scale)
    got = step(base, q, targets, w, scale, grads="q")[1][0].double().cpu()
    b, half = base.double(), HALF[dtype]
    z = e["z"].clone()
    z[torch.arange(nq), t] = -np.inf
    p = torch.exp(z - e["rest"][:, None])
    mean = p @ b
    spread = (p * torch.cdist(mean, b)).sum(1)
    size = (p * b.norm(dim=1)[None]).sum(1)
    miss, bt = -torch.expm1(-e["loss"]), b[t].norm(dim=1)
    dz = float(b.norm(dim=1).max() * q.double().norm(dim=1).max()) * scale * (dim + 8) * U
    # the weights' rounding and the logits'; sums of 32 products each in fp32, in tiles and slots; part and miss are made apart, of rest, lse and loss
    delta = scale * miss * ((half / (1 - half) + 2 * dz) * spread + (nb / 32 + 256 + 64) * U * size + 2 * dz * (mean - b[t]).norm(dim=1)
                            + (2 * (e["rest"].abs() + e["lse"].abs()) + 16) * U * bt)
    last = (rounded(e["dq"], dtype) - e["dq"]).norm(dim=1)
    worst = ((got - e["dq"]).norm(dim=1) / (last + 2 * delta)).max().item()        # (rounded from delta beside: |got - x| <= |round(x) - x| + 2 delta)
    assert worst <= 1.0, worst


@pytest.mark.parametrize("nq,nb,dim", [(100, 20000, 200), (700, 20000, 64), (100, 6000, 1024), (60, 9000, 512), (33, 5000, 93)])
def test_the_weight_of_a_target_keeps_16_bits(nq, nb, dim):
    """bf16, gradient of the rows that are a target: nearly all of it is -w (1 - p) q of one query, which is multiplied to 16 bits, so that its error is that of
    the last rounding (0.0017 of the norm; with 8 bits of that weight 0.0024); the other queries' weights, rounded to 8 bits, are few"""
    base, q, _, _, _ = make(nq, nb, dim, "bf16", seed=nq)
    targets = torch.randperm(nb, generator=torch.Generator().manual_seed(1))[:nq].int()
    g = torch.Generator().manual_seed(2)
    w, scale = 0.5 + torch.rand(nq, generator=g), 1.0
    e = exact(base, q, targets, w, scale)
    got = step(base, q, targets, w, scale, grads="b")[1][0].double().cpu()
    t = targets.long()
    x = q.double().abs()
    own = e["g"][torch.arange(nq), t].abs()
    others = e["g"].abs()[:, t]
    others[torch.arange(nq), torch.arange(nq)] = 0
    dz = float(base.double().norm(dim=1).max() * x.norm(dim=1).max()) * scale * (dim + 8) * U
    delta = scale * ((2.0 ** -8 + 2 * dz) * others.T @ x + (2.0 ** -16 + 2 * dz) * own[:, None] * x + (nq + 8) * U * (others.T @ x + own[:, None] * x))
    want = e["db"][t]
    last = (rounded(want, "bf16") - want).norm()
    assert (got[t] - want).norm() <= last + 2 * delta.norm(), ((got[t] - want).norm() / want.norm(), last / want.norm(), delta.norm() / want.norm())
    assert last + 2 * delta.norm() < 0.0021 * want.norm()          # (the bound tells the two apart)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nb,dim", [(33, 300, 40), (200, 500, 200), (20, 90, 520)])
@pytest.mark.parametrize("size", [1e24, 1e-24, 1e28])
def test_rows_and_queries_of_opposite_sizes(nq, nb, dim, size, dtype):
    """logits of ordinary size made of large queries and small rows, or the other way round: both gradients are far from 1"""
    base, q, targets, w, scale = make(nq, nb, dim, "f32", seed=dim)
    base, q = (base / size).to(DT[dtype]), (q * size).to(DT[dtype])
    e = exact(base, q, targets, w, scale)
    tl, tq, tb = tolerances(base, q, targets, w, scale, e, dtype)
    loss, (dq, db) = step(base, q, targets, w, scale)
    within(loss, e["loss"], tl, "loss")
    within(dq, e["dq"], tq, "dq")
    within(db, e["db"], tb, "db")


# ---- values that are not finite

def sharded(base, q, t, w, scale, cuts):
    b, x, tt, ww = base.cuda(), q.cuda(), t.cuda(), w.cuda()
    parts = [softmax.softmax_shard_dev(b[lo:hi], x, tt, scale, id_base=lo, want_mean=True) for lo, hi in zip(cuts, cuts[1:])]
    lse, loss = softmax.softmax_merge_dev(torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]), tt)
    grads = [softmax.softmax_grad_dev(b[lo:hi], x, tt, scale, lse, loss, ww, rest=p[0], mean=p[4], id_base=lo) for (lo, hi), p in zip(zip(cuts, cuts[1:]), parts)]
    return lse.cpu(), loss.cpu(), sum(g[0].double().cpu() for g in grads), torch.cat([g[1] for g in grads]).cpu()


CUTS = [(0, 300), (0, 150, 300), (0, 70, 70, 299, 300)]


@pytest.mark.parametrize("cuts", CUTS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_a_query_of_nan_shows_over_shards(dtype, cuts):
    """wherever its target lies, and where it has none: not like a query whose target no shard holds"""
    base, q, targets, w, scale = make(20, 300, 40, dtype, seed=30)
    targets[0], targets[6], targets[7], targets[8], targets[9] = -1, 20, 299, 300, -1
    want = sharded(base, q, targets, w, scale, cuts)
    assert want[1][8] == np.inf and want[1][9] == 0
    bad = q.clone()
    bad[6:10, 3] = float("nan")
    lse, loss, dq, db = sharded(base, bad, targets, w, scale, cuts)
    ok = torch.tensor([i for i in range(20) if not 6 <= i <= 9])
    assert torch.equal(loss[ok], want[1][ok]) and torch.equal(lse[ok], want[0][ok]) and torch.equal(dq[ok], want[2][ok])
    assert loss[6:9].isnan().all() and loss[9] == 0 and lse[6:10].isnan().all()
    assert dq[6:9].isnan().all() and not dq[9].any() and db.isnan().all()


@pytest.mark.parametrize("cuts", CUTS[:2])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq", [20, 300])
def test_a_row_of_nan_shows_over_shards(nq, dtype, cuts):
    base, q, targets, w, scale = make(nq, 300, 40, dtype, seed=31)
    targets[0] = -1
    base[200, 1] = float("nan")
    lse, loss, dq, db = sharded(base, q, targets, w, scale, cuts)
    assert loss[1:].isnan().all() and loss[0] == 0 and lse.isnan().all() and dq[1:].isnan().all(1).all() and not dq[0].any()


@pytest.mark.parametrize("cuts", CUTS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq", [20, 300])
def test_a_target_of_infinity(nq, dtype, cuts):
    """z_target = +inf: inf - inf, no perfect answer (loss and lse NaN).  z_target = -inf: loss +inf, lse without it, and the other rows' gradients as they are."""
    base, q, targets, w, scale = make(nq, 300, 40, dtype, seed=32)
    targets[targets == 100] = 101
    base[100, 5] = float("inf")
    q[:, 5] = -q[:, 5].abs().clamp(min=0.01)                      # every query gives row 100 a logit of -inf ...
    targets[3] = 100
    q[4, 5], targets[4] = 0.25, 100                               # ... and this one +inf
    lse, loss, dq, db = sharded(base, q, targets, w, scale, cuts)
    one = step(base, q, targets, w, scale)[0].cpu()
    assert torch.equal(one.isnan(), loss.isnan()) and torch.equal(one == np.inf, loss == np.inf)
    assert loss[4].isnan() and lse[4].isnan() and dq[4].isnan().all()
    keep = torch.tensor([i for i in range(nq) if i != 4])
    without = torch.cat((base[:100], base[101:]))
    t = torch.where(targets > 100, targets - 1, targets)
    t[3], t[4] = -1, -1
    e = exact(without, q, t, w, scale)
    tl, _, _ = tolerances(without, q, t, w, scale, e, dtype)
    rest = [i for i in keep.tolist() if i != 3]
    assert ((one.double() - e["loss"]).abs() <= tl)[rest].all()
    tl = tl * len(cuts)
    assert ((loss.double() - e["loss"]).abs() <= tl)[rest].all() and ((lse.double() - e["lse"]).abs() <= tl + 4 * U * e["lse"].abs())[keep].all()
    assert loss[3] == np.inf
    # db of the other rows where the query of NaN takes no part
    targets[4] = -1
    lse, loss, dq, db = sharded(base, q, targets, w, scale, cuts)
    x, ww = q.double(), w.double().clone()
    ww[4] = 0
    p = torch.exp(e["z"] - e["lse"][:, None]) * ww[:, None]
    for i in rest:
        if t[i] >= 0:
            p[i, t[i]] -= ww[i]
    size = p.abs()
    want = scale * p.T @ x
    # (t = -1 for query 3 in the oracle's tolerances, so they are made here: weights off by the rounding and by 2 |dz|, sums, the last rounding)
    top = float(without.double().norm(dim=1).max() * x.norm(dim=1).max()) * scale
    dz = top * 48 * U + (3 * 2.0 ** -22 * 40 ** 0.5 * top if dtype == "f32" else 0)
    half = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    tol = scale * (half + 4 * dz + (nq + 8) * U) * size.T @ x.abs() + HALF[dtype] * want.abs() + {"f32": 1e-30, "f16": 2.0 ** -24, "bf16": 1e-30}[dtype]
    tol = tol + scale * 2.0 ** -32 * size.amax(0)[:, None] * x.abs().sum(0)[None]
    others = torch.cat((db[:100], db[101:])).double()
    assert torch.isfinite(others).all() and ((others - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,dim", [(20, 40), (300, 40), (9, 520), (200, 700)])
def test_a_row_of_minus_infinity_shows_in_the_queries_gradients(nq, dim, dtype):
    """a row with an infinity whose logits are all -inf takes no part in the losses; 0 times infinity is no number, so the gradients of the queries show it"""
    base, q, targets, w, scale = make(nq, 300, dim, dtype, seed=33)
    targets[targets == 100] = 101
    targets[0] = -1
    base[100, 5] = float("inf")
    q[:, 5] = -q[:, 5].abs().clamp(min=0.01)
    loss, (dq,) = step(base, q, targets, w, scale, grads="q")
    assert torch.isfinite(loss).all() and dq[1:, 5].isnan().all() and not dq[0].any()


@pytest.mark.parametrize("scale", [20.0, 40.0, 80.0])
def test_small_losses_keep_their_digits_over_shards(scale):
    """loss = log(1 + e^(rest - own)) of two shards: rest and own are fp32 values, off by U of themselves, and by 2 U scale as in the one-shard form"""
    base, q = torch.eye(64), torch.eye(64)[:32]
    t = torch.arange(32, dtype=torch.int32)
    lse, loss, dq, db = sharded(base, q, t, torch.ones(32), scale, (0, 20, 64))
    want = torch.log1p(63 * torch.exp(torch.tensor(-scale, dtype=torch.float64)))
    # (the shards' rests are logs of at most 63; the last two terms: 4 of them, and a few roundings of the loss)
    assert ((loss.double() - want).abs() <= want * (3 * scale + 4 * 4.2 + 16) * U).all()


def test_a_merge_is_as_good_as_its_lists():
    """loss = log(1 + e^d), d = rest - own of the lists' fp32 values: d is off by U of itself and by 4 U of its sum's logarithm (fp32 sum of 3 terms, each to 2 ulp), however
    large rest and own are; exponential and logarithm of the loss to 2 ulp each"""
    g = torch.Generator().manual_seed(50)
    nq = 2000
    base = torch.rand(nq, generator=g) * 400 - 200
    rest = base[None] + torch.randn(3, nq, generator=g) * 2
    own = torch.full((3, nq), -np.inf)
    own[torch.arange(nq) % 3, torch.arange(nq)] = base + torch.randn(nq, generator=g) * 4
    t = torch.zeros(nq, dtype=torch.int32)
    lse, loss = softmax.softmax_merge_dev(rest.cuda(), own.cuda(), t.cuda())
    r, o = torch.logsumexp(rest.double(), 0), own.double().amax(0)
    d = r - o
    want = torch.nn.functional.softplus(d, threshold=1e9)
    assert ((loss.cpu().double() - want).abs() <= torch.sigmoid(d) * (d.abs() + 12) * U + 8 * U * want).all()
    assert ((lse.cpu().double() - (o + want)).abs() <= U * (o + want).abs() + 2 * U * o.abs() + 20 * U * (1 + want)).all()


# ---- calls

def asked(monkeypatch):
    """which kinds of scratch calls ask for"""
    kinds, scratch = [], softmax._scratch
    monkeypatch.setattr(softmax, "_scratch", lambda what, *a: kinds.append(what) or scratch(what, *a))
    return kinds


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_without_gradients_no_mean_is_made(monkeypatch, mode):
    base, q, targets, w, scale = make(30, 500, 40, "bf16", seed=34)
    kinds = asked(monkeypatch)
    b, x, t = base.cuda().requires_grad_(), q.cuda().requires_grad_(), targets.cuda()
    want = softmax.softmax_loss(x, b, t, scale)
    with mode():
        loss = softmax.softmax_loss(x, b, t, scale)
    assert torch.equal(loss, want) and not loss.requires_grad
    softmax.softmax_loss(x.detach(), b, t, scale)
    assert kinds == [softmax.MEAN, softmax.STATS, softmax.STATS]


def test_a_learned_scale_goes_into_the_queries():
    """scale is a number; queries * s gives a learned one its gradient: dL/ds = sum_i q_i . dL/d(s q_i)"""
    base, q, targets, w, scale = make(30, 500, 40, "f32", seed=35)
    b, x, t = base.cuda(), q.cuda(), targets.cuda()
    s = torch.tensor(8.0, device="cuda", requires_grad=True)
    with pytest.raises(TypeError, match="queries"):
        softmax.softmax_loss(x, b, t, s)
    with pytest.raises(TypeError, match="queries"):
        softmax.softmax_loss(x, b, t, scale=s.log().exp())
    want = softmax.softmax_loss(x, b, t, 8.0)
    with torch.no_grad():
        assert torch.equal(softmax.softmax_loss(x, b, t, s), want)
    assert torch.equal(softmax.softmax_loss(x, b, t, s.detach()), want)
    loss = softmax.softmax_loss(x * s, b, t)
    (ds,) = torch.autograd.grad(loss, s, w.cuda())
    e = exact(base, q * 8.0, targets, w, 1.0)
    tl, tq, _ = tolerances(base, q * 8.0, targets, w, 1.0, e, "f32")
    within(loss.detach(), e["loss"], tl, "loss")
    x64 = q.double()
    assert abs(ds.item() - (e["dq"] * x64).sum().item()) <= ((tq + (30 * 40) * U * e["dq"].abs()) * x64.abs()).sum().item()


def test_a_whole_step_is_captured():
    """forward and backward of leaves that no eager graph holds, replayed on new inputs between eager steps"""
    sets = [[a.cuda() for a in make(50, 3000, 200, "bf16", seed=40 + k)[:4]] for k in range(3)]

    def run(b, x, t, w):
        loss = softmax.softmax_loss(x, b, t, 8.0)
        return (loss.detach(),) + torch.autograd.grad(loss, (x, b), w)

    def leaves(s):
        return s[0].clone().requires_grad_(), s[1].clone().requires_grad_(), s[2].clone(), s[3].clone()

    want = [run(*leaves(s)) for s in sets]
    held, side, graph = leaves(sets[0]), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        run(*held)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = run(*held)
    torch.cuda.synchronize()
    for k in (1, 2, 0, 1):
        with torch.no_grad():
            for h, s in zip(held, sets[k]):
                h.copy_(s)
        torch.cuda.synchronize()
        graph.replay()
        eager = run(*leaves(sets[k]))
        torch.cuda.synchronize()
        for a, b, c in zip(out, eager, want[k]):
            assert torch.equal(a, c) and torch.equal(b, c), k


# ---- the kernels that the shapes of test_gpu_softmax leave out: widths, types and numbers of queries in other pairs

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nb,dim", [(300, 900, 37), (300, 900, 93), (40, 900, 96), (260, 700, 201), (270, 700, 243), (80, 900, 256), (200, 700, 256), (20, 600, 320), (30, 600, 350), (300, 500, 509),
                                       (20, 500, 512), (300, 400, 701), (300, 300, 1001), (20, 400, 1001)])
def test_loss_and_gradients_of_other_pairs(nq, nb, dim, dtype):
    test_gpu_softmax.test_loss_and_gradients(nq, nb, dim, dtype)
