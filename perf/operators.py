"""The model-side operators over a base: what they compute in plain torch, and the sizes they are measured at.

step   one training step of an embedding model whose classes are the rows of a base (queries in, the id of the right row as the
       target): softmax cross entropy over ALL rows, its loss per query and the gradients of queries and base
loss   the same loss without gradients (evaluating a query set; the perplexity of single queries)
score  inner products of a few queries with every row of a base held in 4 bits with one scale per group of elements
pack   a base into that 4-bit form, and the values the form stands for

With `own` the calls a user of roargraph_amd makes, without it elementary torch operations in 32 bits."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a unit-test sized table, where only latency counts
        {"name": "step-f32-64x1000-d24", "op": "step", "dtype": "f32", "nq": 64, "nb": 1000, "dim": 24, "grad_base": True},
        # fp32 tables as the index itself holds them, a medium batch, wide rows
        {"name": "step-f32-512x250k-d512", "op": "step", "dtype": "f32", "nq": 512, "nb": 250_000, "dim": 512, "grad_base": True},
        # the text-to-image shape of the benchmark at a million rows: the heaviest step, everything trained
        {"name": "step-bf16-2048x1m-d200", "op": "step", "dtype": "bf16", "nq": 2048, "nb": 1_000_000, "dim": 200, "grad_base": True},
        # an adapter of the queries trained against a frozen base
        {"name": "step-bf16-4096x250k-d512-q", "op": "step", "dtype": "bf16", "nq": 4096, "nb": 250_000, "dim": 512, "grad_base": False},
        # ragged everything: odd batch, odd rows, odd width (rows not 16-byte aligned)
        {"name": "step-f16-333x70001-d93", "op": "step", "dtype": "f16", "nq": 333, "nb": 70_001, "dim": 93, "grad_base": True},
        # the benchmark's query set evaluated against part of its base
        {"name": "loss-f32-10000x200k-d200", "op": "loss", "dtype": "f32", "nq": 10_000, "nb": 200_000, "dim": 200},
        # one query against a large base: reading the base is all there is
        {"name": "loss-bf16-1x1m-d512", "op": "loss", "dtype": "bf16", "nq": 1, "nb": 1_000_000, "dim": 512},
        # one query against a small 4-bit base: latency
        {"name": "score-f32-1x2000-d200-g32", "op": "score", "dtype": "f32", "nq": 1, "nb": 2000, "dim": 200, "group": 32, "mins": False},
        # one query against the benchmark's whole base
        {"name": "score-f32-1x10m-d200-g32", "op": "score", "dtype": "f32", "nq": 1, "nb": 10_000_000, "dim": 200, "group": 32, "mins": False},
        # a small batch, wide rows, with minima
        {"name": "score-bf16-8x1m-d512-g64-min", "op": "score", "dtype": "bf16", "nq": 8, "nb": 1_000_000, "dim": 512, "group": 64, "mins": True},
        # packing a base as the index holds it, and an odd one with minima
        {"name": "pack-f32-1m-d200-g32", "op": "pack", "dtype": "f32", "nb": 1_000_000, "dim": 200, "group": 32, "mins": False},
        {"name": "pack-bf16-100003-d301-g128-min", "op": "pack", "dtype": "bf16", "nb": 100_003, "dim": 301, "group": 128, "mins": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("step", "step", "step", "loss", "loss", "score", "score", "pack"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    dim = rng.choice((96, 128, 200, 256, 384, 512, 768, 1024)) if rng.random() < 0.5 else _log(rng, 8, 1024)
    if op in ("step", "loss"):
        nq, nb = _log(rng, 1, 4096), _log(rng, 500, 1_000_000)
        while nq * nb * dim > 2048 * 1_000_000 * 200 // (3 if dtype == "f32" else 1) or nq * nb > 2_048_000_000 or nb * dim > 250_000_000:
            nq, nb = _log(rng, 1, 4096), _log(rng, 500, 1_000_000)
        case = {"op": op, "dtype": dtype, "nq": nq, "nb": nb, "dim": dim}
        if op == "step":
            case["grad_base"] = rng.random() < 0.7
        return case
    nb = _log(rng, 1000, 10_000_000)
    while nb * dim > (2_000_000_000 if op == "score" else 200_000_000):
        nb = _log(rng, 1000, 10_000_000)
    case = {"op": op, "dtype": dtype, "nb": nb, "dim": dim, "group": rng.choice((32, 64, 128)), "mins": rng.random() < 0.5}
    if op == "score":
        case["nq"] = rng.choice((1, 1, 2, 3, 4, 8, 13, 16))
    return case


def _rows(n, dim, gen):
    """unit rows, as embedding models give them"""
    x = torch.randn(n, dim, device="cuda", generator=gen)
    return x.div_(x.norm(dim=1, keepdim=True))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, dim, nb = DTYPES[case["dtype"]], case["dim"], case["nb"]
    s = {"op": case["op"], "dim": dim}
    if case["op"] in ("step", "loss"):
        nq = case["nq"]
        base = _rows(nb, dim, gen)
        targets = torch.randint(nb, (nq,), device="cuda", generator=gen, dtype=torch.int32)
        queries = base[targets.long()] * 0.6 + _rows(nq, dim, gen) * 0.8   # the other modality: near its row, and off it
        if nq > 8:
            targets[torch.randint(nq, (nq // 64 + 1,), device="cuda", generator=gen)] = -1   # queries that have no row here
        s.update(base=base.to(dt), queries=queries.to(dt), targets=targets, scale=20.0, grad_base=case.get("grad_base", False))
        s["weights"] = (torch.rand(nq, device="cuda", generator=gen) + 0.5) / nq
        s["grad"] = case["op"] == "step"
        if s["grad"]:
            s["queries"].requires_grad_(True)
            s["base"].requires_grad_(s["grad_base"])
        return s
    s.update(group=case["group"])
    if case["op"] == "pack":
        s.update(base=_rows(nb, dim, gen).to(dt), mins=case["mins"])
        return s
    groups = -(-dim // case["group"])
    s["codes"] = torch.randint(256, (nb, -(-dim // 8) * 4), device="cuda", generator=gen, dtype=torch.uint8)
    s["scales"] = ((torch.rand(nb, groups, device="cuda", generator=gen) + 0.5) * (0.4 / math.sqrt(dim))).half()
    s["mins"] = (s["scales"].float() * -(torch.rand(nb, groups, device="cuda", generator=gen) + 7)).half() if case["mins"] else None
    s["queries"] = _rows(case["nq"], dim, gen).to(dt)
    return s


def _plain_softmax(s):
    q, b = s["queries"].detach().float(), s["base"].detach().float()
    has = s["targets"] >= 0
    t = s["targets"].long().clamp(min=0)
    z = (q @ b.T).mul_(s["scale"])
    own_z = z.gather(1, t[:, None])[:, 0]
    top = z.amax(dim=1, keepdim=True)
    e = z.sub_(top).exp_()
    total = e.sum(dim=1, keepdim=True)
    loss = torch.where(has, total[:, 0].log() + top[:, 0] - own_z, 0.0)
    if not s["grad"]:
        return loss
    w = torch.where(has, s["weights"], 0.0)
    g = e.mul_(w[:, None] / total)                 # weight x probability
    g.scatter_add_(1, t[:, None], -w[:, None])
    dq = (g @ b).mul_(s["scale"]).to(s["queries"].dtype)
    if not s["grad_base"]:
        return loss, dq
    return loss, dq, (g.T @ q).mul_(s["scale"]).to(s["base"].dtype)


def _unpack(codes, dim):
    c = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(codes.shape[0], -1)
    return c[:, :dim]


def _spread(x, dim, group):
    return x.float().repeat_interleave(group, dim=1)[:, :dim]


def _plain_score(s):
    c = _unpack(s["codes"], s["dim"]).float()
    if s["mins"] is None:
        w = c.sub_(8).mul_(_spread(s["scales"], s["dim"], s["group"]))
    else:
        w = c.mul_(_spread(s["scales"], s["dim"], s["group"])).add_(_spread(s["mins"], s["dim"], s["group"]))
    return s["queries"].float() @ w.T


def _plain_pack(s):
    x, dim, group = s["base"].float(), s["dim"], s["group"]
    groups = -(-dim // group)
    pad = groups * group - dim
    y = torch.cat((x, x[:, -1:].expand(-1, pad)), dim=1).reshape(x.shape[0], groups, group)   # the last group holds fewer elements
    # a value next to the border of two codes goes to the nearer one: the quotient is taken in 64 bits
    if not s["mins"]:
        scale = (y.abs().amax(dim=2) / 7).half()
        w = scale.double()[:, :, None]
        c = torch.where(w > 0, (y.double() / w).round().clamp(-8, 7), 0.0)
        return (c.float() * scale.float()[:, :, None]).reshape(x.shape[0], -1)[:, :dim].contiguous(), scale
    low = y.amin(dim=2)
    scale, low = ((y.amax(dim=2) - low) / 15).half(), low.half()
    w = scale.double()[:, :, None]
    c = torch.where(w > 0, ((y.double() - low.double()[:, :, None]) / w).round().clamp(0, 15), 0.0)
    value = c.float() * scale.float()[:, :, None] + low.float()[:, :, None]
    return value.reshape(x.shape[0], -1)[:, :dim].contiguous(), scale, low


def run(state):
    s = state
    if own:
        from roargraph_amd import q4, softmax
        if s["op"] == "score":
            return q4.q4_score(s["queries"], q4.Q4Base(s["codes"], s["scales"], s["mins"], s["dim"], s["group"]))
        if s["op"] == "pack":
            packed = q4.q4_pack(s["base"], group=s["group"], mins=s["mins"])
            return (q4.q4_unpack(packed), packed.scales) + ((packed.mins,) if s["mins"] else ())
        loss = softmax.softmax_loss(s["queries"], s["base"], s["targets"], scale=s["scale"])
        if not s["grad"]:
            return loss
        leaves = (s["queries"], s["base"]) if s["grad_base"] else (s["queries"],)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves, s["weights"])
    return {"step": _plain_softmax, "loss": _plain_softmax, "score": _plain_score, "pack": _plain_pack}[s["op"]](s)


def work(case):
    n, nb, dim = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]], case["nb"], case["dim"]
    if case["op"] in ("step", "loss"):
        nq = case["nq"]
        read = (nq + nb) * dim * n + nq * 8
        if case["op"] == "loss":
            return {"bytes": read + nq * 4, "flops": 2 * nq * nb * dim}
        both = case["grad_base"]
        return {"bytes": read + nq * 8 + (nq + (nb if both else 0)) * dim * n, "flops": (6 if both else 4) * nq * nb * dim}
    groups = -(-dim // case["group"])
    held = nb * (-(-dim // 2) + groups * (4 if case["mins"] else 2))
    if case["op"] == "score":
        return {"bytes": held + case["nq"] * (dim * n + nb * 4), "flops": 2 * case["nq"] * nb * dim}
    return {"bytes": nb * dim * (n + 4) + held, "flops": 3 * nb * dim}


def _exact_softmax(s):
    q, b, scale = s["queries"].detach().double(), s["base"].detach(), float(s["scale"])
    nq, nb, t = q.shape[0], b.shape[0], s["targets"].long()
    piece = max(1, min(nb, 400_000_000 // nq))
    spans = [(i, min(nb, i + piece)) for i in range(0, nb, piece)]
    lse = torch.full((nq,), -math.inf, device=q.device, dtype=torch.float64)
    for lo, hi in spans:
        lse = torch.logaddexp(lse, torch.logsumexp(scale * (q @ b[lo:hi].double().T), dim=1))
    ask = t >= 0
    right = b[t.clamp(min=0)].double()
    loss = torch.where(ask, lse - scale * (q * right).sum(dim=1), 0.0)
    if not s["grad"]:
        return loss
    w = torch.where(ask, s["weights"].double(), 0.0)
    dq = -(w * scale)[:, None] * right
    db = torch.empty(b.shape, device=b.device, dtype=torch.float64) if s["grad_base"] else None
    for lo, hi in spans:
        c = b[lo:hi].double()
        g = torch.exp(scale * (q @ c.T) - lse[:, None]) * (w * scale)[:, None]
        dq += g @ c
        if db is not None:
            db[lo:hi] = g.T @ q
    if db is None:
        return loss, dq
    db.index_add_(0, t.clamp(min=0), -(w * scale)[:, None] * q)
    return loss, dq, db


def _exact_score(s):
    dim, out = s["dim"], []
    q = s["queries"].double()
    at = torch.arange(dim, device=q.device)
    for codes, scales, mins in zip(s["codes"].split(500_000), s["scales"].split(500_000),
                                   s["mins"].split(500_000) if s["mins"] is not None else (None,) * 10_000):
        c = (codes[:, at // 2].int() >> (4 * (at % 2)).int()) & 15
        g = at // s["group"]
        w = scales.double()[:, g] * (c - 8) if mins is None else scales.double()[:, g] * c + mins.double()[:, g]
        out.append(q @ w.T)
    return torch.cat(out, dim=1)


def _exact_pack(s):
    values, scales, lows = [], [], []
    for x in s["base"].split(250_000):
        value = torch.empty(x.shape, device=x.device, dtype=torch.float64)
        kept = []
        for a in range(0, s["dim"], s["group"]):
            part = x[:, a:a + s["group"]].float()
            low = part.amin(dim=1)
            # the scale is what 16 bits hold of the 32-bit quotient, by definition; all else in 64
            step = ((part.amax(dim=1) - low) / 15 if s["mins"] else part.abs().amax(dim=1) / 7).half()
            zero = low.half().double() if s["mins"] else torch.zeros_like(low).double()
            d = step.double()
            code = torch.round((part.double() - zero[:, None]) / torch.where(d > 0, d, 1.0)[:, None])
            code = torch.where(d[:, None] > 0, code.clamp(*((0, 15) if s["mins"] else (-8, 7))), 0.0)
            value[:, a:a + s["group"]] = code * d[:, None] + zero[:, None]
            kept.append((step, low.half()))
        values.append(value)
        scales.append(torch.stack([k[0] for k in kept], dim=1))
        lows.append(torch.stack([k[1] for k in kept], dim=1))
    got = torch.cat(values), torch.cat(scales).double()
    return got + (torch.cat(lows).double(),) if s["mins"] else got


def exact(case, seed):
    s = prepare(case, seed)
    return {"step": _exact_softmax, "loss": _exact_softmax, "score": _exact_score, "pack": _exact_pack}[s["op"]](s)
