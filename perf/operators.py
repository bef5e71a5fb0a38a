"""Timed cases of the token operators: embedding lookup with its gradient, block norms with gate and residual scale, distillation from
a teacher's top logits.  `run` computes them in plain torch operations, or (`own`) through omnihd_amd.ops."""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


sys.path.insert(1, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omnihd-scenes_amd"))


def listed():
    return [
        # serving: one decoding step of 64 sequences looks its tokens up
        dict(name="embed serve", op="embed", tokens=64, vocab=32000, dim=4096, table="bf16", out="bf16", ids="i64", pad=False, scale=1.0, train=False),
        # an fp32 parameter under mixed precision, a small batch, tokens of one frequent-word law, with padding
        dict(name="embed train fp32 table", op="embed", tokens=8192, vocab=32000, dim=1024, table="f32", out="bf16", ids="i64", pad=True, scale=32.0, train=True),
        # a large batch: the gradient's sums and the zero rows of the table both count
        dict(name="embed train large", op="embed", tokens=65536, vocab=100000, dim=2048, table="bf16", out="bf16", ids="i64", pad=True, scale=1.0, train=True),
        # rows that no vector load fits
        dict(name="embed train odd", op="embed", tokens=5003, vocab=20011, dim=333, table="f32", out="f32", ids="i32", pad=False, scale=0.5, train=True),
        # serving: eight sequences, one token each, between two blocks
        dict(name="join serve", op="join", batch=8, length=1, dim=4096, act="bf16", stream="bf16", weights="bf16", gate="channel", post=True, next=True, scale=1.0, train=False),
        # a training step between two blocks of a wide model
        dict(name="join train", op="join", batch=4, length=4096, dim=4096, act="bf16", stream="bf16", weights="f32", gate="channel", post=True, next=True, scale=0.9, train=True),
        # odd lengths and width, an fp32 residual stream, one gate per sample
        dict(name="join train odd", op="join", batch=3, length=1037, dim=1021, act="bf16", stream="f32", weights="f32", gate="sample", post=True, next=True, scale=1.0, train=True),
        # the first norm over the cells of the 160 x 240 BEV grid at 256 channels, two samples
        dict(name="norm train bev", op="norm", batch=2, length=38400, dim=256, act="f16", stream="f16", weights="f32", train=True),
        # a few rows against a vocabulary: what one launch costs
        dict(name="distill small", op="distill", rows=32, vocab=32000, top=20, logits="bf16", teacher="f32", ids="i64", temperature=2.0, masked=0.0, holes=0.0, pitch=0, reduction="mean", train=True),
        # the occupancy head: 240 x 160 x 16 voxels, 12 classes, the teacher's best four
        dict(name="distill occupancy", op="distill", rows=614400, vocab=12, top=4, logits="f32", teacher="f32", ids="i32", temperature=1.0, masked=0.1, holes=0.0, pitch=0, reduction="mean", train=True),
        # a training batch against a large vocabulary
        dict(name="distill large", op="distill", rows=4096, vocab=131072, top=64, logits="bf16", teacher="bf16", ids="i64", temperature=1.0, masked=0.0, holes=0.0, pitch=0, reduction="mean", train=True),
        # odd vocabulary (rows start at any address), masked rows, slots that the teacher left empty
        dict(name="distill odd", op="distill", rows=1021, vocab=50021, top=33, logits="f16", teacher="f32", ids="i32", temperature=1.5, masked=0.25, holes=0.2, pitch=0, reduction="sum", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "join", "join", "norm", "distill", "distill"])
    largest = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    while True:
        train = rng.random() < 0.75
        act, other = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32"), ("f16", "f32")])
        if op == "embed":
            dim = _log(rng, 24, 6000)
            dim = dim if rng.random() < 0.3 else -(-dim // 8) * 8
            c = dict(op=op, tokens=_log(rng, 1, 131072), vocab=_log(rng, 500, 200000), dim=dim, table=other, out=act,
                     ids=rng.choice(["i64", "i32"]), pad=rng.random() < 0.5, scale=round(rng.uniform(0.2, 40.0), 3), train=train)
        elif op in ("join", "norm"):
            dim = _log(rng, 40, 12000)
            dim = dim if rng.random() < 0.3 else -(-dim // 8) * 8
            c = dict(op=op, batch=rng.randint(1, 9), length=_log(rng, 1, 20000), dim=dim, act=act, stream=other, weights=rng.choice(["f32", act]), train=train)
            if op == "join":
                post = rng.random() < 0.8
                c.update(gate=rng.choice(["none", "channel", "sample", "token", "full"]), post=post, next=not post or rng.random() < 0.8,
                         scale=round(rng.uniform(0.3, 1.5), 3))
        else:
            vocab = _log(rng, 5, 262144)
            c = dict(op=op, rows=_log(rng, 1, 65536 if vocab > 100 else 1000000), vocab=vocab, top=min(_log(rng, 1, 200), vocab // 2), logits=act, teacher=rng.choice(["f32", act]),
                     ids=rng.choice(["i64", "i32"]), temperature=round(rng.uniform(0.5, 4.0), 3), masked=rng.choice([0.0, 0.3]), holes=rng.choice([0.0, 0.2]),
                     pitch=rng.choice([0, 0, 8, 13]), reduction=rng.choice(["mean", "sum", "none"]), train=train)
        if work(c)["bytes"] <= largest:
            return c


def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(scale)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    c = case
    s = {"case": c}
    if c["op"] == "embed":
        n, V, D = c["tokens"], c["vocab"], c["dim"]
        u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        rank = torch.exp(u * math.log(V)).long().clamp_(1, V) - 1          # frequency of the r-th word ~ 1 / r
        s["ids"] = (rank * 7919 % V).to(torch.int64 if c["ids"] == "i64" else torch.int32)
        s["pad"] = 3 if c["pad"] else None
        if c["pad"]:                                                        # the ends of a batch of ragged sequences
            s["ids"][torch.rand(n, generator=gen, device="cuda") < 0.1] = 3
        s["table"] = _normal(gen, V, D, dtype=TYPES[c["table"]], scale=0.02).requires_grad_(c["train"])
        if c["train"]:
            s["g"] = _normal(gen, n, D, dtype=TYPES[c["out"]])
    elif c["op"] in ("join", "norm"):
        B, L, D = c["batch"], c["length"], c["dim"]
        act, stream, wt = TYPES[c["act"]], TYPES[c["stream"]], TYPES[c["weights"]]
        weight = lambda: (1 + _normal(gen, D, scale=0.1)).to(wt).requires_grad_(c["train"])  # noqa: E731
        s["x"] = _normal(gen, B, L, D, dtype=stream, scale=1.5).requires_grad_(c["train"])
        if c["op"] == "norm":
            s["next"] = weight()
        else:
            s["y"] = _normal(gen, B, L, D, dtype=act, scale=3.0).requires_grad_(c["train"])
            s["post"] = weight() if c["post"] else None
            s["next"] = weight() if c["next"] else None
            shape = {"none": None, "channel": (D,), "sample": (B, 1, D), "token": (B, L, 1), "full": (B, L, D)}[c["gate"]]
            s["gate"] = None if shape is None else _normal(gen, *shape, scale=0.5).to(act if c["gate"] == "full" else wt).requires_grad_(c["train"])
            if c["train"]:
                s["gx"] = _normal(gen, B, L, D, dtype=stream)
        if c["train"]:
            s["gh"] = _normal(gen, B, L, D, dtype=act)
    else:
        N, V, K = c["rows"], c["vocab"], c["top"]
        start = torch.randint(0, V, (N, 1), generator=gen, device="cuda")
        step = torch.randint(1, V // K + 1, (N, 1), generator=gen, device="cuda")
        ids = (start + step * torch.arange(K, device="cuda")) % V           # K different entries
        t = _normal(gen, N, K, scale=1.5).sort(dim=1, descending=True)[0] + 6.0
        z = _normal(gen, N, V + c["pitch"], dtype=TYPES[c["logits"]], scale=1.5)
        z = z[:, :V]
        z.scatter_add_(1, ids, (t * 0.8).to(z.dtype))                       # a student on its way to the teacher
        if c["holes"]:
            ids = torch.where(torch.rand(N, K, generator=gen, device="cuda") < c["holes"], torch.full_like(ids, -1), ids)
        s["ids"] = ids.to(torch.int64 if c["ids"] == "i64" else torch.int32)
        s["t"] = t.to(TYPES[c["teacher"]])
        s["z"] = z.detach().requires_grad_(c["train"])
        s["w"] = (torch.rand(N, generator=gen, device="cuda") >= c["masked"]).float() if c["masked"] else None
        if c["reduction"] == "none" and c["train"]:
            s["g"] = torch.rand(N, generator=gen, device="cuda")
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from omnihd_amd import ops
    c = s["case"]
    if c["op"] == "embed":
        out = ops.token_embedding(s["ids"], s["table"], scale=c["scale"], padding_idx=s["pad"], out_dtype=TYPES[c["out"]])
        if not c["train"]:
            return {"out": out}
        return {"out": out.detach(), "table": torch.autograd.grad(out, s["table"], s["g"])[0]}
    if c["op"] == "norm":
        h = ops.block_norm(s["x"], s["next"], eps=1e-6, out_dtype=TYPES[c["act"]])
        if not c["train"]:
            return {"h": h}
        gx, gw = torch.autograd.grad(h, (s["x"], s["next"]), s["gh"])
        return {"h": h.detach(), "gx": gx, "next": gw}
    if c["op"] == "join":
        got = ops.block_join(s["x"], s["y"], post_weight=s["post"], gate=s["gate"], residual_scale=c["scale"], next_weight=s["next"], eps=1e-6)
        x1, h = got if c["next"] else (got, None)
        outs = {"x": x1.detach()}
        if c["next"]:
            outs["h"] = h.detach()
        if c["train"]:
            leaves = {k: s[k] for k in ("x", "y", "post", "gate", "next") if s[k] is not None}
            grads = torch.autograd.grad((x1, h) if c["next"] else (x1,), list(leaves.values()), (s["gx"], s["gh"]) if c["next"] else (s["gx"],))
            outs.update({"g_" + k: g for k, g in zip(leaves, grads)})
        return outs
    loss = ops.topk_distill_loss(s["z"], s["t"], s["ids"], temperature=c["temperature"], row_weight=s["w"], reduction=c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    return {"loss": loss.detach(), "z": torch.autograd.grad(loss, s["z"], s.get("g"))[0]}


def _run_plain(s):
    c = s["case"]
    with torch.no_grad():
        if c["op"] == "embed":
            ids = s["ids"].long()
            outs = {"out": (s["table"][ids].float() * c["scale"]).to(TYPES[c["out"]])}
            if c["train"]:
                acc = torch.zeros(c["vocab"], c["dim"], device="cuda").index_add_(0, ids, s["g"].float())
                if s["pad"] is not None:
                    acc[s["pad"]] = 0
                outs["table"] = acc.mul_(c["scale"]).to(TYPES[c["table"]])
            return outs
        if c["op"] in ("join", "norm"):
            return _plain_block(s)
        return _plain_distill(s)


def _plain_block(s):
    c = s["case"]
    eps, act, stream, wt = 1e-6, TYPES[c["act"]], TYPES[c["stream"]], TYPES[c["weights"]]
    join = c["op"] == "join"
    r = c["scale"] if join else 1.0
    x = s["x"].float()
    gate = post = 1.0
    outs = {}
    if join:
        n = s["y"].float()
        if s["post"] is not None:
            ry = torch.rsqrt(n.square().mean(-1, keepdim=True) + eps)
            n, post = n * ry, s["post"].float()
        if s["gate"] is not None:
            gate = s["gate"].float()
        x = r * x + gate * (n * post)
        outs["x"] = x.to(stream)
    if s["next"] is not None:
        rx = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
        u = s["next"].float()
        outs["h"] = (x * rx * u).to(act)
    if not c["train"]:
        return outs
    t = s["gx"].float() if join else 0.0
    pre = "g_" if join else ""
    if s["next"] is not None:
        gh, xh = s["gh"].float(), x * rx
        a = gh * u
        t = t + rx * (a - xh * (a * xh).mean(-1, keepdim=True))
        g_next = (gh * xh).sum((0, 1)).to(wt)
    if not join:
        outs["gx"], outs["next"] = t.to(stream), g_next
        return outs
    outs[pre + "x"] = (r * t).to(stream)
    m = t * gate * post
    if s["post"] is not None:
        outs[pre + "y"] = (ry * (m - n * (m * n).mean(-1, keepdim=True))).to(act)
        outs[pre + "post"] = (t * gate * n).sum((0, 1)).to(wt)
    else:
        outs[pre + "y"] = m.to(act)
    if s["gate"] is not None:
        over = {"channel": (0, 1), "sample": (1,), "token": (2,), "full": ()}[c["gate"]]
        d = t * n * post
        d = d.sum(over, keepdim=True).reshape(s["gate"].shape) if over else d
        outs[pre + "gate"] = d.to(s["gate"].dtype)
    if s["next"] is not None:
        outs[pre + "next"] = g_next
    return outs


def _plain_distill(s):
    c, T = s["case"], s["case"]["temperature"]
    z = s["z"].float() / T
    z = z - z.amax(1, keepdim=True)
    lnq = z - torch.exp(z).sum(1, keepdim=True).log()
    ids = s["ids"].long()
    filled = ids >= 0
    ids = ids.clamp_min(0)
    t = torch.where(filled, s["t"].float() / T, torch.full_like(s["t"], -math.inf, dtype=torch.float32))
    top = t.amax(1, keepdim=True)
    some = torch.isfinite(top)
    e = torch.where(filled, torch.exp(t - torch.where(some, top, torch.zeros_like(top))), torch.zeros_like(t))
    mass = e.sum(1, keepdim=True)
    p = torch.where(some, e / mass, torch.zeros_like(e))
    lnp = torch.where(p > 0, p.clamp_min(1e-45).log(), torch.zeros_like(p))
    row = T * T * (p * (lnp - torch.where(filled, lnq.gather(1, ids), torch.zeros_like(p)))).sum(1)
    w = torch.ones_like(row) if s["w"] is None else s["w"]
    row = row * w
    loss = row.sum(dtype=torch.float64).float() if c["reduction"] != "none" else row
    k = w * T
    if c["reduction"] == "mean":
        loss, k = loss / c["rows"], k / c["rows"]
    if not c["train"]:
        return {"loss": loss}
    if c["reduction"] == "none":
        k = k * s["g"]
    q = torch.exp(lnq) * some
    q.scatter_add_(1, ids, -p)
    return {"loss": loss, "z": (q * k[:, None]).to(s["z"].dtype)}


def work(case):
    c = case
    if c["op"] == "embed":
        n, V, D, t, o = c["tokens"], c["vocab"], c["dim"], SIZE[c["table"]], SIZE[c["out"]]
        r = torch.arange(1, V + 1, dtype=torch.float64)
        seen = float((-torch.expm1(n * torch.log1p(-torch.log1p(1 / r) / math.log(V + 1)))).sum())   # distinct rows of n tokens
        b = n * (8 if c["ids"] == "i64" else 4) + seen * D * t + n * D * o
        return {"bytes": b + (n * D * o + V * D * t if c["train"] else 0), "flops": n * D * (2 if c["train"] else 1)}
    if c["op"] in ("join", "norm"):
        e, a, x = c["batch"] * c["length"] * c["dim"], SIZE[c["act"]], SIZE[c["stream"]]
        if c["op"] == "norm":
            return {"bytes": e * ((x + a) + (a + x if c["train"] else 0)), "flops": e * (4 + (10 if c["train"] else 0))}
        full = a * e if c["gate"] == "full" else 0
        b = e * (2 * x + a + (a if c["next"] else 0)) + full
        if c["train"]:
            b += e * (2 * x + a + (a if c["next"] else 0)) + full
        return {"bytes": b, "flops": e * (10 + (20 if c["train"] else 0))}
    N, V, K, z = c["rows"], c["vocab"], c["top"], SIZE[c["logits"]]
    b = N * V * z * (2 if c["train"] else 1) + N * K * (SIZE[c["teacher"]] + (8 if c["ids"] == "i64" else 4))
    return {"bytes": b, "flops": N * V * (8 if c["train"] else 4)}


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    d = lambda k: None if s.get(k) is None else s[k].detach().double()  # noqa: E731
    if c["op"] == "embed":
        ids = s["ids"].long()
        outs = {"out": torch.index_select(d("table"), 0, ids) * c["scale"]}
        if c["train"]:
            keep = torch.ones_like(ids, dtype=torch.bool) if s["pad"] is None else ids != s["pad"]
            outs["table"] = torch.zeros(c["vocab"], c["dim"], dtype=torch.float64, device="cuda").index_put_((ids[keep],), d("g")[keep] * c["scale"], accumulate=True)
        return outs
    if c["op"] in ("join", "norm"):
        names = [k for k in ("x", "y", "post", "gate", "next") if s.get(k) is not None]
        v = {k: d(k).requires_grad_(c["train"]) for k in names}
        unit = lambda a: a / torch.sqrt(a.pow(2).sum(-1, keepdim=True) / c["dim"] + 1e-6)  # noqa: E731
        x = v["x"]
        outs = {}
        if c["op"] == "join":
            n = unit(v["y"]) * v["post"] if "post" in v else v["y"]
            x = x * c["scale"] + (n * v["gate"] if "gate" in v else n)
            outs["x"] = x
        if "next" in v:
            outs["h"] = unit(x) * v["next"]
        if not c["train"]:
            return outs
        ups = [d({"x": "gx", "h": "gh"}[k]) for k in outs]
        grads = dict(zip(names, torch.autograd.grad(list(outs.values()), list(v.values()), ups)))
        outs = {k: o.detach() for k, o in outs.items()}
        if c["op"] == "norm":
            return {**outs, "gx": grads["x"], "next": grads["next"]}
        return {**outs, **{"g_" + k: g for k, g in grads.items()}}
    T, N, V = c["temperature"], c["rows"], c["vocab"]
    rows, dz = torch.zeros(N, dtype=torch.float64, device="cuda"), torch.zeros(N, V, dtype=torch.float64, device="cuda") if c["train"] else None
    w = torch.ones(N, dtype=torch.float64, device="cuda") if s["w"] is None else d("w")
    k = w / N if c["reduction"] == "mean" else w * s["g"].double() if "g" in s else w
    size = max(1, (1 << 27) // V)
    for lo in range(0, N, size):
        at = slice(lo, min(N, lo + size))
        ids = s["ids"][at].long()
        hole = ids < 0
        lse = torch.logsumexp(s["z"][at].detach().double() / T, 1, keepdim=True)
        t = (s["t"][at].double() / T).masked_fill(hole, -math.inf)
        p = torch.softmax(t, 1).masked_fill(hole.all(1, keepdim=True), 0.0)
        zk = s["z"][at].detach().double().gather(1, ids.clamp_min(0)) / T
        rows[at] = T * T * (torch.special.xlogy(p, p) - p * (zk - lse)).sum(1) * w[at]
        if c["train"]:
            q = torch.exp(s["z"][at].detach().double() / T - lse).masked_fill_(hole.all(1, keepdim=True), 0.0)
            dz[at] = q.scatter_add_(1, ids.clamp_min(0), -p).mul_(T * k[at, None])
    loss = rows if c["reduction"] == "none" else rows.sum() / (N if c["reduction"] == "mean" else 1)
    return {"loss": loss, "z": dz} if c["train"] else {"loss": loss}
