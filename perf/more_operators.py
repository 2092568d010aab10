"""Both ends of a network over discrete things: the lookup of an embedding table and the losses behind a last dense layer, at the
sizes that this package's networks give them.

Things are species of atoms (about a hundred), or the entries of a larger vocabulary of structures.  Channel counts are those of the
networks run elsewhere in this repository: 112, 192, 204, 1280 channels of invariants, heads of 2048.

Kinds of cases:

  embedding  scale * weight[ids], forward alone or with the gradient of the table
  ce         the mean (or each row's) cross entropy of x w + bias and a class per row, forward alone or with all gradients; some rows have no class
  distill    the mean divergence of x w + bias from a teacher's `top` largest logits per row, forward alone or with all gradients; some
             entries, and some rows altogether, are missing

Plain forms are in 32 bits and round once at the end.  Losses are float32 whatever the type of x.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_IGNORE = -100


def listed():
    return [
        # the species of a small batch of molecules at inference: bound by its latency
        dict(name="emb_infer_small", kind="embedding", dtype="f32", n=64, v=100, d=192, skew=3, padding=False, train=False),
        # the atoms of a point cloud, training: a hundred rows share all gradients
        dict(name="emb_train_cloud", kind="embedding", dtype="f32", n=65536, v=100, d=112, skew=3, padding=False, train=True),
        # a ragged batch padded to one length, odd sizes
        dict(name="emb_train_ragged", kind="embedding", dtype="f16", n=14763, v=5003, d=204, skew=2, padding=True, train=True),
        # a large vocabulary, most of whose rows a step does not meet
        dict(name="emb_train_large", kind="embedding", dtype="bf16", n=32768, v=65536, d=2048, skew=2, padding=False, train=True),
        # one row is scored against a vocabulary: the weights are read once
        dict(name="ce_score_one", kind="ce", dtype="bf16", m=1, k=1280, n=32768, bias=True, wt=True, reduction="none", train=False),
        # the masked atoms of a small batch and their species, training: bound by its latency
        dict(name="ce_train_small", kind="ce", dtype="f32", m=64, k=192, n=100, bias=True, wt=False, reduction="mean", train=True),
        # a ragged batch, odd sizes, weights whose rows do not begin on 16-byte boundaries
        dict(name="ce_train_ragged", kind="ce", dtype="f16", m=777, k=204, n=1003, bias=True, wt=False, reduction="mean", train=True),
        # an ordinary step in the type that the products compute in
        dict(name="ce_train_mid", kind="ce", dtype="f32", m=1000, k=1280, n=8192, bias=True, wt=False, reduction="mean", train=True),
        # a large vocabulary whose matrix is the embedding's table
        dict(name="ce_train_large", kind="ce", dtype="bf16", m=4096, k=2048, n=65536, bias=False, wt=True, reduction="mean", train=True),
        # a validation batch against a teacher, odd sizes
        dict(name="distill_loss_ragged", kind="distill", dtype="bf16", m=333, k=131, n=5003, top=7, temperature=2.0, bias=True, wt=False, train=False),
        # an ordinary step with a teacher's few largest logits
        dict(name="distill_train_mid", kind="distill", dtype="bf16", m=1000, k=1280, n=8192, top=16, temperature=2.0, bias=True, wt=False, train=True),
        # a large vocabulary and many of the teacher's logits
        dict(name="distill_train_large", kind="distill", dtype="bf16", m=4096, k=1280, n=32768, top=64, temperature=1.0, bias=False, wt=True, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    kind = rng.choice(["embedding", "ce", "distill"])
    dtype = rng.choice(list(_TYPES))
    if kind == "embedding":
        return dict(kind=kind, dtype=dtype, n=_log(rng, 1, 1 << 20), v=_log(rng, 2, 262144), d=_log(rng, 8, 4096), skew=rng.choice([1, 2, 3]),
                    padding=rng.random() < 0.3, train=rng.random() < 0.7)
    c = dict(kind=kind, dtype=dtype, m=_log(rng, 1, 16384), k=_log(rng, 16, 4096), n=_log(rng, 16, 131072), bias=rng.random() < 0.6, wt=rng.random() < 0.5,
             train=rng.random() < 0.7)
    if kind == "ce":
        c["reduction"] = rng.choice(["mean", "mean", "sum", "none"])
    else:
        c["top"] = _log(rng, 1, min(64, c["n"]))
        c["temperature"] = rng.choice([1.0, 1.5, 2.0, 4.0])
    return c


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        a = most.setdefault(c["kind"], [0.0, 0.0])
        a[0], a[1] = max(a[0], w["bytes"]), max(a[1], w["flops"])
    while True:
        c = _drawn(rng)
        w = work(c)
        # no more than the largest listed case of the kind; float32 products cost several times as much as 16-bit ones
        dear = 8 if c["dtype"] == "f32" and c["kind"] != "embedding" else 1
        if w["bytes"] <= most[c["kind"]][0] and dear * w["flops"] <= most[c["kind"]][1]:
            return c


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[c["dtype"]]
    dev = "cuda"

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(t)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=dev, dtype=torch.float64)

    s = dict(case=c)
    if c["kind"] == "embedding":
        # a few entries are met often, most of them hardly ever
        s["ids"] = (uniform(c["n"]) ** c["skew"] * c["v"]).long().clamp(max=c["v"] - 1)
        s["padding_idx"] = 0 if c["padding"] else None
        if c["padding"]:
            s["ids"][uniform(c["n"]) < 0.2] = 0
        s["weight"] = normal(c["v"], c["d"])
        s["scale"] = math.sqrt(c["d"])
        s["gy"] = normal(c["n"], c["d"]) if c["train"] else None
        inputs = ["weight"]
    else:
        m, k, n = c["m"], c["k"], c["n"]
        s["x"] = normal(m, k)
        s["w"] = normal(n, k, scale=2 / math.sqrt(k)).t() if c["wt"] else normal(k, n, scale=2 / math.sqrt(k))
        s["bias"] = normal(n, scale=0.5) if c["bias"] else None
        missing = uniform(m) < 0.1
        missing[0] = False
        if c["kind"] == "ce":
            s["target"] = (uniform(m) ** 2 * n).long().clamp(max=n - 1)
            s["target"][missing] = _IGNORE
            shape = (m,) if c["reduction"] == "none" else ()
        else:
            top = c["top"]
            # distinct entries per row, the list ending early in some rows
            first = (uniform(m, 1) * n).long()
            s["ids"] = (first + torch.arange(top, device=dev) * (n // top)) % n
            live = (uniform(m, 1) * top).long() + top // 2 + 1
            s["ids"][(torch.arange(top, device=dev) >= live) | missing[:, None]] = -1
            s["logits"] = torch.sort(torch.randn(m, top, generator=g, device=dev) * 1.5 + 4, dim=1, descending=True)[0].to(t)
            shape = ()
        # float16 is trained with a scaled loss
        s["gy"] = torch.full(shape, 4096.0 if c["dtype"] == "f16" else 1.0, device=dev) if c["train"] else None
        if c["train"] and shape:
            s["gy"] = s["gy"] * (0.5 + uniform(*shape)).float() / m
        inputs = [q for q in ("x", "w", "bias") if s[q] is not None]
    s["inputs"] = inputs
    if c["train"]:
        for q in inputs:
            s[q].requires_grad_()
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------------


def _plain_embedding(s):
    c, t = s["case"], s["weight"].dtype
    y = (s["weight"][s["ids"]].float() * s["scale"]).to(t)
    if not c["train"]:
        return y
    gw = torch.zeros(c["v"], c["d"], device=y.device)
    gw.index_add_(0, s["ids"], s["gy"].float())
    if s["padding_idx"] is not None:
        gw[s["padding_idx"]] = 0
    return [y, (gw * s["scale"]).to(t)]


def _logits(s, temperature):
    z = s["x"].float() @ s["w"].float()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    return z / temperature


def _plain_gradients(s, dz):
    t = s["x"].dtype
    out = [(dz @ s["w"].float().t()).to(t), (s["x"].float().t() @ dz).to(t)]
    if s["bias"] is not None:
        out.append(dz.sum(0).to(t))
    return out


def _softmax(z):
    top = z.max(1, keepdim=True)[0]
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    return e / total, (top + torch.log(total))[:, 0]


def _plain_ce(s):
    c = s["case"]
    z = _logits(s, 1.0)
    live = s["target"] != _IGNORE
    t = torch.where(live, s["target"], 0)[:, None]
    p, lse = _softmax(z)
    loss = (lse - z.gather(1, t)[:, 0]) * live
    count = live.sum().float() if c["reduction"] == "mean" else 1.0
    loss = loss if c["reduction"] == "none" else loss.double().sum().float() / count
    if not c["train"]:
        return loss
    p.scatter_add_(1, t, torch.full_like(t, -1.0, dtype=p.dtype))
    return [loss, *_plain_gradients(s, p * (s["gy"] / count * live)[:, None])]


def _plain_distill(s):
    c, temp = s["case"], s["case"]["temperature"]
    z = _logits(s, temp)
    entry = s["ids"] >= 0
    live = entry.any(1)
    ids = torch.where(entry, s["ids"], 0)
    t = torch.where(entry, s["logits"].float() / temp, -1e30)
    q = torch.exp(t - t.max(1, keepdim=True)[0]) * entry
    q = q / q.sum(1, keepdim=True).clamp(min=1e-30)
    p, lse = _softmax(z)
    log_q = torch.log(torch.where(q > 0, q, 1.0))
    loss = (q * (log_q - z.gather(1, ids) + lse[:, None])).sum(1)
    count = live.sum().float().clamp(min=1)
    loss = (loss * live).double().sum().float() / count * temp ** 2
    if not c["train"]:
        return loss
    p.scatter_add_(1, ids, -q)
    return [loss, *_plain_gradients(s, p * (s["gy"] / count * temp * live)[:, None])]


# ---- one pass ----------------------------------------------------------------------------------------------------------------


def run(s):
    c = s["case"]
    if not own:
        with torch.no_grad():
            return {"embedding": _plain_embedding, "ce": _plain_ce, "distill": _plain_distill}[c["kind"]](s)
    import gelib_b200 as gelib
    if c["kind"] == "embedding":
        y = gelib.embedding(s["ids"], s["weight"], scale=s["scale"], padding_idx=s["padding_idx"])
    elif c["kind"] == "ce":
        y = gelib.linear_cross_entropy(s["x"], s["w"], s["target"], s["bias"], ignore_index=_IGNORE, reduction=c["reduction"])
    else:
        y = gelib.linear_distillation(s["x"], s["w"], s["ids"], s["logits"], s["bias"], temperature=c["temperature"])
    if not c["train"]:
        return y
    return [y, *torch.autograd.grad(y, [s[q] for q in s["inputs"]], s["gy"])]


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "embedding":
        met = c["v"] * (1 - math.exp(-c["n"] / c["v"]))   # rows that are read, at the most
        e = (met + c["n"]) * c["d"]
        if c["train"]:
            e += (c["n"] + c["v"]) * c["d"]
        return {"bytes": size * e + 8 * c["n"] * (2 if c["train"] else 1), "flops": float(c["n"] * c["d"] * (2 if c["train"] else 1))}
    m, k, n = c["m"], c["k"], c["n"]
    e = (m * k + k * n + n * c["bias"]) * (2 if c["train"] else 1)
    rest = 8 * m if c["kind"] == "ce" else (8 + size) * m * c["top"]
    return {"bytes": size * e + rest + 4 * m, "flops": 2.0 * m * k * n * (3 if c["train"] else 1)}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------


def exact(case, seed):
    s, c = prepare(case, seed), case
    ins = [s[q].detach().double().requires_grad_(c["train"]) for q in s["inputs"]]
    v = dict(zip(s["inputs"], ins))
    gy = s["gy"].double() if c["train"] else None
    if c["kind"] == "embedding":
        y = s["scale"] * v["weight"].detach()[s["ids"]]
        if not c["train"]:
            return y
        # rows of the gradient as differences of running sums over the sorted entries would lose digits: added one by one in 64 bits
        gw = torch.zeros_like(ins[0]).detach().scatter_add_(0, s["ids"][:, None].expand(-1, c["d"]), gy * s["scale"])
        if c["padding"]:
            gw[s["padding_idx"]].zero_()
        return [y, gw]
    z = torch.matmul(v["x"], v["w"])
    z = z + v["bias"] if c["bias"] else z
    if c["kind"] == "ce":
        rows = (s["target"] != _IGNORE).nonzero()[:, 0]
        of_live = torch.logsumexp(z[rows], 1) - z[rows, s["target"][rows]]
        loss = torch.zeros(c["m"], dtype=torch.float64, device=z.device).index_put((rows,), of_live)
        y = {"none": lambda: loss, "sum": lambda: of_live.sum(), "mean": lambda: of_live.mean()}[c["reduction"]]()
    else:
        temp = c["temperature"]
        rows, cols = (s["ids"] >= 0).nonzero(as_tuple=True)
        t = torch.full(s["ids"].shape, -math.inf, dtype=torch.float64, device=z.device)
        t[rows, cols] = s["logits"].double()[rows, cols] / temp
        log_q = torch.log_softmax(t, 1)[rows, cols]
        log_p = z[rows, s["ids"][rows, cols]] / temp - torch.logsumexp(z / temp, 1)[rows]
        y = temp ** 2 * (log_q.exp() * (log_q - log_p)).sum() / rows.unique().numel()
    if not c["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, ins, gy)]
