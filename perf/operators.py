"""The readout of an equivariant network and its training step: group norm with an activation, the dense layer with its
epilogue, and the AdamW step, at the sizes that this package's networks give them.

The invariants of a network are the l=0 parts of its products, (batch, [grid], channels) with the channels last.  Their channel
counts follow from the products that are run elsewhere in this repository: 8 channels up to l=2 give 192, the ragged layer
12/9/7/5 x 10/7/3 gives 204, 16 channels up to l=4 give 1280, 1 x 16 channels up to l=6 give 112, 32 channels up to l=6 give
7168, diagonal products of 128 channels up to l=8 give 1152.

Kinds of cases:

  norm    group_norm of (b, s, n) with an activation, forward alone or with all gradients
  linear  act(x w + bias) + residual, forward alone or with all gradients
  adamw   one step over the weights of a network: `layers` layers of complex mixing matrices (l <= maxl, n channels), then a head of
          dense matrices n0 -> hidden -> ... -> 1 with biases, norm weights and norm biases; states in 32 or in 8 bits; the head in
          float32, or in bfloat16 with float32 master copies

Plain forms are in 32 bits and round once at the end.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BLOCK = 256  # elements that share a scale, where states are held in 8 bits


def listed():
    return [
        # one small molecule batch at inference: a call made from a loop, bound by its latency
        dict(name="norm_infer_small", kind="norm", dtype="f32", b=64, s=1, n=192, groups=8, act="silu", train=False),
        # an array of atoms per sample, odd channel counts (17 a group), training
        dict(name="norm_train_ragged", kind="norm", dtype="bf16", b=777, s=19, n=204, groups=12, act="gelu_tanh", train=True),
        # the invariants of the headline product, a row per sample, training
        dict(name="norm_train_wide", kind="norm", dtype="bf16", b=4096, s=1, n=7168, groups=32, act="silu", train=True),
        # point clouds: one sample's statistics run over all its points
        dict(name="norm_train_cloud", kind="norm", dtype="f32", b=4, s=65536, n=112, groups=7, act="silu", train=True),
        # one object at a time: a single row through a layer
        dict(name="linear_infer_one", kind="linear", dtype="bf16", m=1, k=1280, n=1280, act="silu", bias=True, residual=True, wt=False, train=False),
        # the ragged layer on its ragged batch, training, weights kept as (out, in)
        dict(name="linear_train_ragged", kind="linear", dtype="bf16", m=777, k=204, n=131, act="gelu_tanh", bias=True, residual=False, wt=True, train=True),
        # the usual layer, in the type that the products compute in
        dict(name="linear_train_mid", kind="linear", dtype="f32", m=1000, k=1280, n=512, act="silu", bias=True, residual=False, wt=False, train=True),
        # a residual layer over the points of a cloud: many rows, few channels
        dict(name="linear_train_cloud", kind="linear", dtype="f32", m=65536, k=112, n=112, act="silu", bias=True, residual=True, wt=False, train=True),
        # the first layer after the headline product
        dict(name="linear_train_wide", kind="linear", dtype="bf16", m=4096, k=7168, n=2048, act="silu", bias=True, residual=False, wt=False, train=True),
        # the weights of a small network: two dozen tensors, most of them tiny
        dict(name="adamw_small", kind="adamw", bits=32, low=False, layers=3, maxl=2, n=8, n0=192, hidden=64, depth=2),
        # the weights behind the headline product: a few large matrices among small ones
        dict(name="adamw_large", kind="adamw", bits=32, low=False, layers=4, maxl=6, n=32, n0=7168, hidden=4096, depth=2),
        # the same with states in 8 bits, the head in bfloat16
        dict(name="adamw_large_8bit", kind="adamw", bits=8, low=True, layers=4, maxl=6, n=32, n0=7168, hidden=4096, depth=2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    kind = rng.choice(["norm", "linear", "adamw"])
    act = rng.choice(["none", "relu", "silu", "gelu_tanh"])
    if kind == "norm":
        groups = rng.choice([1, 2, 4, 7, 8, 12, 16, 32])
        return dict(kind=kind, dtype=rng.choice(list(_TYPES)), b=_log(rng, 1, 4096), s=rng.choice([1, _log(rng, 1, 65536)]),
                    n=groups * _log(rng, 1, 224), groups=groups, act=act, train=rng.random() < 0.6)
    if kind == "linear":
        return dict(kind=kind, dtype=rng.choice(list(_TYPES)), m=_log(rng, 1, 65536), k=_log(rng, 16, 7168), n=_log(rng, 8, 2048), act=act,
                    bias=rng.random() < 0.7, residual=rng.random() < 0.5, wt=rng.random() < 0.5, train=rng.random() < 0.6)
    return dict(kind=kind, bits=rng.choice([32, 8]), low=rng.random() < 0.5, layers=rng.randint(1, 8), maxl=rng.randint(0, 6), n=_log(rng, 4, 64),
                n0=_log(rng, 16, 7168), hidden=_log(rng, 16, 4096), depth=rng.randint(1, 4))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        a = most.setdefault(c["kind"], [0.0, 0.0])
        a[0], a[1] = max(a[0], w["bytes"]), max(a[1], w["flops"])
    while True:
        c = _drawn(rng)
        w = work(c)
        # a few microseconds of work at the least, no more than the largest listed case of the kind
        if w["bytes"] <= most[c["kind"]][0] and w["flops"] <= most[c["kind"]][1] and (c["kind"] != "norm" or c["b"] * c["s"] * c["n"] >= 256):
            return c


# ---- the weights of a network ------------------------------------------------------------------------------------------------


def _shapes(c):
    """(shape, complex) of the mixing matrices, and of the head's tensors."""
    mixing = [((c["n"], c["n"]), True)] * (c["layers"] * (c["maxl"] + 1))
    head, width = [((c["n0"],), False)] * 2, c["n0"]
    for _ in range(c["depth"]):
        head += [((width, c["hidden"]), False), ((c["hidden"],), False)]
        width = c["hidden"]
    return mixing, head + [((width, 1), False), ((1,), False)]


def _floats(shape, cplx):
    return math.prod(shape) * (2 if cplx else 1)


def _padded(shapes):
    return sum(-(-_floats(*s) // _BLOCK) * _BLOCK for s in shapes)


def _views(flat, shapes, cplx=True, each=1):
    """The tensors of a network as views of one buffer in which each begins at a multiple of 256 elements; `each` elements share one
    entry of the buffer, and cplx=False keeps complex tensors as pairs of numbers in one dimension."""
    got, at = [], 0
    for shape, is_c in shapes:
        n = _floats(shape, is_c)
        if each > 1:
            got.append(flat[at // each:(at + n + each - 1) // each])
        elif not cplx:
            got.append(flat[at:at + n])
        elif is_c:
            got.append(torch.view_as_complex(flat[at:at + n].view(-1, 2)).view(shape))
        else:
            got.append(flat[at:at + n].view(shape))
        at += -(-n // _BLOCK) * _BLOCK
    return got


def _to_codes(x):
    """x, in blocks of 256, as e4m3 codes and a power of two per block that brings the largest value into [128, 256)."""
    b = x.view(-1, _BLOCK)
    scale = torch.exp2((torch.floor(torch.log2(b.abs().amax(1))) - 7).clamp(min=-100))
    return (b / scale[:, None]).to(torch.float8_e4m3fn).view(-1), scale


def _prepare_adamw(case, g):
    mixing, head = _shapes(case)
    shapes = mixing + head
    na, nb = _padded(mixing), _padded(head)
    n = na + nb
    dev = "cuda"
    real = torch.zeros(n, dtype=torch.bool, device=dev)
    for v in _views(real, shapes, cplx=False):
        v.fill_(True)

    def normal(scale):
        return torch.randn(n, generator=g, device=dev) * scale * real

    # gradients whose size differs from tensor to tensor and from weight to weight, as those of a network do
    size = torch.exp(torch.randn(n // _BLOCK, generator=g, device=dev)).repeat_interleave(_BLOCK) * 1e-2
    grad = normal(1.0) * size
    m = 0.5 * grad + normal(0.3) * size
    r = (size * (0.3 + torch.rand(n, generator=g, device=dev))) * real
    p = normal(0.2)
    s = dict(case=case, na=na, p=p, grad=grad, step=1000, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, seed=int(case["n0"]) + 17)
    s["grads"] = _views(grad[:na], mixing) + _views(grad[na:], head)
    s["params"] = _views(p[:na], mixing) + _views(p[na:], head)
    if case["low"]:  # the head in bfloat16; p keeps its master copies
        s["low_p"] = p[na:].to(torch.bfloat16)
        s["low_grad"] = grad[na:].to(torch.bfloat16)
        s["master"] = [None] * len(mixing) + s["params"][len(mixing):]
        s["params"] = s["params"][:len(mixing)] + _views(s["low_p"], head)
        s["grads"] = s["grads"][:len(mixing)] + _views(s["low_grad"], head)
    else:
        s["master"] = None
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _to_codes(m)
        s["v"], s["v_scale"] = _to_codes(r)
        s["exp_avg_scale"], s["exp_avg_sq_scale"] = _views(s["m_scale"], shapes, each=_BLOCK), _views(s["v_scale"], shapes, each=_BLOCK)
    else:
        s["m"], s["v"] = m, r * r
        s["exp_avg_scale"] = s["exp_avg_sq_scale"] = None
    s["exp_avg"], s["exp_avg_sq"] = _views(s["m"], shapes, cplx=False), _views(s["v"], shapes, cplx=False)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "adamw":
        return _prepare_adamw(case, g)
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(t)

    train, n = case["train"], case["n"]
    if case["kind"] == "norm":
        s = dict(x=normal(case["b"], case["s"], n, scale=1.5, mean=0.3), weight=normal(n, scale=0.2, mean=1.0), bias=normal(n, scale=0.2))
        s["gy"] = normal(case["b"], case["s"], n) if train else None
        inputs = ["x", "weight", "bias"]
    else:
        m, k = case["m"], case["k"]
        w = normal(n, k, scale=1 / math.sqrt(k)).t() if case["wt"] else normal(k, n, scale=1 / math.sqrt(k))
        s = dict(x=normal(m, k), w=w, bias=normal(n, scale=0.3) if case["bias"] else None, residual=normal(m, n) if case["residual"] else None)
        s["gy"] = normal(m, n) if train else None
        inputs = [q for q in ("x", "w", "bias", "residual") if s[q] is not None]
    s.update(case=case, inputs=inputs)
    if train:
        for q in inputs:
            s[q].requires_grad_()
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------------


def _sigmoid(z):
    return 1 / (1 + torch.exp(-z))


def _act(z, act):
    """The activation and its derivative."""
    if act == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if act == "silu":
        q = _sigmoid(z)
        return z * q, q * (1 + z * (1 - q))
    if act == "gelu_tanh":  # 0.5 (1 + tanh u) is the logistic function of 2u
        c = 2 * math.sqrt(2 / math.pi)
        q = _sigmoid(c * (z + 0.044715 * z * z * z))
        return z * q, q + z * q * (1 - q) * c * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _plain_norm(s):
    c, t = s["case"], s["x"].dtype
    x, w, b = (s[q].float() for q in ("x", "weight", "bias"))
    xg = x.view(c["b"], c["s"], c["groups"], -1)
    d = xg - xg.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    xh = (d * rstd).view(x.shape)
    y, dy = _act(xh * w + b, c["act"])
    if not c["train"]:
        return y.to(t)
    gz = s["gy"].float() * dy
    gh = (gz * w).view(xg.shape)
    hg = xh.view(xg.shape)
    gx = rstd * (gh - gh.mean((1, 3), keepdim=True) - hg * (gh * hg).mean((1, 3), keepdim=True))
    return y.to(t), gx.view(x.shape).to(t), (gz * xh).sum((0, 1)).to(t), gz.sum((0, 1)).to(t)


def _plain_linear(s):
    c, t = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, dy = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not c["train"]:
        return y.to(t)
    gz = s["gy"].float() * dy
    out = [y.to(t), (gz @ w.t()).to(t), (x.t() @ gz).to(t)]
    if s["bias"] is not None:
        out.append(gz.sum(0).to(t))
    if s["residual"] is not None:
        out.append(s["gy"])
    return out


def _random_bits(seed, n, device):
    """32 bits for each of the n elements of a step, from its seed and the element's number (tensors one after the other, each padded to
    a multiple of 256): two rounds of multiplication and shifts, in arithmetic modulo 2^32."""
    low = 0xFFFFFFFF
    i = torch.arange(n, device=device)
    h = ((i & low) * 0x9E3779B1 + (i >> 32) * 0x7FEB352D + seed % (1 << 32) * 0x6A09E667 + (seed >> 32) % (1 << 32) * 0x3C6EF373) & low
    h = ((h ^ (h >> 15)) * 0x2C1B3C6D) & low
    h = ((h ^ (h >> 12)) * 0x297A2D39) & low
    return h ^ (h >> 15)


def _values(codes, scale):
    """What the codes stand for."""
    return codes.float() * scale.repeat_interleave(_BLOCK)


def _round_to_codes(x, u, least):
    """x, in blocks of 256, as codes and scales.  u in [0, 2^16) decides which of a value's two neighbours on the grid is taken: the upper one
    with a probability that is the value's distance from the lower one.  least: what is above zero does not become zero."""
    b = x.view(-1, _BLOCK)
    e = torch.frexp(b.abs().amax(1, keepdim=True))[1] - 8
    scale = torch.exp2(torch.where(b.abs().amax(1, keepdim=True) > 0, e, -100).clamp(min=-100).float())
    y = (b.abs() / scale).view(-1)
    small = y < 2.0 ** -6
    bits = torch.where(small, y + 2.0 ** -6, y).view(torch.int32)  # three bits of mantissa, or steps of 2^-9
    q = ((bits + (u * 16 + 8).int()) & ~0xFFFFF).view(torch.float32)
    q = torch.where(small, q - 2.0 ** -6, q)
    if least:
        q = torch.where(x > 0, q.clamp(min=2.0 ** -9), q)
    return (q * torch.sign(x)).to(torch.float8_e4m3fn), scale.view(-1)


def _plain_adamw(s):
    c, na = s["case"], s["na"]
    s["step"] += 1
    (b1, b2), lr, t = s["betas"], s["lr"], s["step"]
    g = torch.cat([s["grad"][:na], s["low_grad"].float()]) if c["low"] else s["grad"]
    if c["bits"] == 8:
        m, r = _values(s["m"], s["m_scale"]), _values(s["v"], s["v_scale"])
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = s["p"] * (1 - lr * s["weight_decay"]) - lr / (1 - b1 ** t) * m / (torch.sqrt(v) / math.sqrt(1 - b2 ** t) + s["eps"])
    s["p"].copy_(p)
    if c["low"]:
        s["low_p"].copy_(p[na:])
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"p": s["p"], "low_p": s.get("low_p"), "m": s["m"], "v": s["v"]}
    u = _random_bits(s["seed"] + t, m.numel(), m.device)
    out = {"p": s["p"], "low_p": s.get("low_p")}
    for name, x, bits, least in (("m", m, u & 0xFFFF, False), ("v", torch.sqrt(v), u >> 16, True)):
        codes, scale = _round_to_codes(x, bits, least)
        s[name].copy_(codes)
        s[name + "_scale"].copy_(scale)
        out[name] = _values(codes, scale).to(torch.bfloat16)
    return out


# ---- one pass ----------------------------------------------------------------------------------------------------------------


def run(s):
    c = s["case"]
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "linear": _plain_linear, "adamw": _plain_adamw}[c["kind"]](s)
    import gelib_b200 as gelib
    if c["kind"] == "adamw":
        s["step"] += 1
        gelib.adamw_step(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], step=s["step"], lr=s["lr"], betas=s["betas"], eps=s["eps"],
                         weight_decay=s["weight_decay"], exp_avg_scale=s["exp_avg_scale"], exp_avg_sq_scale=s["exp_avg_sq_scale"],
                         master=s["master"], seed=s["seed"] + s["step"])
        out = {"p": s["p"], "low_p": s.get("low_p"), "m": s["m"], "v": s["v"]}
        if c["bits"] == 8:  # a state in 8 bits is given as the values that it stands for (of v the root, which is what is held)
            out["m"], out["v"] = gelib.block8_values(s["m"], s["m_scale"]), gelib.block8_values(s["v"], s["v_scale"])
        return out
    if c["kind"] == "norm":
        y = gelib.group_norm(s["x"], c["groups"], s["weight"], s["bias"], eps=1e-5, activation=c["act"])
    else:
        y = gelib.linear(s["x"], s["w"], s["bias"], residual=s["residual"], activation=c["act"])
    if not c["train"]:
        return y
    return [y, *torch.autograd.grad(y, [s[q] for q in s["inputs"]], s["gy"])]


def work(case):
    c = case
    if c["kind"] == "adamw":
        mixing, head = _shapes(c)
        a, b = (sum(_floats(*q) for q in h) for h in (mixing, head))
        states = 16 if c["bits"] == 32 else 4 + 16 / _BLOCK + 4  # both read and written; in 8 bits their values are given too
        return {"bytes": (12 + states) * a + ((14 if c["low"] else 12) + states) * b, "flops": (16 if c["bits"] == 32 else 60) * (a + b)}
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "norm":
        e = c["b"] * c["s"] * c["n"]
        return {"bytes": size * (4 if c["train"] else 2) * e + size * c["n"] * (4 if c["train"] else 2), "flops": (40 if c["train"] else 15) * e}
    m, k, n = c["m"], c["k"], c["n"]
    e = m * k + k * n + m * n + n * c["bias"] + m * n * c["residual"]
    if c["train"]:
        e += m * n + m * k + k * n + n * c["bias"]
    return {"bytes": size * e, "flops": 2.0 * m * k * n * (3 if c["train"] else 1)}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------


def _exact_act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def _exact_rounding(x, u, least):
    """The neighbours of x on the grid of its block, below and above, and which of them u takes."""
    y = x.abs().view(-1, _BLOCK)
    top = y.amax(1, keepdim=True)
    scale = torch.exp2((torch.floor(torch.log2(top)) - 7).clamp(min=-100))
    y = y / scale
    step = torch.exp2((torch.floor(torch.log2(y)) - 3).clamp(min=-9))
    q = torch.floor(y / step + (u.double().view_as(y) * 16 + 8) / 2 ** 20) * step
    if least:
        q = torch.where((y > 0) & (q == 0), 2.0 ** -9, q)
    return torch.copysign((q * scale).view(-1), x)


def _exact_adamw(s):
    c = s["case"]
    t = s["step"] + 1
    lr, (b1, b2) = s["lr"], s["betas"]
    p, g = s["p"].double(), s["grad"].double()
    if c["low"]:
        g[s["na"]:] = s["low_grad"].double()
    m, v = s["m"].double(), s["v"].double()
    if c["bits"] == 8:
        m = (m.view(-1, _BLOCK) * s["m_scale"].double()[:, None]).view(-1)
        v = (v.view(-1, _BLOCK) * s["v_scale"].double()[:, None]).view(-1).square()
    m = m + (1 - b1) * (g - m)
    v = v + (1 - b2) * (g * g - v)
    p = p - lr * s["weight_decay"] * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + s["eps"])
    out = {"p": p, "low_p": p[s["na"]:] if c["low"] else None, "m": m, "v": v}
    if c["bits"] == 8:
        u = _random_bits(s["seed"] + t, m.numel(), m.device)  # the random numbers are part of the operator's definition
        out["m"], out["v"] = _exact_rounding(m, u % 65536, False), _exact_rounding(v.sqrt(), u // 65536, True)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "adamw":
        return _exact_adamw(s)
    ins = [s[q].detach().double().requires_grad_(c["train"]) for q in s["inputs"]]
    v = dict(zip(s["inputs"], ins))
    if c["kind"] == "norm":
        x = v["x"].transpose(1, 2).reshape(c["b"], c["groups"], -1)
        var, mean = torch.var_mean(x, 2, correction=0, keepdim=True)
        xh = ((x - mean) / (var + 1e-5).sqrt()).view(c["b"], c["n"], c["s"]).transpose(1, 2)
        y = _exact_act(xh * v["weight"] + v["bias"], c["act"])
    else:
        z = torch.matmul(v["x"], v["w"])
        y = _exact_act(z + v["bias"] if c["bias"] else z, c["act"])
        y = y + v["residual"] if c["residual"] else y
    if not c["train"]:
        return y
    grads = torch.autograd.grad(y, ins, s["gy"].double())
    return [y.detach(), *grads]
