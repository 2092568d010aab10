"""Losses behind a last dense layer, and their gradients, against float64.

Tolerances.  z = x w + bias is off by EPS = 64 * 2^-24 of the sum of magnitudes of its terms (roundings of a sum, mostly cancelling; float32 factors are
split in three).  The logarithm of the sum of exp z is off by the mean of that under p, a row's p by that much relative to itself, and each by EPS of the
numbers that meet in them (exponents, logarithms and shares are good to a few units in the last place).  dz is rounded to 16 bits as an operand of
16-bit products: half a unit in its last place (float16: of 2^14 dz, 2^-25 at the least).  What is stored is rounded by half a unit in its last place.
"""
import math

import pytest
import torch

EPS = 64 * 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
LEAST = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -39}
SIZES = [(1, 1, 1), (1, 1280, 1000), (2, 64, 5), (3, 16, 8), (8, 40, 300), (64, 192, 100), (7, 33, 65), (130, 100, 257), (257, 129, 129), (128, 64, 256), (777, 204, 131),
         (300, 64, 2000), (1000, 96, 4099), (5000, 24, 40), (33, 2048, 33), (20, 31, 20011)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(m, k, n, dtype, wt=False, offset=0, pad=0, top=0, seed=0, dev="cuda"):
    """x, w, bias and the classes; with top the teacher's logits too."""
    gen = torch.Generator(device=dev).manual_seed(m + k + n + seed)

    def one(r, c, scale=1.0, extra=0):
        flat = (torch.randn(r * (c + extra) + offset, generator=gen, device=dev) * scale).to(dtype)
        return flat[offset:].view(r, c + extra)[:, :c]

    def numbers(*shape):
        return (torch.rand(*shape, generator=gen, device=dev) * n).long().clamp(max=n - 1)

    w = one(n, k, 2 * k ** -0.5, pad).t() if wt else one(k, n, 2 * k ** -0.5, pad)
    x, bias = one(m, k, extra=pad), one(1, n, 0.5)[0]
    missing = torch.rand(m, generator=gen, device=dev) < (0.15 if m > 1 else 0)
    if not top:
        target = numbers(m)
        target[missing] = -100
        return x, w, bias, target, None
    ids = numbers(m, top)
    ids[torch.rand(m, top, generator=gen, device=dev) < 0.2] = -1
    ids[missing] = -7
    return x, w, bias, ids, (torch.randn(m, top, generator=gen, device=dev) * 2 + 3).to(dtype)


def reference(x, w, bias, target, logits, temperature, gy, reduction):
    """(value, allowed error) of the loss, gx, gw, gb in float64."""
    half, tiny, least = HALF[x.dtype], TINY[x.dtype], LEAST[x.dtype]
    t = temperature if logits is not None else 1.0
    x, w = x.double(), w.double()
    b = torch.zeros(w.size(1), dtype=torch.float64, device=x.device) if bias is None else bias.double()
    if logits is None:
        entry = (target != -100)[:, None]
        ids, q = target[:, None].clamp(min=0), entry.double()
        log_q, off_q = torch.zeros_like(q), torch.zeros_like(q)
    else:
        entry = (target >= 0) & (logits != -math.inf)
        ids = target.clamp(min=0)
        s = torch.where(entry, logits.double() / t, -math.inf)
        some = entry.any(1, keepdim=True)
        log_q = torch.where(entry, s - torch.where(some, torch.logsumexp(s, 1, keepdim=True), 0.0), 0.0)
        q = torch.where(entry, log_q.exp(), 0.0)
        off_q = q * EPS * (1 + torch.where(entry, s.abs(), 0.0) + log_q.abs())
    live = entry.any(1)
    x = torch.where(live[:, None], x, 0.0)   # what stands in the other rows does not matter
    z = (x @ w + b) / t
    off_z = EPS * (x.abs() @ w.abs() + b.abs()) / t + EPS * z.abs()
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = (z - lse).exp()
    off_lse = (p * off_z).sum(1, keepdim=True) + EPS * (1 + lse.abs())
    log_p = z.gather(1, ids) - lse
    off_log = off_z.gather(1, ids) + off_lse + EPS * (log_q.abs() + z.gather(1, ids).abs() + lse.abs())
    rows = t * t * (q * (log_q - log_p)).sum(1)
    off_rows = t * t * (q * off_log + off_q * (1 + log_q.abs() + log_p.abs())).sum(1)
    count = max(1, int(live.sum())) if reduction == "mean" else 1
    gy = gy.double()
    if reduction == "none":
        loss, off_loss = rows, off_rows
    else:
        loss, off_loss = rows.sum() / count, (off_rows.sum() + EPS * rows.abs().sum()) / count
        gy = gy / count
    g = (t * gy * live)[:, None] if reduction == "none" else t * gy * live[:, None]
    sparse = torch.zeros_like(p).scatter_add_(1, ids, q)
    off_dz = p * (off_z + off_lse) + EPS * (p + sparse) + torch.zeros_like(p).scatter_add_(1, ids, off_q)
    dz = (p - sparse) * g
    off_dz = off_dz * g.abs() + 4 * EPS * dz.abs()
    off_dz = off_dz + half * (dz.abs() + off_dz) + least * g.abs().max()
    size = dz.abs() + off_dz

    def stored(v, off):
        return v, off + half * (v.abs() + off) + tiny

    return ((loss, off_loss), stored(dz @ w.t(), off_dz @ w.abs().t() + EPS * (size @ w.abs().t())),
            stored(x.t() @ dz, x.abs().t() @ off_dz + EPS * (x.abs().t() @ size)), stored(dz.sum(0), off_dz.sum(0) + EPS * size.sum(0)))


def call(x, w, bias, target, logits, temperature=2.0, reduction="mean"):
    import gelib_b200 as G
    if logits is None:
        return G.linear_cross_entropy(x, w, target, bias, reduction=reduction)
    return G.linear_distillation(x, w, target, logits, bias, temperature, reduction)


def run(x, w, bias, target, logits, gy, temperature=2.0, reduction="mean"):
    leaves = [t.detach().requires_grad_() for t in (x, w, bias) if t is not None]
    loss = call(leaves[0], leaves[1], leaves[2] if bias is not None else None, target, logits, temperature, reduction)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, gy)]


def near(got, want, what):
    """What lies within its error of 65520 or beyond is an infinity of its sign in float16."""
    value, allowed = want
    off = (got.double() - value).abs()
    right = off <= allowed
    if got.dtype == torch.float16:
        right |= (got.double() == value.sign() * math.inf) & (value.abs() + allowed >= 65520)
    wrong = got.shape != value.shape or not bool(right.all())
    assert not wrong, (what, (off / allowed).max().item())


def check(args, reduction="mean", temperature=2.0, gy=None):
    x, w, bias, target, logits = args
    if gy is None:
        gy = torch.tensor(512.0 if x.dtype == torch.float16 else 0.75, device=x.device)
        if reduction == "none":
            gy = gy * (0.25 + torch.rand(x.size(0), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")) / x.size(0)
    got = run(x, w, bias, target, logits, gy, temperature, reduction)
    wants = reference(x, w, bias, target, logits, temperature, gy, reduction)
    assert got[0].dtype == torch.float32
    for t, want, what in zip(got, wants, ("loss", "gx", "gw", "gb")):
        assert what == "loss" or t.dtype == x.dtype
        near(t, want, (what, reduction))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["plain", "transposed", "odd", "odd transposed"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_cross_entropy_against_float64(m, k, n, layout, dtype):
    """odd: one element off their alignment, rows three elements longer than the matrix."""
    odd = "odd" in layout
    args = make(m, k, n, dtype, "transposed" in layout, offset=1 if odd else 0, pad=3 if odd else 0)
    check(args, ("mean", "sum", "none")[(m + k + n + odd) % 3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["plain", "odd transposed"])
@pytest.mark.parametrize("m,k,n,top", [(1, 8, 3, 1), (1, 100, 50, 70), (64, 192, 100, 7), (33, 65, 300, 300), (777, 204, 1003, 16), (300, 64, 5003, 64), (9, 24, 4000, 1024)])
def test_distillation_against_float64(m, k, n, top, layout, dtype):
    odd = "odd" in layout
    args = make(m, k, n, dtype, "transposed" in layout, offset=1 if odd else 0, pad=3 if odd else 0, top=top)
    for reduction, temperature in (("mean", 1.0), ("none", 3.0)) if m < 300 else (("sum", 1.5),):
        check(args, reduction, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_in_pieces_of_the_classes(dtype, top):
    """More numbers of z than are worked on at a time, with and without sums that are split."""
    check(make(40000, 16, 4500, dtype, wt=True, top=top))
    check(make(70000, 8, 2100, dtype, top=top), "none")


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("m", list(range(1, 20)) + [31, 32, 33, 63, 65, 127, 128, 129, 255, 257])
def test_every_small_number_of_rows(m, top):
    for dtype in (torch.float32, torch.bfloat16):
        check(make(m, 72, 136, dtype, wt=m % 2 == 0, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 7, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 191, 255, 256, 257, 300, 511, 513])
def test_every_small_number_of_classes(n):
    for dtype in DTYPES:
        for top in (0, 3):
            check(make(140, 40, n, dtype, wt=n % 3 == 0, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [0, 6])
def test_without_bias_only_some_gradients_and_repeats(dtype, top):
    x, w, bias, target, logits = make(200, 100, 72, dtype, top=top)
    check((x, w, None, target, logits))
    gy = torch.tensor(1.0, device="cuda")
    all_of = run(x, w, bias, target, logits, gy)
    again = run(x, w, bias, target, logits, gy)
    assert all(torch.equal(a, b) for a, b in zip(all_of, again))
    with torch.no_grad():
        assert torch.equal(call(x, w, bias, target, logits), all_of[0])
    for i in range(3):
        a = [x.clone(), w.clone(), bias.clone()]
        a[i].requires_grad_()
        call(*a, target, logits).backward()
        assert torch.equal(a[i].grad, all_of[1 + i])
    for wide in ((40000, 24, 200), (48, 1500, 300), (3, 2000, 9000)):
        args = make(*wide, dtype, top=top)
        first, second = (run(*args, gy) for _ in range(2))
        assert all(torch.equal(p, q) for p, q in zip(first, second))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [0, 6, 12])
@pytest.mark.parametrize("m,k,n,wt", [(150, 64, 90, False), (150, 64, 90, True), (150, 63, 90, False), (600, 72, 3000, True), (2, 64, 90, False)])
def test_rows_without_a_loss(m, k, n, wt, dtype, top):
    """Whatever stands in such rows, and in the teacher's missing entries, changes no bit of anything; all rows like that: zeros."""
    x, w, bias, target, logits = make(m, k, n, dtype, wt=wt, top=top)
    if m == 2:
        target[1] = -100
    gy = torch.tensor(1.0, device="cuda")
    for bad in (float("nan"), float("inf")):
        clean = run(x, w, bias, target, logits, gy)
        x2 = x.clone()
        if top:
            logits2 = torch.where(target < 0, bad, logits)
            x2[(target < 0).all(1)] = bad
        else:
            logits2 = None
            x2[target == -100] = bad
        assert not torch.equal(x2, x)
        got = run(x2, w, bias, target, logits2, gy)
        assert all(torch.equal(a, b) for a, b in zip(got, clean))
        none = run(x2, w, bias, target, logits2, torch.ones(m, device="cuda"), reduction="none")
        rows = (target < 0).all(1) if top else target < 0
        assert (none[0][rows] == 0).all() and (none[1][rows] == 0).all()
    nothing = torch.full_like(target, -100)
    for reduction in ("mean", "sum"):
        for t in run(torch.full_like(x, float("nan")), w, bias, nothing, logits, gy, reduction=reduction):
            assert (t == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_classes_that_do_not_exist(dtype, top):
    """The row's loss and gradients are NaN and no other row's; nothing is read or written out of place."""
    x, w, bias, target, logits = make(140, 64, 90, dtype, top=top)
    gy = torch.ones(140, device="cuda")
    clean = run(x, w, bias, target, logits, gy, reduction="none")
    for bad in (90, 91, 2 ** 31 - 1, 2 ** 31, 2 ** 33 + 3, 2 ** 62) + (() if top else (-1, -2, -101, -2 ** 40)):
        t = target.clone()
        if top:
            t[5, 3] = bad
        else:
            t[5] = bad
        got = run(x, w, bias, t, logits, gy, reduction="none")
        rows = torch.arange(140, device="cuda") != 5
        assert got[0][5].isnan() and got[1][5].isnan().all() and got[2].isnan().all() and got[3].isnan().all()
        assert torch.equal(got[0][rows], clean[0][rows]) and torch.equal(got[1][rows], clean[1][rows])
        assert run(x, w, bias, t, logits, gy[0])[0].isnan()


@pytest.mark.gpu
def test_another_number_for_rows_without_a_class():
    import gelib_b200 as G
    x, w, bias, target, _ = make(100, 32, 20, torch.float32)
    for ignore in (3, -1, 20, -2 ** 40, 2 ** 40):
        t = torch.where(target == -100, ignore, target)
        a = G.linear_cross_entropy(x, w, t, bias, ignore_index=ignore)
        b = G.linear_cross_entropy(x, w, torch.where(t == ignore, -100, t), bias)
        assert torch.equal(a, b) and a > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_classes_that_a_bias_takes_out(dtype):
    """A bias of -infinity: such a class has no share; all of them: no number."""
    x, w, bias, target, _ = make(150, 64, 300, dtype)
    out = torch.arange(300, device="cuda") % 3 == 0
    target = torch.where(target % 3 == 0, (target + 1).clamp(max=299), target)
    target[target % 3 == 0] = 1
    masked = torch.where(out, -math.inf, bias)
    gy = torch.tensor(1.0, device="cuda")
    got = run(x, w, masked, target, None, gy)
    t = torch.where(target < 0, target, target - target // 3 - 1)
    small = [x, w[:, ~out].contiguous(), bias[~out].contiguous(), t, None]
    wants = reference(*small, 1.0, gy, "mean")
    near(got[0], wants[0], "loss")
    near(got[1], wants[1], "gx")
    near(got[2][:, ~out], wants[2], "gw")
    near(got[3][~out], wants[3], "gb")
    assert (got[2][:, out] == 0).all() and (got[3][out] == 0).all()
    lowest = torch.where(out, torch.finfo(dtype).min, bias)   # the type's lowest number does the same
    again = run(x, w, lowest, target, None, gy)
    near(again[0], wants[0], "loss")
    near(again[2][:, ~out], wants[2], "gw")
    assert run(x, w, torch.full_like(bias, -math.inf), target, None, gy)[0].isnan()
    target[0] = 0
    assert run(x, w, masked, target, None, gy)[0] == math.inf


@pytest.mark.gpu
def test_large_logits_and_sure_classes():
    """z of a thousand and more: the largest is taken off before exponents, and a class that is certain has a loss of zero."""
    for dtype in DTYPES:
        x, w, bias, target, _ = make(200, 64, 300, dtype)
        check((x * 200, w, bias, target, None))
        sure = torch.zeros_like(bias)
        sure[7] = 4000.0
        got = run(x, w, sure, torch.full_like(target, 7), None, torch.tensor(1.0, device="cuda"))
        assert all((t == 0).all() for t in got)
        # both passes have the same z, however long its sums
        for k in (1280, 1281, 2048, 5000):
            x, w, bias, target, _ = make(150, k, 300, dtype)
            got = run(x, w, sure, torch.full_like(target, 7), None, torch.tensor(1.0, device="cuda"))
            assert all((t == 0).all() for t in got), k
            check((x, w, bias, target, None))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_no_numbers_stay_in_their_rows(dtype):
    x, w, bias, target, _ = make(140, 64, 300, dtype)
    target = target.clamp(min=0)
    gy = torch.ones(140, device="cuda")
    clean = run(x, w, bias, target, None, gy, reduction="none")
    for bad in (float("nan"), float("inf")):
        x2 = x.clone()
        x2[9, 3] = bad
        got = run(x2, w, bias, target, None, gy, reduction="none")
        rows = torch.arange(140, device="cuda") != 9
        assert torch.equal(got[0][rows], clean[0][rows]) and torch.equal(got[1][rows], clean[1][rows])
        assert not torch.isfinite(got[0][9])


@pytest.mark.gpu
def test_a_teacher_like_a_class_and_its_entries_in_any_order():
    """One entry is a class; the order of entries, missing ones among them, changes nothing but roundings; several entries of one class add up."""
    import gelib_b200 as G
    x, w, bias, target, _ = make(100, 48, 70, torch.float32)
    one = G.linear_distillation(x, w, target[:, None], torch.full((100, 1), 5.0, device="cuda"), bias)
    assert torch.equal(one, G.linear_cross_entropy(x, w, target, bias))
    x, w, bias, ids, logits = make(100, 48, 70, torch.float32, top=9)
    gy = torch.tensor(1.0, device="cuda")
    a = run(x, w, bias, ids, logits, gy)
    b = run(x, w, bias, ids.flip(1), logits.flip(1), gy)
    for p, q in zip(a, b):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-6 * float(q.abs().max()))
    same = ids.clone()
    same[:] = 11
    single = run(x, w, bias, torch.full((100, 1), 11, device="cuda"), logits[:, :1], gy)
    for p, q in zip(run(x, w, bias, same, logits, gy)[1:], single[1:]):
        assert torch.allclose(p, q, rtol=1e-4, atol=1e-6 * float(q.abs().max()))
    for other in (torch.bfloat16, torch.float16):   # the teacher's type is its own
        check((x, w, bias, ids.int(), logits.to(other)))
    gone = logits.clone()
    gone[:, 4] = -math.inf
    check((x, w, bias, ids, gone))
    apart = logits.clone()
    apart[:, 2] = 300.0   # shares that are no numbers of float32 above zero
    check((x, w, bias, ids, apart), temperature=1.0)
    apart[3, 5], ids[3, 5] = float("nan"), 1
    assert run(x, w, bias, ids, apart, torch.ones(100, device="cuda"), reduction="none")[0][3].isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 5])
def test_gradients_against_differences(top):
    """Differences of the operator itself: a step of 2^-5 along a direction leaves a third of its square, and the losses' error over the step."""
    x, w, bias, target, logits = make(40, 24, 17, torch.float32, top=top)
    gy = torch.ones(40, device="cuda")
    _, gx, gw, gb = run(x, w, bias, target, logits, gy, reduction="none")
    step = 2.0 ** -5
    for i, grad in enumerate((gx, gw, gb)):
        d = torch.randn(grad.shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")
        d = d / d.norm()
        sides = []
        for sign in (1, -1):
            a = [x, w, bias]
            a[i] = a[i] + sign * step * d
            sides.append(call(*a, target, logits, reduction="none").double().sum())
        slope, want = (sides[0] - sides[1]) / (2 * step), (grad.double() * d.double()).sum()
        # third derivatives of a row's loss along a unit direction of z are at most 1; |dz| <= |x| |dw| + |dx| |w| per row and T <= 2
        size = 8 * max(1.0, float(x.norm(dim=1).max()), float(w.norm())) ** 3
        assert abs(slope - want) <= step ** 2 / 6 * size * 0.5 + EPS / step * float(sides[0].abs())


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 5])
def test_shapes_strides_and_streams(top):
    x, w, bias, target, logits = make(60, 48, 40, torch.float32, top=top)
    for reduction in ("mean", "none"):
        def go(x, w, target, logits):
            return call(x, w, bias, target, logits, reduction=reduction)

        want = go(x, w, target, logits)
        lead = (3, 4, 5)

        def shaped(t):
            return None if t is None else t.view(*lead, *t.shape[1:])

        assert torch.equal(go(x.view(3, 4, 5, 48), w, shaped(target), shaped(logits)), want.view(lead) if reduction == "none" else want)
        one = go(x[7], w, target[7], None if logits is None else logits[7])
        assert one.dim() == 0 and (reduction == "mean" or torch.allclose(one, want[7], rtol=1e-5))
        assert torch.equal(go(x.t().contiguous().t(), w, target, logits), want)
        assert torch.equal(go(torch.view_as_complex(torch.stack([x, x], -1)).real, w, target, logits), want)
        assert torch.equal(go(x, torch.stack([w, w], -1)[..., 0], torch.stack([target, target], -1)[..., 0], None if logits is None else logits.t().contiguous().t()), want)
        assert torch.equal(go(x[:1].expand(60, 48), w, target, logits), go(x[:1].expand(60, 48).contiguous(), w, target, logits))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = go(x, w, target, logits)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(other, want)
    leaf = x.clone().requires_grad_()
    rows = call(leaf, w, bias, target, logits, reduction="none")
    a, = torch.autograd.grad(rows, leaf, torch.ones(1, device="cuda").expand(60), retain_graph=True)   # gradients of other strides
    b, = torch.autograd.grad(rows, leaf, torch.ones(120, device="cuda")[::2], retain_graph=True)
    c, = torch.autograd.grad(rows.sum(), leaf)
    assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_upstream_gradients_of_all_sizes():
    """float16: rows whose gradients differ by many powers of two, zero among them, and scaled losses."""
    for dtype in DTYPES:
        args = make(200, 64, 300, dtype)
        for scale in (2.0 ** -20, 1.0, 2.0 ** 10):
            if dtype == torch.float16 and scale < 1:
                continue
            check(args, "sum", gy=torch.tensor(scale, device="cuda"))
            gy = scale * 2.0 ** -(torch.arange(200, device="cuda") % 9).float()
            gy[::4] = 0
            check(args, "none", gy=gy)
            check(args, "none", gy=-gy)
        for t in run(*args, torch.zeros(200, device="cuda"), reduction="none")[1:]:
            assert (t == 0).all()


@pytest.mark.gpu
def test_a_table_that_is_looked_up_and_scored():
    """Both ends by one table, as they are used: the gradients of the table add up."""
    import gelib_b200 as G
    for dtype in DTYPES:
        gen = torch.Generator(device="cuda").manual_seed(3)
        table = (torch.randn(50, 32, generator=gen, device="cuda") * 0.3).to(dtype).requires_grad_()
        ids = torch.randint(50, (200,), generator=gen, device="cuda")
        target = torch.randint(50, (200,), generator=gen, device="cuda")
        scale = 512.0 if dtype == torch.float16 else 1.0
        loss = G.linear_cross_entropy(G.group_norm(G.embedding(ids, table, 2.0), 1, activation="silu"), table.t(), target)
        got, = torch.autograd.grad(loss * scale, table)
        wide = table.detach().double().requires_grad_()
        h = torch.nn.functional.silu(torch.nn.functional.layer_norm(2 * wide[ids], (32,)))
        want, = torch.autograd.grad(torch.nn.functional.cross_entropy(h @ wide.t(), target) * scale, wide)
        # five roundings of half a unit in the last place on the way, the largest numbers' at the most
        allowed = (1e-5 + 8 * HALF[dtype]) * want.abs().max() + TINY[dtype]
        assert (got.double() - want).abs().max() <= allowed


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 5])
def test_two_captured_graphs_and_eager_calls_in_between(top):
    graphs = []
    for seed, (m, k, n) in enumerate(((100, 48, 300), (600, 64, 2000))):
        x, w, bias, target, logits = make(m, k, n, torch.bfloat16, top=top, seed=seed)
        gy = torch.tensor(1.0, device="cuda")

        def step(args=(x, w, bias, target, logits, gy)):
            return run(*args)

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, (x, w, bias, target, logits, gy)))
    for turn in range(2):
        for graph, out, (x, w, bias, target, logits, gy) in graphs:
            x.mul_(0.5)
            target.copy_(target.flip(0))
            gy.mul_(1.5)
            run(x[:40], w, bias, target[:40], None if logits is None else logits[:40], gy)
            graph.replay()
        for graph, out, (x, w, bias, target, logits, gy) in graphs:
            for t, want in zip(out, reference(x, w, bias, target, logits, 2.0, gy, "mean")):
                near(t, want, "replayed")


@pytest.mark.gpu
def test_two_threads():
    """Calls of different sizes and types at the same time, each on a stream of its own."""
    import threading
    torch.cuda.synchronize()
    failed = []

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                args = make(100 + 37 * seed, 64, 500 + 300 * seed, DTYPES[seed % 3], top=5 * (seed % 2), seed=seed)
                for _ in range(10):
                    check(args)
        except Exception as e:   # shown by the thread that waits
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]


@pytest.mark.gpu
def test_sizes_of_nothing():
    import gelib_b200 as G
    w, b = torch.ones(8, 5, device="cuda", requires_grad=True), torch.ones(5, device="cuda", requires_grad=True)
    x = torch.ones(0, 8, device="cuda", requires_grad=True)
    none = torch.zeros(0, dtype=torch.long, device="cuda")
    for reduction in ("none", "sum", "mean"):
        for loss in (G.linear_cross_entropy(x, w, none, b, reduction=reduction),
                     G.linear_distillation(x, w, none.view(0, 1).expand(0, 3), torch.zeros(0, 3, device="cuda"), b, reduction=reduction)):
            assert loss.shape == ((0,) if reduction == "none" else ()) and (loss == 0).all()
            gx, gw, gb = torch.autograd.grad(loss, (x, w, b), torch.ones_like(loss))
            assert gx.shape == (0, 8) and gw.shape == (8, 5) and (gw == 0).all() and (gb == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("which", ["x", "w", "bias"])
@pytest.mark.parametrize("top", [0, 5])
def test_derivatives_that_do_not_exist_are_refused(which, native, top, monkeypatch):
    import torch.autograd.forward_ad as forward_ad
    import gelib_b200 as G
    if not native:
        monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    x, w, bias, target, logits = make(6, 5, 4, torch.float32, top=top)
    a = {"x": x, "w": w, "bias": bias}
    leaf = a[which] = a[which].clone().requires_grad_()
    g, = torch.autograd.grad(call(a["x"], a["w"], a["bias"], target, logits), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()
    with forward_ad.dual_level():
        a[which] = forward_ad.make_dual(leaf.detach(), torch.ones_like(leaf))
        with pytest.raises(RuntimeError, match="jvp|forward"):
            call(a["x"], a["w"], a["bias"], target, logits)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 5])
def test_the_python_host_side_gives_the_same(top, monkeypatch):
    import gelib_b200 as G
    for wt in (False, True):
        args = make(70, 90, 36, torch.bfloat16, wt=wt, top=top)
        for reduction in ("mean", "none"):
            gy = torch.ones(70 if reduction == "none" else (), device="cuda")
            want = run(*args, gy, reduction=reduction)
            with monkeypatch.context() as m:
                m.setattr(G._lib, "_native", G._lib._Declines())
                assert all(torch.equal(a, b) for a, b in zip(run(*args, gy, reduction=reduction), want))


@pytest.mark.gpu
def test_module():
    import gelib_b200 as G
    head = G.Classifier(24, 10, device="cuda")
    x, target = torch.randn(5, 24, device="cuda"), torch.tensor([1, 2, 3, -100, 9], device="cuda")
    z = head(x)
    loss = head.cross_entropy(x, target)
    assert torch.allclose(loss, torch.nn.functional.cross_entropy(z, target), rtol=1e-5)
    loss.backward()
    assert head.weight.grad is not None and head.bias.grad is not None
    same = head.distillation(x, torch.arange(10, device="cuda").expand(5, 10), z.detach())   # its own teacher
    assert same.abs() < 1e-5


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_reported():
    """On the host's side alone: the kernel is told not to wait, gives up, and says so to the next call and to async_status."""
    import gelib_b200 as G
    x, w, bias, target, _ = make(200, 64, 300, torch.bfloat16)
    want = run(x, w, bias, target, None, torch.tensor(1.0, device="cuda"))
    for part in ("forward", "backward"):
        leaf = x.clone().requires_grad_()
        loss = None if part == "forward" else call(leaf, w, bias, target, None)
        G._lib.set_option("inject_timeout", "1")
        try:
            if part == "forward":
                call(x, w, bias, target, None)
            else:
                torch.autograd.grad(loss, leaf)
            torch.cuda.synchronize()
        finally:
            G._lib.set_option("inject_timeout", "0")
        with pytest.raises(RuntimeError, match="wait"):
            G._lib.async_status()
    got = run(x, w, bias, target, None, torch.tensor(1.0, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("wt", [False, True])
def test_weights_of_more_than_2_to_31_elements(wt):
    """The last classes of a vocabulary of a million: their logits, and their gradients, against those of these classes alone."""
    import gelib_b200 as G
    if torch.cuda.get_device_properties(0).total_memory < 60 * 2 ** 30:
        pytest.skip("needs 60 GB of device memory")
    k, n, m, tail = 2056, (1 << 20) + 264, 20, 520
    assert k * n > 2 ** 31
    w = torch.zeros((n, k) if wt else (k, n), dtype=torch.bfloat16, device="cuda")
    w = w.t() if wt else w
    gen = torch.Generator(device="cuda").manual_seed(0)
    w[:, -tail:] = (torch.randn(k, tail, generator=gen, device="cuda") * k ** -0.5).to(w.dtype)
    x = torch.randn(m, k, generator=gen, device="cuda").to(w.dtype)
    target = n - 1 - torch.arange(m, device="cuda") % tail
    gy = torch.ones(m, device="cuda")
    loss, gx, gw = run(x, w, None, target, None, gy, reduction="none")
    # all other classes have z = 0: as one class with a bias of log of their number
    small = torch.cat([torch.zeros(k, 1, dtype=w.dtype, device="cuda"), w[:, -tail:]], 1).double()
    z = x.double() @ small
    z[:, 0] += math.log(n - tail)
    lse = torch.logsumexp(z, 1, keepdim=True)
    want = lse[:, 0] - z[torch.arange(m, device="cuda"), target - (n - tail) + 1]
    off = EPS * (x.double().abs() @ small.abs() + z.abs()).amax(1) * 2 + EPS * (1 + lse[:, 0].abs())
    assert ((loss.double() - want).abs() <= off).all()
    dz = (z - lse).exp()
    dz[torch.arange(m, device="cuda"), target - (n - tail) + 1] -= 1
    want_gx, want_gw = dz[:, 1:] @ small[:, 1:].t(), x.double().t() @ dz[:, 1:]
    # dz and the result are rounded to 16 bits
    size = dz[:, 1:].abs() + off[:, None]
    assert ((gx.double() - want_gx).abs() <= 2.0 ** -8 * (size @ small[:, 1:].abs().t() + want_gx.abs()) * 1.1 + 1e-6).all()
    assert ((gw[:, -tail:].double() - want_gw).abs() <= 2.0 ** -8 * (x.double().abs().t() @ size + want_gw.abs()) * 1.1 + 1e-6).all()
    first = x.double().t() @ ((z[:, :1] - lse).exp() / (n - tail)).expand(m, 8)   # a class of the many
    assert ((gw[:, :8].double() - first).abs() <= 2.0 ** -6 * first.abs() + 1e-9).all()


@pytest.mark.gpu
def test_more_than_2_to_31_numbers_of_dz():
    """A piece of dz beyond 2^31 elements: rows far down have the gradients that they have by themselves."""
    if torch.cuda.get_device_properties(0).total_memory < 60 * 2 ** 30:
        pytest.skip("needs 60 GB of device memory")
    m, k, n = 1100000, 16, 2048
    assert m * n > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(m, k, generator=gen, device="cuda").to(torch.bfloat16)
    w = (torch.randn(k, n, generator=gen, device="cuda") * 0.3).to(torch.bfloat16)
    target = torch.randint(n, (m,), generator=gen, device="cuda")
    loss, gx, gw = run(x, w, None, target, None, torch.ones(m, device="cuda"), reduction="none")
    for at in (0, m // 2 + 77, m - 300):
        rows = slice(at, at + 300)
        wants = reference(x[rows], w, None, target[rows], None, 1.0, torch.ones(300, device="cuda"), "none")
        near(loss[rows], wants[0], "loss")
        near(gx[rows], wants[1], "gx")
    want = torch.zeros(k, n, dtype=torch.float64, device="cuda")
    allowed = torch.zeros_like(want)
    for at in range(0, m, 110000):
        rows = slice(at, at + 110000)
        p = torch.softmax(x[rows].double() @ w.double(), 1)
        p[torch.arange(p.size(0), device="cuda"), target[rows]] -= 1
        want += x[rows].double().t() @ p
        allowed += x[rows].double().abs().t() @ p.abs()
    assert ((gw.double() - want).abs() <= (2.0 ** -8 + EPS) * allowed * 1.01 + 2.0 ** -8 * want.abs()).all()


def test_cpu_tensors_are_refused(cabi):
    import gelib_b200 as G
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        G.linear_cross_entropy(torch.zeros(2, 8), torch.zeros(8, 4), torch.zeros(2, dtype=torch.long))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        G.linear_distillation(torch.zeros(2, 8), torch.zeros(8, 4), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3))


def test_values_that_are_refused_before_tensors_are_looked_at(cabi):
    import gelib_b200 as G
    with pytest.raises(ValueError, match="reduction"):
        G.linear_cross_entropy(None, None, None, reduction="max")
    for temperature in (0, -1, 1e-16, 1e16, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            G.linear_distillation(None, None, None, None, temperature=temperature)


@pytest.mark.gpu
def test_hot_and_cold_teachers():
    for temperature in (1e-3, 0.1, 30.0, 1e4):
        check(make(100, 48, 70, torch.float32, top=9), temperature=temperature)


REFUSALS = {
    "sizes": ("n_in", dict(x=torch.zeros(2, 7))),
    "no channels": ("at least one", dict(x=torch.zeros(2, 0), w=torch.zeros(0, 4))),
    "no classes": ("at least one", dict(w=torch.zeros(8, 0), bias=None)),
    "bias": (r"bias must have shape \(4,\)", dict(bias=torch.zeros(8))),
    "type of w": ("w must be of x's type", dict(w=torch.zeros(8, 4, dtype=torch.bfloat16))),
    "double": ("float32, bfloat16 or float16", dict(x=torch.zeros(2, 8, dtype=torch.float64))),
    "type of target": ("int64 or int32", dict(target=torch.zeros(2))),
    "shape of target": (r"must have shape \(2,", dict(target=torch.zeros(3, dtype=torch.long))),
    "target elsewhere": ("on the device of x", dict(target=torch.zeros(2, dtype=torch.long))),
    "logits": ("logits must have shape", dict(logits=torch.zeros(2))),
    "rows of logits": ("logits must have shape", dict(logits=torch.zeros(3, 3))),
    "too many entries": ("1 to 1024", dict(logits=torch.zeros(2, 1025))),
    "no entries": ("1 to 1024", dict(logits=torch.zeros(2, 0))),
    "type of logits": ("float32, bfloat16 or float16", dict(logits=torch.zeros(2, 3, dtype=torch.float64))),
    "gradient of logits": ("no gradient", dict(logits=torch.zeros(2, 3, requires_grad=True))),
}


@pytest.mark.gpu
@pytest.mark.parametrize("which", list(REFUSALS))
def test_refusals(which):
    import gelib_b200 as G
    message, change = REFUSALS[which]
    args = dict(x=torch.zeros(2, 8), w=torch.zeros(8, 4), target=torch.zeros(2, dtype=torch.long), bias=torch.zeros(4), logits=torch.zeros(2, 3))
    args.update(change)
    args = {k: v.to("cuda").detach().requires_grad_(v.requires_grad) if v is not None and not (which == "target elsewhere" and k == "target") else v for k, v in args.items()}
    if "logits" not in which and "entries" not in which:
        with pytest.raises(RuntimeError, match=message):
            G.linear_cross_entropy(args["x"], args["w"], args["target"], args["bias"])
    target = args["target"]
    ids = target if "target" in which else torch.zeros(args["logits"].shape, dtype=torch.long, device="cuda")
    with pytest.raises(RuntimeError, match=message):
        G.linear_distillation(args["x"], args["w"], ids, args["logits"], args["bias"])


C_REFUSALS = {
    "no input channels": dict(k=0),
    "no classes": dict(n=0),
    "2^30": dict(m=2 ** 31),
    "65536 input channels": dict(k=65537, ldx=70000, ldw=70000),
    "unknown type": dict(type=3),
    "8 or 4 bytes": dict(index_bytes=3),
    "unknown reduction": dict(reduction=3),
    "GELIB_LOSS_MAX_TOP": dict(top=1025),
    "several classes": dict(top=2),
    "temperature": dict(teacher=4096, temperature=0.0),
    "rows overlap": dict(ldx=7),
    "null pointer": dict(target=0),
    "not aligned to its type": dict(gx=4097),
    "state is not": dict(state=4100),
    "workspace is not": dict(space=4100),
    "no workspace": dict(space=0),
}


@pytest.mark.parametrize("message", list(C_REFUSALS))
@pytest.mark.parametrize("backward", [False, True])
def test_arguments_of_the_c_abi(cabi, message, backward):
    """No kernel is launched: the addresses stand for nothing."""
    import ctypes
    from gelib_b200._lib import LinearLossArgs
    change = dict(C_REFUSALS[message])
    space = change.pop("space", 4096)
    a = LinearLossArgs(x=4096, w=4096, target=4096, loss=4096, state=4096, gy=4096, gx=4096, m=200, k=8, n=400, ldx=8, ldw=400, top=1, index_bytes=8, temperature=1.0, reduction=2)
    for name, value in change.items():
        setattr(a, name, value)
    fn = cabi.gelib_linear_loss_back if backward else cabi.gelib_linear_loss
    assert fn(ctypes.byref(a), space, None) == 2 and message in cabi.gelib_last_error().decode()


@pytest.mark.parametrize("kind,bytes_", [(0, 4), (1, 2), (2, 2)])
def test_workspaces_stay_below_the_logits(cabi, kind, bytes_):
    """Neither call has room for z of a large batch over a large vocabulary."""
    import ctypes
    from gelib_b200._lib import LinearLossArgs
    m, k, n = 65536, 1024, 262144
    a = LinearLossArgs(x=4096, w=4096, bias=4096, target=4096, loss=4096, state=4096, gy=4096, gx=4096, gw=4096, gb=4096, m=m, k=k, n=n, ldx=k, ldw=n, top=1, index_bytes=8,
                       temperature=1.0, type=kind)
    logits = m * n * bytes_
    for backward in (0, 1):
        assert 0 < cabi.gelib_linear_loss_workspace(ctypes.byref(a), backward) < logits / 6
    assert cabi.gelib_linear_loss_state_bytes(ctypes.byref(a)) < 16 * m
