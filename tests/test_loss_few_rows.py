"""Losses of up to eight rows, whose forward products have kernels of their own."""
import math

import pytest
import torch

from test_losses import DTYPES, call, make, near, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("m", [1, 2, 3, 8, 9])
def test_a_sure_class_has_no_gradient(m, wt, dtype):
    """z of thousands from products whose sums are rounded: a gradient's z is that of its own log-sum, to the last bit.

    p of the class is 1 in float32 and its dz 0, so that gradients hold the other classes' shares and no more: their sum over the rows, times T, times the
    largest factor, and a hundredth for roundings (from 1280 channels on the shares are below e^-1000).
    """
    for k in (64, 1280, 2056):
        x, w, bias, target, _ = make(m, k, 300, dtype, wt=wt)
        x.abs_()
        w[:, 7] = 4.0   # z is near 3.2 k there
        gy = torch.tensor(1.0, device="cuda")
        most = max(1.0, float(x.max()), float(w.abs().max()))
        for b in (None, bias):
            z = x.double() @ w.double() + (0 if b is None else b.double())
            for t, logits in ((1.0, None), (2.0, torch.full((m, 1), 3.0, device="cuda"))):
                others = torch.exp((z - z[:, 7:8]) / t)
                others[:, 7] = 0
                assert float(others.sum(1).max()) < 2.0 ** -30
                allowed = 1.01 * t * most * float(others.sum())
                sure = torch.full((m,) if logits is None else (m, 1), 7, device="cuda")
                got = run(x, w, b, sure, logits, gy, temperature=t)
                assert got[0] == 0 and all((g.abs() <= allowed).all() for g in got[1:]), (k, t, allowed, [g.abs().max().item() for g in got])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("m", [1, 2, 5, 8])
def test_large_logits(m, top, dtype):
    """A share below 2^-126 is zero (float32's smallest normal number): so much of dz / g T more is allowed than where z is small, times x or w and summed."""
    for wt in (False, True):
        x, w, bias, target, logits = make(m, 1030, 300, dtype, wt=wt, top=top)
        x = x * 50
        gy = torch.ones(m, device="cuda")
        for b in (bias, None):
            got = run(x, w, b, target, logits, gy, reduction="none")
            wants = reference(x, w, b, target, logits, 2.0, gy, "none")
            least = 2.0 * 2.0 ** -126
            gone = (0, least * w.double().abs().sum(1), least * x.double().abs().sum(0)[:, None], least * m)
            for t, (value, allowed), more in zip(got, wants, gone):
                near(t, (value, allowed + more), (wt, b is None))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [0, 5])
def test_one_gradient_at_a_time_twice_and_on_two_streams(top, dtype):
    """The log-sums that a backward call makes for itself are its own: calls on one loss do not meet."""
    x, w, bias, target, logits = make(2, 200, 3000, dtype, top=top)
    gy = torch.tensor(1.0, device="cuda")
    want = run(x, w, bias, target, logits, gy)
    for i in range(3):
        a = [x, w, bias]
        a[i] = a[i].clone().requires_grad_()
        loss = call(*a, target, logits)
        assert torch.equal(loss.detach(), want[0])
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for turn in range(4):
            with torch.cuda.stream(streams[turn % 2]):
                got.append(torch.autograd.grad(loss, a[i], gy, retain_graph=True)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(g, want[1 + i]) for g in got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("m", [2, 3, 8])
def test_classes_that_do_not_exist(m, top, wt, dtype):
    """The row's loss and gradients are NaN and no other row's."""
    x, w, bias, target, logits = make(m, 64, 90, dtype, wt=wt, top=top)
    gy = torch.ones(m, device="cuda")
    clean = run(x, w, bias, target, logits, gy, reduction="none")
    others = torch.arange(m, device="cuda") != 1
    for bad in (90, 91, 2 ** 31 - 1, 2 ** 31, 2 ** 33 + 3, 2 ** 62) + (() if top else (-1, -2, -101, -2 ** 40)):
        t = target.clone()
        if top:
            t[1, 3] = bad
        else:
            t[1] = bad
        got = run(x, w, bias, t, logits, gy, reduction="none")
        assert got[0][1].isnan() and got[1][1].isnan().all() and got[2].isnan().all() and got[3].isnan().all()
        assert torch.equal(got[0][others], clean[0][others]) and torch.equal(got[1][others], clean[1][others])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 8])
def test_classes_that_a_bias_takes_out(m, dtype):
    """All classes out, and values that are no numbers: NaN, in their rows alone."""
    x, w, bias, target, _ = make(m, 64, 300, dtype)
    target = target.clamp(min=0)
    gy = torch.ones(m, device="cuda")
    assert all(t.isnan().all() for t in run(x, w, torch.full_like(bias, -math.inf), target, None, gy, reduction="none")[:2])
    out = torch.where(torch.arange(300, device="cuda") % 3 == 0, -math.inf, bias)
    target = torch.where(target % 3 == 0, 1, target)
    got = run(x, w, out, target, None, gy, reduction="none")
    assert all(torch.isfinite(t).all() for t in got) and (got[3][::3] == 0).all() and (got[2][:, ::3] == 0).all()
    if m == 1:
        return
    clean = run(x, w, bias, target, None, gy, reduction="none")
    for bad in (math.nan, math.inf):
        odd = x.clone()
        odd[1, 3] = bad
        got = run(odd, w, bias, target, None, gy, reduction="none")
        others = torch.arange(m, device="cuda") != 1
        assert not torch.isfinite(got[0][1]) and torch.equal(got[0][others], clean[0][others]) and torch.equal(got[1][others], clean[1][others])


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("m,dtype", [(1, torch.bfloat16), (2, torch.float16), (8, torch.float32)])
def test_a_captured_step_beside_eager_ones(m, dtype, top):
    x, w, bias, target, logits = make(m, 200, 3000, dtype, top=top)
    gy = torch.tensor(64.0, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(x, w, bias, target, logits, gy)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, w, bias, target, logits, gy)
    for turn in range(3):
        x.mul_(1.5)
        w.neg_()
        gy.mul_(0.5)
        graph.replay()
        eager = run(x, w, bias, target, logits, gy)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        for t, want in zip(out, reference(x, w, bias, target, logits, 2.0, gy, "mean")):
            near(t, want, "replayed")


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("m", [1, 8])
def test_the_python_host_side_gives_the_same(m, top, monkeypatch):
    import gelib_b200 as G
    for wt in (False, True):
        for dtype in DTYPES:
            args = make(m, 90, 36, dtype, wt=wt, top=top)
            gy = torch.ones(m, device="cuda")
            want = run(*args, gy, reduction="none")
            with monkeypatch.context() as patch:
                patch.setattr(G._lib, "_native", G._lib._Declines())
                assert all(torch.equal(a, b) for a, b in zip(run(*args, gy, reduction="none"), want))
