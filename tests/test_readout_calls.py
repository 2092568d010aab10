"""How group norm and dense layers are called: forward-mode derivatives, several threads at a time, workspaces, very many statistics."""
import threading

import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("which", ["x", "w", "bias", "residual", "norm x", "norm weight", "norm bias"])
def test_forward_mode_is_refused(which, native, monkeypatch):
    """These operators have no forward-mode derivative: an operand with a tangent is refused, and none is dropped."""
    import gelib_b200 as G
    if not native:
        monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    a = {"x": torch.randn(4, 6, device="cuda"), "w": torch.randn(6, 5, device="cuda"), "bias": torch.randn(5, device="cuda"),
         "residual": torch.randn(4, 5, device="cuda"), "norm x": torch.randn(4, 6, device="cuda"), "norm weight": torch.randn(6, device="cuda"),
         "norm bias": torch.randn(6, device="cuda")}

    def call():
        if which.startswith("norm"):
            return G.group_norm(a["norm x"], 2, a["norm weight"], a["norm bias"])
        return G.linear(a["x"], a["w"], a["bias"], a["residual"])

    call()
    with forward_ad.dual_level():
        a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
        with pytest.raises(RuntimeError, match="jvp|forward"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("sizes", [((110, 128), (190, 128)), ((1200, 8192), (1200, 16384))])
def test_two_threads_with_different_sizes(cabi, sizes, backward):
    """Both sizes take the same kernels with more shared memory than a block has by itself, one of them much more.  Straight to the C ABI, where the
    interpreter's lock is held the least."""
    import ctypes
    errors, go = [], threading.Barrier(2)

    def work(s, n):
        x, y, gw, gb = (torch.randn(*shape, device="cuda") for shape in ((1, s, n), (1, s, n), (n,), (n,)))
        mean, rstd = torch.zeros(1, 1, device="cuda"), torch.ones(1, 1, device="cuda")
        bytes_ = cabi.gelib_group_norm_workspace(1, s, n, 1, 0, int(backward))
        space = torch.empty(max(1, bytes_), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        tail = (space.data_ptr(), ctypes.c_void_p(stream.cuda_stream))
        if backward:
            fn, args = cabi.gelib_group_norm_back, (y, gw, gb, x, x, None, None, mean, rstd)
            args = tuple(t if t is None else t.data_ptr() for t in args) + (1, s, n, 1, 0, 0) + tail
        else:
            fn, args = cabi.gelib_group_norm, (y.data_ptr(), None, None, x.data_ptr(), None, None, 1, s, n, 1, 1e-5, 0, 0) + tail
        go.wait()
        failed = sum(fn(*args) != 0 for _ in range(2000))
        stream.synchronize()
        errors.extend([cabi.gelib_last_error()] if failed else [])

    threads = [threading.Thread(target=work, args=size) for size in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


@pytest.mark.parametrize("s,n,groups,kind", [(2, 16384, 1, 1), (4, 7168, 1, 1), (2, 7168, 1, 0), (600, 4096, 4, 0)])
def test_workspace_of_the_gradient_stays_small(cabi, s, n, groups, kind):
    """Parameter gradients are partial sums per block that an SM holds, whatever the batch: at most two blocks on each of 148 SMs."""
    size = 4 if kind == 0 else 2
    for b in (1, 100, 4096, 100000):
        most = 2 * 296 * n * 4 + 64 * b * groups * max(1, s // 16)
        assert cabi.gelib_group_norm_workspace(b, s, n, groups, kind, 1) <= most, b
    b = 100000
    assert cabi.gelib_group_norm_workspace(b, s, n, groups, kind, 1) < b * s * n * size / 16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,s,n,groups", [(700, 2, 16384, 1), (700, 4, 7168, 1), (500, 900, 520, 4), (3, 3000, 520, 4)])
def test_gradients_of_more_pieces_than_blocks(b, s, n, groups, dtype):
    import gelib_b200 as G
    gen = torch.Generator(device="cuda").manual_seed(b + s)
    x, gy = (torch.randn(b, s, n, generator=gen, device="cuda").to(dtype) for _ in range(2))
    w, bias = (torch.randn(n, generator=gen, device="cuda").to(dtype) for _ in range(2))
    leaves = [t.requires_grad_() for t in (x, w, bias)]
    got = torch.autograd.grad(G.group_norm(x, groups, w, bias, activation="silu"), leaves, gy)
    for alone in range(3):   # each by itself, and the same when it is asked for again
        again, = torch.autograd.grad(G.group_norm(x, groups, w, bias, activation="silu"), leaves[alone], gy)
        assert torch.equal(again, got[alone])
    wants, sizes = [torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2)], [torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2)]
    for at in range(0, b, 100):
        with torch.no_grad():
            v = x[at:at + 100].double().view(-1, s, groups, n // groups)
            var, mean = torch.var_mean(v, (1, 3), correction=0, keepdim=True)
            h = ((v - mean) * (var + 1e-5).rsqrt()).reshape(-1, s, n)
            z = h * w.double() + bias.double()
            q = torch.sigmoid(z)
            g = gy[at:at + 100].double()
            gz = g * q * (1 + z * (1 - q))
            more = g.abs() * 1.2 * (1 + h.abs() * w.double().abs() + z.abs())
            for i, (a, c) in enumerate(((gz * h, more * (h.abs() + 1)), (gz, more))):
                wants[i] += a.sum((0, 1))
                sizes[i] += c.sum((0, 1))
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    for g, want, size in zip(got[1:], wants, sizes):
        assert ((g.double() - want).abs() <= 64 * 2.0 ** -24 * size + half * (want.abs() + 64 * 2.0 ** -24 * size)).all()


@pytest.mark.gpu
def test_more_than_2_to_31_statistics():
    import gelib_b200 as G
    if torch.cuda.get_device_properties(0).total_memory < 100 * 2 ** 30:
        pytest.skip("needs 100 GB of device memory")
    b, n, groups = 262200, 16384, 8192
    assert b * groups > 2 ** 31
    x = torch.empty(b, n, dtype=torch.float16, device="cuda").normal_().requires_grad_()
    y = G.group_norm(x, groups, activation="relu")
    gx, = torch.autograd.grad(y, x, x.detach())
    for at in (0, b - 1):
        one = x[at:at + 1].detach().clone().requires_grad_()
        want = G.group_norm(one, groups, activation="relu")
        gone, = torch.autograd.grad(want, one, one.detach())
        for got, ref in ((y[at:at + 1], want), (gx[at:at + 1], gone)):
            assert torch.allclose(got.float(), ref.float(), rtol=2.0 ** -10, atol=1e-4)
