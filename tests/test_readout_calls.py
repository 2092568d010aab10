"""How group norm and dense layers are called: forward-mode derivatives, several threads at a time."""
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
