"""How group norm and dense layers are called."""
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
