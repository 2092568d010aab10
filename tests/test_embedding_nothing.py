"""Complex embedding tables of no rows, no channels or no numbers."""
import pytest
import torch


@pytest.mark.gpu
def test_complex_tables_of_nothing():
    """No rows, no channels, no numbers: results and gradients of the right shapes, and NaN where a number names no row."""
    import gelib_b200 as G
    for n, v, d in ((0, 0, 3), (2, 0, 3), (0, 5, 3), (4, 5, 0), (0, 0, 0)):
        weight = torch.ones(v, d, device="cuda", dtype=torch.complex64, requires_grad=True)
        y = G.embedding(torch.zeros(n, dtype=torch.long, device="cuda"), weight, 2.0)
        assert y.shape == (n, d) and y.dtype == torch.complex64
        assert v > 0 or torch.view_as_real(y.detach()).isnan().all()
        gw, = torch.autograd.grad(y, weight, torch.ones_like(y))
        assert gw.shape == (v, d) and gw.dtype == torch.complex64 and (gw == 0).all()


def test_a_complex_table_of_no_rows_on_the_host_is_refused_like_others(cabi):
    import gelib_b200 as G
    for v in (0, 5):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            G.embedding(torch.zeros(2, dtype=torch.long), torch.zeros(v, 3, dtype=torch.complex64))


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_nothing_is_sorted_where_no_gradient_follows(native, monkeypatch):
    """One launch for the lookup, two with the sort: whatever the strides of the ids, and by either host side."""
    import gelib_b200 as G
    if not native:
        monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    ids = torch.arange(200, device="cuda") % 7
    for weight in (torch.randn(7, 16, device="cuda", requires_grad=True), torch.randn(7, 16, device="cuda", dtype=torch.complex64, requires_grad=True)):
        for numbers in (ids, ids[::2]):
            launches = []
            for wanted in (True, False):
                with torch.set_grad_enabled(wanted):
                    before = G._lib.lib().gelib_kernel_launch_count()
                    y = G.embedding(numbers, weight)
                    launches.append(G._lib.lib().gelib_kernel_launch_count() - before)
                assert y.requires_grad == wanted and torch.equal(y, weight[numbers])
            assert launches == [2, 1]
