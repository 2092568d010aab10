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
