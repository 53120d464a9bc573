"""Layer norm of so many columns that the column sums' launch cannot have a workgroup for every 16 of them."""
import pytest
import torch

from categoricalnf_amd import functional as Fn

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("cols", [2 ** 24 - 8, 2 ** 25 + 40])
def test_parameter_gradients_of_millions_of_columns(cols):
    """Two rows; against the formula in 64 bits.  A row's statistics are sums of cols / 1024 terms in a lane and 32 more: with n of them off
    by 2 n 2^-24 of the row's largest |x| and of rstd; a column's sums are of two terms."""
    gen = torch.Generator("cuda").manual_seed(3)
    x, g = (torch.randn(2, cols, device="cuda", generator=gen).bfloat16() for _ in range(2))
    w, b = torch.ones(cols, device="cuda", requires_grad=True), torch.zeros(cols, device="cuda", requires_grad=True)
    y = Fn.layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), g)
    g64, n = g.double(), cols / 1024 + 32
    assert float((db.double() - g64.sum(0)).abs().max()) <= 2 * U * float(db.abs().max())
    xh = x.double()
    xh -= xh.mean(1, keepdim=True)
    xh *= torch.rsqrt(xh.square().mean(1, keepdim=True) + 1e-5)
    want = (g64 * xh).sum(0)
    size = float(xh.abs().max())
    slack = (g64.abs().sum(0) * (2 * n * U * 2 * size + 4 * U * size))
    assert bool(((dw.double() - want).abs() <= slack).all())
