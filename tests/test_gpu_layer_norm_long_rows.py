"""Layer normalisation of rows of more than 2^26 values, whose parameter gradients are longer than one launch has threads."""
import pytest
import torch

from distributed_tensorflow_amd.ops import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(1, (1 << 26) + 8), (2, (1 << 26) + 11), (3, (1 << 25) + 5)])
def test_parameter_gradients(rows, cols):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    dy = torch.randn(rows, cols, generator=gen, device="cuda")
    stats = torch.stack([torch.linspace(-0.5, 0.5, rows), torch.linspace(0.8, 1.3, rows)]).cuda()
    dx, dg, db = K.layer_norm_bwd(dy, x, None, stats, want_dx=False)
    assert dx is None
    # a column's sum: for each row a difference, a product with rstd, one with dy and a sum, five roundings of 2^-24 with
    # the first of up to (|x| + |mean|); columns at the start, around 2^25 and 2^26, and at the end
    for lo in (0, (1 << 25) - 64, cols - 128):
        s = slice(lo, lo + 128)
        mean, rstd = stats[0].double().view(-1, 1), stats[1].double().view(-1, 1)
        xd, dd = x[:, s].double(), dy[:, s].double()
        terms = dd * (xd - mean) * rstd
        size = (dd.abs() * (xd.abs() + mean.abs()) * rstd).sum(0)
        assert ((dg[s].double() - terms.sum(0)).abs() <= (4 + rows) * 2.0 ** -24 * size).all()
        assert ((db[s].double() - dd.sum(0)).abs() <= rows * 2.0 ** -24 * dd.abs().sum(0)).all()
    # and every one: in fp32, a few roundings more
    want = (dy * ((x - stats[0].view(-1, 1)) * stats[1].view(-1, 1)))
    off = (dg - want.sum(0)).abs() - 2.0 ** -20 * want.abs().sum(0)
    assert off.max().item() <= 0.0
    assert ((db - dy.sum(0)).abs() - 2.0 ** -20 * dy.abs().sum(0)).max().item() <= 0.0
