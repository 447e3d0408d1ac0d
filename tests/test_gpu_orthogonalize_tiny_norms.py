"""Newton-Schulz kernels where the norm is not far above the 1e-7 next to it, and one row has nearly all of it.

Then X_0 is small and has one large entry in its square, which is multiplied with 4.775 in 16 bits.  Tolerance, to first
order: in every step a singular value s may be off by 2^-22 (operands of 22 bits, a product of two) of the terms
3.4445 s + 4.7750 s^3 + 2.0315 s^5, and every later step multiplies that by its slope; doubled for what is of second order.
"""
import pytest
import torch

from distributed_tensorflow_amd.ops import functional as F
from distributed_tensorflow_amd.ops import ref

pytestmark = pytest.mark.gpu


def _allowed(g, steps=5):
    s = torch.linalg.svdvals(g.double())
    s = s / (s.norm() + 1e-7)
    off = torch.zeros_like(s)
    for _ in range(steps):
        off = off * (3.4445 - 3 * 4.7750 * s ** 2 + 5 * 2.0315 * s ** 4).abs() + \
            2.0 ** -22 * (3.4445 * s + 4.7750 * s ** 3 + 2.0315 * s ** 5)
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    return 2 * off.norm().item()


# |X_0| just below powers of two, between them, and above where the lift begins
SIZES = [f * 2.0 ** -e for f in (0.5001, 0.72, 0.8, 0.9001, 0.93, 0.97, 0.9999) for e in (0, 1, 2, 3, 7, 12)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 40), (3, 2), (64, 100), (80, 200), (300, 140)])
def test_one_row_has_the_norm(rows, cols, dtype):
    g = torch.zeros(len(SIZES), rows, cols)
    g[:, 0, 0] = 1.0
    g += 1e-3 * torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows))
    for m, size in zip(g, SIZES):
        m *= size / (1 - size) * 1e-7 / m.double().norm().item()
    g = g.to(dtype)
    got = F.orthogonalize(g.cuda()).cpu()
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    for o, m, size in zip(got, g, SIZES):
        want = ref.newton_schulz(m.double())
        off, allowed = (o.double() - want).norm().item(), _allowed(m) + half * want.norm().item() * (1 + 1e-3)
        assert off <= allowed, "|X_0| = %g: %.3g against %.3g" % (size, off, allowed)


def test_in_a_muon_step():
    from distributed_tensorflow_amd.optim import OptRegion, make_optimizer

    size = 0.97 * 2.0 ** -5
    g = torch.zeros(96, 160)
    g[7] = torch.randn(160, generator=torch.Generator().manual_seed(3))
    g *= size / (1 - size) * 1e-7 / g.double().norm().item()
    region = OptRegion("r", torch.zeros(g.numel()).cuda(), g.reshape(-1).cuda(), None, True, [(0, 96, 160)])
    make_optimizer("muon", [region], 1.0, momentum=0.0, nesterov=False).step()
    off = (region.w.cpu().double().view(96, 160) + ref.newton_schulz(g.double())).norm().item()
    assert off <= _allowed(g)
