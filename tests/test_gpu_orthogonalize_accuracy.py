"""How far the Newton-Schulz kernels are off, against the same iteration in plain fp32.

Up to 3 million values the yardstick is ``ref`` in fp32 on the CPU, whose sums go by blocks: operands of 22 bits where fp32
has 24 make up to four times its roundings, of random sign and next to the sums' own, so 3 times its error is allowed, and
5 * 2^-23 of the norm for what the last two iterations of 22 bits must be (2^-23 for the last, the slope of 3.9 for the one
before) where fp32 comes out nearer by luck.  Above that it is the card's own fp32 products, and no more than their error is
allowed: reductions of thousands of values in one accumulator must not gather a bias.
"""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import functional as F
from distributed_tensorflow_amd.ops import ref
from distributed_tensorflow_amd.optim import OptRegion, make_optimizer

pytestmark = pytest.mark.gpu

FLOOR = 5 * 2.0 ** -23


def _matrix(rows, cols, kind):
    gen = torch.Generator().manual_seed(rows + cols)
    g = torch.randn(rows, cols, generator=gen)
    if kind == "directions":   # a few strong directions over noise, as averaged gradients have
        k = max(1, min(rows, cols) // 8)
        g = g + (torch.randn(rows, k, generator=gen) * torch.arange(1, k + 1) ** -0.5) @ torch.randn(k, cols, generator=gen)
    if kind == "offset":       # every product of the same sign
        g = g + 1.0
    return g


@pytest.mark.parametrize("kind", ["noise", "directions", "offset"])
@pytest.mark.parametrize("rows,cols", [(1, 7), (8, 8), (12, 500), (32, 72), (64, 64), (64, 576), (576, 64), (64, 8192), (1500, 17),
                                       (64, 8300), (128, 256), (256, 2304), (1531, 777), (512, 4608), (1000, 1000)])
def test_within_three_times_fp32(rows, cols, kind):
    g = _matrix(rows, cols, kind)
    want = ref.newton_schulz(g.double())
    fp32 = (ref.newton_schulz(g).double() - want).norm().item()
    off = (F.orthogonalize(g.cuda()).cpu().double() - want).norm().item()
    assert off <= 3 * fp32 + FLOOR * want.norm().item(), "%.3g, fp32 %.3g" % (off, fp32)


@pytest.mark.parametrize("kind", ["noise", "directions", "offset"])
@pytest.mark.parametrize("rows,cols", [(2500, 2500), (2048, 8192), (4096, 4096), (8192, 8192), (100, 65536), (65536, 200)])
def test_long_reductions(rows, cols, kind):
    g = _matrix(rows, cols, kind).cuda()
    want = ref.newton_schulz(g.double())
    fp32 = (ref.newton_schulz(g).double() - want).norm().item()
    off = (F.orthogonalize(g).double() - want).norm().item()
    assert off <= fp32, "%.3g, fp32 %.3g" % (off, fp32)


@pytest.mark.parametrize("kind", ["noise", "directions", "offset"])
@pytest.mark.parametrize("rows,cols", [(8, 8), (12, 500), (32, 72), (500, 33), (64, 576), (64, 8192), (300, 200)])
def test_the_muon_step_is_as_accurate(rows, cols, kind):
    g = _matrix(rows, cols, kind)
    want = ref.newton_schulz(g.double())
    fp32 = (ref.newton_schulz(g).double() - want).norm().item()
    region = OptRegion("r", torch.zeros(g.numel()).cuda(), g.reshape(-1).cuda(), None, True, [(0, rows, cols)])
    make_optimizer("muon", [region], 1.0, momentum=0.0, nesterov=False).step()
    got = region.w.cpu().double().view(rows, cols) / -math.sqrt(max(1.0, rows / cols))
    off = (got - want).norm().item()
    assert off <= 3 * fp32 + FLOOR * want.norm().item(), "%.3g, fp32 %.3g" % (off, fp32)
