"""Newton-Schulz kernels on matrices whose rows differ in size by orders of magnitude.

Small rows grow by up to 3.4445 per step relative to large ones, until they matter as much as these, and so does what was
rounded away in them.  The yardstick is the error of the same iteration in plain fp32 (``ref`` on the CPU), which keeps
24 bits in entries of any size.  A kernel's operands carry 22 bits, four times fp32's rounding at worst and about 2.5 times for
errors of random sign next to fp32's other roundings: 3 times its error is allowed.  On small matrices fp32 may come out
nearer by luck than its roundings; what the last two iterations of 22 bits must be allowed is 2^-23 for the last and at most
3.9 times that, the iteration's steepest slope on [0.68, 1.21], for the one before: 5 * 2^-23 of the norm.
"""
import pytest
import torch

from distributed_tensorflow_amd.ops import functional as F
from distributed_tensorflow_amd.ops import newton_schulz as ns
from distributed_tensorflow_amd.ops import ref

pytestmark = pytest.mark.gpu

STEPS = [5, 8, 10, ns.MAX_STEPS]
FLOOR = 5 * 2.0 ** -23


def _graded(rows, cols, small):
    """Half of the rows times ``small``."""
    g = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows + cols))
    g[rows // 2:] *= small
    return g


def _errors(g, steps):
    want = ref.newton_schulz(g.double(), steps)
    got = F.orthogonalize(g.cuda(), steps=steps).cpu().double() - want
    return want, got, ref.newton_schulz(g, steps).double() - want


@pytest.mark.parametrize("steps", STEPS)
@pytest.mark.parametrize("small", [1e-2, 1e-4, 1e-6, 1e-8, 1e-12])
@pytest.mark.parametrize("rows,cols", [(8, 8), (64, 576), (576, 64), (128, 256), (256, 128), (600, 1030), (1024, 1024)])
def test_rows_of_two_sizes(rows, cols, small, steps):
    want, got, fp32 = _errors(_graded(rows, cols, small), steps)
    off, allowed = got.norm().item(), 3 * fp32.norm().item() + FLOOR * want.norm().item()
    assert off <= allowed, "%.3g against %.3g, fp32 %.3g" % (off, allowed, fp32.norm().item())


@pytest.mark.parametrize("small", [1e-2, 1e-4, 1e-6, 1e-8])
@pytest.mark.parametrize("rows,cols", [(8, 8), (64, 576), (576, 64), (128, 256), (256, 128), (600, 1030)])
def test_the_small_rows_by_themselves(rows, cols, small):
    # next to the yardstick: entries below 2^-29 are rounded to multiples of 2^-50, off by 2^-51 at most, in X_0 and
    # (after growing by 3.4445 each time) the iterates after it, 1.41 * 2^-51 * 3.4445^5 in the result, and as much again
    # through A and B
    want, got, fp32 = _errors(_graded(rows, cols, small), 5)
    half = slice(rows // 2, rows)
    off, size = got[half].norm().item(), want[half].norm().item()
    step = 2 * 1.41 * 2.0 ** -51 * 3.4445 ** 5 * (rows // 2 * cols) ** 0.5
    allowed = 3 * fp32[half].norm().item() + FLOOR * size + step
    assert off <= allowed, "%.3g against %.3g of %.3g" % (off, allowed, size)


@pytest.mark.parametrize("steps", [5, ns.MAX_STEPS])
@pytest.mark.parametrize("kind", ["rows", "columns", "both", "entries"])
@pytest.mark.parametrize("rows,cols", [(64, 576), (500, 33), (256, 512)])
def test_sizes_spread_over_ten_decades(rows, cols, kind, steps):
    gen = torch.Generator().manual_seed(5)
    g = torch.randn(rows, cols, generator=gen)
    r, c = (10 ** (-10 * torch.rand(shape, generator=gen)) for shape in ((rows, 1), (1, cols)))
    g = g * {"rows": r, "columns": c, "both": r * c, "entries": 10 ** (-10 * torch.rand(rows, cols, generator=gen))}[kind]
    want, got, fp32 = _errors(g, steps)
    off, allowed = got.norm().item(), 3 * fp32.norm().item() + FLOOR * want.norm().item()
    assert off <= allowed, "%.3g against %.3g" % (off, allowed)


def test_small_rows_in_a_muon_step():
    from distributed_tensorflow_amd.optim import OptRegion, make_optimizer

    g = _graded(128, 256, 1e-6).reshape(-1)
    w = torch.zeros_like(g)
    region = OptRegion("r", w.cuda(), g.cuda(), None, True, [(0, 128, 256)])
    make_optimizer("muon", [region], 1.0, momentum=0.0, nesterov=False, ns_steps=ns.MAX_STEPS).step()
    want = -ref.newton_schulz(g.view(128, 256).double(), ns.MAX_STEPS)
    fp32 = (ref.newton_schulz(g.view(128, 256), ns.MAX_STEPS).double() + want).norm().item()
    off = (region.w.cpu().double().view(128, 256) - want).norm().item()
    assert off <= 3 * fp32 + FLOOR * want.norm().item()


def test_more_steps_than_small_entries_have_bits_for_are_refused():
    for x in (torch.zeros(4, 8), torch.zeros(4, 8, device="cuda")):
        with pytest.raises(ValueError, match="steps"):
            F.orthogonalize(x, steps=13)
