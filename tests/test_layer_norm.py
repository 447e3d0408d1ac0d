"""Layer normalisation on the CPU: the oracle, the module, its place in the flower head and in checkpoints."""
import pytest
import torch

from distributed_tensorflow_amd.models.layers import LayerNorm, cast_for_device
from distributed_tensorflow_amd.ops import functional as F
from distributed_tensorflow_amd.ops import kernels as K


@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 5, 24), (4, 1000)])
def test_oracle_matches_the_definition(shape):
    gen = torch.Generator().manual_seed(shape[-1])
    x = torch.randn(shape, generator=gen, dtype=torch.float64, requires_grad=True)
    gamma = torch.randn(shape[-1], generator=gen, dtype=torch.float64, requires_grad=True)
    beta = torch.randn(shape[-1], generator=gen, dtype=torch.float64, requires_grad=True)
    y = F.layer_norm(x, gamma, beta, eps=1e-3)
    want = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-3).sqrt() * gamma + beta
    torch.testing.assert_close(y, want, rtol=1e-12, atol=1e-12)
    few = [t.detach()[..., :7].clone().requires_grad_(True) for t in (x[:1], gamma, beta)]
    assert torch.autograd.gradcheck(lambda *a: F.layer_norm(*a, eps=1e-3), few)


def test_module_keeps_its_parameters_fp32():
    m = cast_for_device(LayerNorm(16), "cpu", torch.bfloat16)
    assert m.gamma.dtype == m.beta.dtype == torch.float32
    x = torch.randn(3, 16)
    torch.testing.assert_close(m(x), torch.nn.functional.layer_norm(x, (16,)), rtol=1e-5, atol=1e-5)


def test_refusals():
    x = torch.zeros(4, 8)
    for bad in [lambda: F.layer_norm(x, torch.ones(7)), lambda: F.layer_norm(x, None, torch.ones(2, 4)),
                lambda: F.layer_norm(x[:, :0]), lambda: F.layer_norm(torch.tensor(1.0)),
                lambda: K.layer_norm_fwd(x, None, None, 1e-5), lambda: K.layer_norm_bwd(x, x, None, torch.zeros(2, 4))]:
        with pytest.raises(ValueError):
            bad()


def test_row_layouts_are_recognised():
    t = torch.zeros(4, 6, 100)
    for x, pitch in [(t, 100), (t[..., 10:42], 100), (t[:, :1, 3:50], 600), (t[1:2, 2:3, 5:9], 4), (t[:, 2], 600)]:
        rows, got = K._ln_rows(x)
        assert got == pitch and rows.data_ptr() == x.data_ptr()
    for x in (t.transpose(1, 2), t[:, 1:4, :50], t[..., ::2], t[:1, :1].expand(4, 6, 100)):
        rows, got = K._ln_rows(x)
        assert rows.is_contiguous() and got == x.shape[-1] and torch.equal(rows, x)
