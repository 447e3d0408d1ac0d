"""Forward-mode derivatives of layer normalisation and orthogonalisation: right on the CPU or refused, never dropped."""
import pytest
import torch
from torch.autograd import forward_ad

from distributed_tensorflow_amd.ops import functional as F


def test_layer_norm_on_the_cpu_keeps_the_tangent():
    gen = torch.Generator().manual_seed(1)
    x, t = (torch.randn(3, 8, dtype=torch.float64, generator=gen) for _ in range(2))
    gamma = torch.randn(8, dtype=torch.float64, generator=gen)
    with forward_ad.dual_level():
        got = forward_ad.unpack_dual(F.layer_norm(forward_ad.make_dual(x, t), gamma)).tangent
    h = 1e-6   # central differences: h^2 * f''' and 2^-53 / h of values of size 1
    want = (F.layer_norm(x + h * t, gamma) - F.layer_norm(x - h * t, gamma)) / (2 * h)
    torch.testing.assert_close(got, want, rtol=1e-7, atol=1e-7)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_orthogonalize_refuses_tangents(device):
    x = torch.randn(4, 8, device=device)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="differentiable"):
            F.orthogonalize(forward_ad.make_dual(x, torch.ones_like(x)))
        F.orthogonalize(x)   # a plain tensor, whatever the level
    F.orthogonalize(x)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
def test_layer_norm_on_the_gpu_refuses_tangents(which):
    args = [torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda"), torch.zeros(8, device="cuda")]
    plain = F.layer_norm(*args)
    with forward_ad.dual_level():
        assert torch.equal(F.layer_norm(*args), plain)
        for grad in (False, True):   # with and without a graph to build
            dual = [forward_ad.make_dual(a.clone(), torch.ones_like(a)) if i == which else a.clone().requires_grad_(grad)
                    for i, a in enumerate(args)]
            with pytest.raises(ValueError, match="forward-mode"):
                F.layer_norm(*dual)
