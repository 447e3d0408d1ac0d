"""Layer normalisation of rows whose mean is large against their spread.

The variance is the mean square around the computed mean, so the mean's error e enters it as e^2 (the deviations from the true
mean add up to zero); taken as E[x^2] - E[x]^2 it would be off by thousands of roundings of mean^2, here up to 1e8 times the
variance.  u = 2^-24, K u the relative error of a row's sum (K = 64 + cols / 128: what a thread and the tree add up):

    e_mean = K u mean|x| + u |mean|
    e_var  = e_mean^2 + (K + 4) u (var + e_mean^2)           e_rstd = rstd (e_var rstd^2 / 2 + 3 u)
    e_xhat = rstd (e_mean + u |x - mean|) + |x - mean| e_rstd + 2 u |xhat|

and from there through the sums and products of the outputs, rounded once to their type.
"""
import pytest
import torch

from distributed_tensorflow_amd.ops import kernels as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _exact(x, gamma, beta, dy, eps):
    x, dy, g, b = x.double(), dy.double(), gamma.double(), beta.double()
    rows, cols = x.shape
    k = 64 + cols / 128
    mean = x.mean(1, keepdim=True)
    dev = x - mean
    var = (dev ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = dev * rstd
    e_mean = k * U * x.abs().mean(1, keepdim=True) + U * mean.abs()
    e_var = e_mean ** 2 + (k + 4) * U * (var + e_mean ** 2)
    e_rstd = rstd * (e_var * rstd ** 2 / 2 + 3 * U)
    e_xh = rstd * (e_mean + U * dev.abs()) + dev.abs() * e_rstd + 2 * U * xh.abs()
    y = xh * g + b
    e_y = g.abs() * e_xh + 3 * U * (xh * g).abs() + U * y.abs()
    d = dy * g
    m0, m1 = d.mean(1, keepdim=True), (d * xh).mean(1, keepdim=True)
    dx = rstd * (d - m0 - xh * m1)
    e_m0 = (k + 2) * U * d.abs().mean(1, keepdim=True)
    e_m1 = (k + 4) * U * (d * xh).abs().mean(1, keepdim=True) + (d.abs() * e_xh).mean(1, keepdim=True)
    e_dx = rstd * (4 * U * (d.abs() + m0.abs() + (xh * m1).abs()) + e_m0 + m1.abs() * e_xh + xh.abs() * e_m1 + e_xh * e_m1) \
        + dx.abs() / rstd * e_rstd + 2 * U * dx.abs()
    kr = 256 + rows / 128
    dg, db = (dy * xh).sum(0), dy.sum(0)
    e_dg = (dy.abs() * e_xh).sum(0) + kr * U * (dy * xh).abs().sum(0)
    return (y, dx, dg, db), (e_y, e_dx, e_dg, kr * U * dy.abs().sum(0))


# rows of a few lanes, of a wave, of several, of a workgroup of 256, 512 and 1024 threads, and those that are walked again
@pytest.mark.parametrize("dtype,offset", [(torch.float32, 1e3), (torch.float32, -1e4), (torch.float16, 900.0), (torch.bfloat16, 100.0)],
                         ids=["fp32-1e3", "fp32-1e4", "fp16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(40, 24), (40, 136), (3000, 64), (30, 520), (30, 1001), (1030, 2049), (20, 4100), (12, 7000),
                                       (6, 16390), (5, 40000)])
def test_offset_rows(rows, cols, dtype, offset):
    gen = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = (torch.randn(rows, cols, generator=gen, device="cuda") + offset).to(dtype)
    x[1::2] = (x[1::2] - 2 * offset).to(dtype)   # every other row on the other side of zero
    dy = (torch.randn(rows, cols, generator=gen, device="cuda") * 0.3).to(dtype)
    gamma = torch.randn(cols, generator=gen, device="cuda") * 0.3 + 1.0
    beta = torch.randn(cols, generator=gen, device="cuda") * 0.2
    y, stats = K.layer_norm_fwd(x, gamma, beta, 1e-5, want_stats=True)
    grads = K.layer_norm_bwd(dy, x, gamma, stats)
    want, err = _exact(x, gamma, beta, dy, 1e-5)
    half = torch.finfo(dtype).eps / 2
    for got, w, e, name in zip((y,) + grads, want, err, ("y", "dx", "dgamma", "dbeta")):
        h = half if got.dtype == dtype else 0.0
        tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
        worst = ((got.double() - w).abs() / (e + h * (w.abs() + e) + tiny)).max().item()
        assert worst <= 1.0, "%s: %.3g times its tolerance" % (name, worst)
