"""Layer-normalisation kernels against the formulas in 64 bits.

Tolerances: u = 2^-24 is the relative error of one fp32 operation.  A sum over a row adds at most 32 values in a thread
(cols / 1024 vectors of 8 in the looping kernels) and then ten levels of a tree, so its error is below K u times the sum of
magnitudes with K = 64 + cols / 128.  These propagate through the formulas below; an output in 8, 11 or 24 bits is
then rounded once, by at most ``eps / 2`` of its type relative to the value.
"""
import pytest
import torch

from distributed_tensorflow_amd.models.layers import LayerNorm
from distributed_tensorflow_amd.ops import functional as F
from distributed_tensorflow_amd.ops import kernels as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _exact(x, gamma, beta, dy, eps):
    """64-bit outputs and the error each may have in fp32 arithmetic, before its rounding."""
    x, dy = x.double(), dy.double()
    rows, cols = x.shape
    g = torch.ones(cols, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    b = torch.zeros(cols, dtype=torch.float64, device=x.device) if beta is None else beta.double()
    k = 64 + cols / 128
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = xh * g + b
    e_mean = k * U * x.abs().mean(1, keepdim=True) + U * mean.abs()
    # the variance: the mean's error enters to second order, x - mean is rounded at the size of its operands
    e_rstd = (k * U + 4 * U) * rstd + rstd ** 2 * (e_mean + U * x.abs().amax(1, keepdim=True))
    e_xh = rstd * (e_mean + U * (x.abs() + mean.abs())) + (x - mean).abs() * e_rstd + 2 * U * xh.abs()
    e_y = g.abs() * e_xh + 3 * U * (xh * g).abs() + U * y.abs()
    d = dy * g
    m0, m1 = d.mean(1, keepdim=True), (d * xh).mean(1, keepdim=True)
    dx = rstd * (d - m0 - xh * m1)
    e_m0 = (k + 2) * U * d.abs().mean(1, keepdim=True)
    e_m1 = (k + 4) * U * (d * xh).abs().mean(1, keepdim=True) + (d.abs() * e_xh).mean(1, keepdim=True)
    e_dx = rstd * (4 * U * (d.abs() + m0.abs() + (xh * m1).abs()) + e_m0 + m1.abs() * e_xh + xh.abs() * e_m1) \
        + dx.abs() / rstd * e_rstd + 2 * U * dx.abs()
    # column sums: a thread's share of the rows one after the other, partial rows in strides of 32, one tree
    kr = 256 + rows / 128
    dg, db = (dy * xh).sum(0), dy.sum(0)
    e_dg = (dy.abs() * e_xh).sum(0) + kr * U * (dy * xh).abs().sum(0)
    e_db = kr * U * dy.abs().sum(0)
    return (y, dx, dg, db), (e_y, e_dx, e_dg, e_db)


def _check(got, want, err, what):
    half = torch.finfo(got.dtype).eps / 2
    # results below the type's normal range are rounded to a multiple of its smallest value
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got.double() - want).abs()
    allowed = err + half * (want.abs() + err) + tiny
    worst = (off / allowed).max().item() if off.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, "%s: %.3g times its tolerance" % (what, worst)


def _inputs(rows, cols, dtype, seed, pitch=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pitch = pitch or cols
    x = (torch.randn(rows, pitch, generator=gen, device="cuda") * 1.7 + 0.4).to(dtype)[:, :cols]
    dy = (torch.randn(rows, pitch, generator=gen, device="cuda") * 0.3).to(dtype)[:, :cols]
    gamma = torch.randn(cols, generator=gen, device="cuda") * 0.3 + 1.0
    beta = torch.randn(cols, generator=gen, device="cuda") * 0.2
    return x, dy, gamma, beta


SIZES = [(1, 1), (2, 3), (1, 8), (5, 7), (9, 64), (4, 65), (33, 128), (1030, 72), (17, 255), (1, 2048), (260, 513), (33, 1001),
         (67, 2049), (31, 4100), (7, 8200), (5, 16390), (3, 33001), (2, 40000), (4099, 16), (301, 136), (77, 191), (70, 330), (19, 760), (11, 1500),
         # more rows than the one-launch form takes
         (1100, 136), (1030, 200), (1029, 520), (1040, 1001), (1027, 1500), (1030, 2049), (1030, 4100), (1026, 8200), (1025, 16390),
         (1024, 2048), (1024, 2050),
         # the longest rows of fp32 that the backward holds
         (3, 16381), (600, 16384),
         (6, 2900), (6, 3301), (5, 6201), (5, 12001), (5, 14001), (4, 24001), (1030, 2900), (1029, 6201), (1026, 12001)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_forward_and_gradients(rows, cols, dtype):
    x, dy, gamma, beta = _inputs(rows, cols, dtype, rows * 7 + cols)
    for t in (x, gamma, beta):
        t.requires_grad_(True)
    y = F.layer_norm(x, gamma, beta, eps=1e-5)
    assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
    dx, dg, db = torch.autograd.grad(y, (x, gamma, beta), dy)
    assert dx.dtype == dtype and dg.dtype == db.dtype == torch.float32
    want, err = _exact(x.detach(), gamma.detach(), beta.detach(), dy, 1e-5)
    for got, w, e, name in zip((y.detach(), dx, dg, db), want, err, ("y", "dx", "dgamma", "dbeta")):
        _check(got, w, e, name)
    with torch.no_grad():
        assert torch.equal(F.layer_norm(x, gamma, beta, eps=1e-5), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,cols,pitch", [(70, 288, 768), (5, 64, 69), (12, 1001, 1003), (9, 4096, 4101), (3, 40000, 40003)])
def test_channel_slices_need_no_copy(rows, cols, pitch, dtype):
    x, dy, gamma, beta = _inputs(rows, cols, dtype, pitch, pitch)
    assert not x.is_contiguous() and K._ln_rows(x)[0] is x
    y, stats = K.layer_norm_fwd(x, gamma, beta, 1e-3, want_stats=True)
    grads = K.layer_norm_bwd(dy, x, gamma, stats)
    want, err = _exact(x, gamma, beta, dy, 1e-3)
    for got, w, e, name in zip((y,) + grads, want, err, ("y", "dx", "dgamma", "dbeta")):
        _check(got, w, e, name)


def test_a_slice_leaves_the_rest_of_its_buffer_alone():
    buf = torch.full((6, 100), 7.0, device="cuda")
    before = buf.clone()
    y = F.layer_norm(buf[:, 8:72])
    assert torch.equal(buf, before) and y.abs().max().item() == 0.0   # constant rows: (x - mean) is zero


@pytest.mark.parametrize("make", [lambda t: t.transpose(0, 1), lambda t: t[:, ::2], lambda t: t[:1].expand(40, -1),
                                  lambda t: t.view(2, 20, 4, 24).permute(1, 0, 2, 3), lambda t: t.view(4, 10, 96)[:, 1:7],
                                  lambda t: t.view(4, 10, 96)[:, ::3, 5:61], lambda t: t[0], lambda t: t.view(40, 1, 96)])
def test_any_layout(make):
    x = make(torch.randn(40, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)))
    y = F.layer_norm(x)
    rows = x.reshape(-1, x.shape[-1])
    want, err = _exact(rows, None, None, rows, 1e-5)
    assert y.shape == x.shape and y.is_contiguous()
    _check(y.view(rows.shape), want[0], err[0], "y")


@pytest.mark.parametrize("with_gamma,with_beta", [(False, False), (True, False), (False, True)])
def test_without_scale_or_offset(with_gamma, with_beta):
    x, dy, gamma, beta = _inputs(37, 200, torch.float32, 5)
    g, b = gamma if with_gamma else None, beta if with_beta else None
    x.requires_grad_(True)
    wrt = [x] + [t.requires_grad_(True) for t in (g, b) if t is not None]
    y = F.layer_norm(x, g, b)
    got = [y.detach()] + list(torch.autograd.grad(y, wrt, dy))
    want, err = _exact(x.detach(), None if g is None else g.detach(), None if b is None else b.detach(), dy, 1e-5)
    keep = [0, 1] + [2] * with_gamma + [3] * with_beta
    for t, i in zip(got, keep):
        _check(t, want[i], err[i], str(i))


def test_gradients_only_where_wanted():
    x, dy, gamma, beta = _inputs(50, 2304, torch.bfloat16, 6)
    _, stats = K.layer_norm_fwd(x, gamma, beta, 1e-5, want_stats=True)
    full = K.layer_norm_bwd(dy, x, gamma, stats)
    for want in [(True, False, False), (False, True, False), (False, False, True), (False, True, True), (False, False, False)]:
        for w, t, f in zip(want, K.layer_norm_bwd(dy, x, gamma, stats, *want), full):
            assert (t is None) if not w else torch.equal(t, f)


def test_gradient_agrees_with_differences():
    # fp32, central differences of step h in 64 bits of the kernel's own outputs: the loss is a sum of a few values of
    # size ~1, its rounding (2^-22) over 2 h = 2^-5 gives 2^-17, the third-order term h^2 / 6 * |f'''| is ~2^-12 * 2
    x, dy, gamma, beta = _inputs(2, 24, torch.float32, 11)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(F.layer_norm(x, gamma, beta), x, dy)
    h = 2.0 ** -6
    for c in (0, 7, 23):
        diff = 0.0
        for sign in (1, -1):
            moved = x.detach().clone()
            moved[1, c] += sign * h
            diff += sign * (F.layer_norm(moved, gamma, beta).double() * dy.double()).sum().item()
        assert abs(diff / (2 * h) - dx[1, c].item()) < 2.0 ** -10


def test_broadcast_upstream_gradient():
    x, _, gamma, beta = _inputs(64, 96, torch.float32, 8)
    x.requires_grad_(True)
    F.layer_norm(x, gamma, beta).sum().backward()     # autograd hands the backward a gradient of stride 0
    dy = torch.ones(64, 96, device="cuda")
    want, err = _exact(x.detach(), gamma, beta, dy, 1e-5)
    _check(x.grad, want[1], err[1], "dx")


def test_rows_of_extremes_do_not_touch_their_neighbours():
    x, dy, gamma, beta = _inputs(40, 136, torch.float32, 9)
    clean = K.layer_norm_fwd(x, gamma, beta, 1e-5, want_stats=True)
    dx = K.layer_norm_bwd(dy, x, gamma, clean[1])[0]
    bad = x.clone()
    bad[3, 5], bad[4, 0], bad[5, 135] = float("nan"), float("inf"), float("-inf")
    bad[6] = torch.finfo(torch.float32).min
    y, stats = K.layer_norm_fwd(bad, gamma, beta, 1e-5, want_stats=True)
    dxb = K.layer_norm_bwd(dy, bad, gamma, stats)[0]
    rest = [i for i in range(40) if i not in (3, 4, 5, 6)]
    assert torch.equal(y[rest], clean[0][rest]) and torch.equal(dxb[rest], dx[rest])
    assert y[3:6].isnan().all() and not y[rest].isnan().any()


def test_constant_and_zero_rows():
    x = torch.zeros(3, 1000, device="cuda")
    x[1] = 5.0
    beta = torch.arange(1000, device="cuda").float()
    y = F.layer_norm(x, None, beta, eps=1e-5)
    # the mean of equal values: 1000 roundings of 5 at most leave |x - mean| <= 74 u * 5 = 2.2e-5, times 1 / sqrt(eps) = 316
    assert torch.equal(y[0], beta) and torch.equal(y[2], beta) and (y[1] - beta).abs().max().item() < 7e-3


def test_no_rows():
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    gamma = torch.ones(64, device="cuda", requires_grad=True)
    beta = torch.zeros(64, device="cuda", requires_grad=True)
    y = F.layer_norm(x, gamma, beta)
    y.sum().backward()
    assert y.shape == (0, 64) and x.grad.shape == (0, 64)
    assert torch.equal(gamma.grad, torch.zeros_like(gamma)) and torch.equal(beta.grad, torch.zeros_like(beta))


def test_repeatable():
    x, dy, gamma, beta = _inputs(20000, 64, torch.bfloat16, 12)
    _, stats = K.layer_norm_fwd(x, gamma, beta, 1e-5, want_stats=True)
    first = K.layer_norm_bwd(dy, x, gamma, stats)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, K.layer_norm_bwd(dy, x, gamma, stats)))


def test_more_than_2_to_31_elements():
    rows, cols = (1 << 20) + 5, 2056
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").fill_(1.0)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x[-3:] = torch.randn(3, cols, generator=gen, device="cuda").bfloat16()
    dy = torch.zeros_like(x)
    dy[-2:] = 0.25
    gamma = torch.randn(cols, generator=gen, device="cuda")
    y, stats = K.layer_norm_fwd(x, gamma, None, 1e-5, want_stats=True)
    dx, dg, db = K.layer_norm_bwd(dy, x, gamma, stats)
    want, err = _exact(x[-3:], gamma, None, dy[-3:], 1e-5)
    for got, w, e, name in zip((y[-3:], dx[-3:], dg, db), want, err, ("y", "dx", "dgamma", "dbeta")):
        _check(got, w, e, name)
    assert not y[0].any() and not dx[:-3].any()


def test_captured_forward_and_backward_replays():
    x, dy, gamma, beta = _inputs(300, 520, torch.bfloat16, 13)
    fresh = [_inputs(300, 520, torch.bfloat16, 20 + i)[:2] for i in range(3)]

    def once():
        y, stats = K.layer_norm_fwd(x, gamma, beta, 1e-5, want_stats=True)
        return (y,) + K.layer_norm_bwd(dy, x, gamma, stats)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for nx, ndy in fresh:
        x.copy_(nx)
        dy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, once()))


def test_on_another_stream():
    x, dy, gamma, beta = _inputs(500, 1024, torch.bfloat16, 14)
    want = K.layer_norm_fwd(x, gamma, beta, 1e-5)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.layer_norm(x, gamma, beta)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_gradients_go_straight_into_flat_buffers():
    m = LayerNorm(72).cuda()
    with torch.no_grad():
        m.gamma.normal_()
    x, dy, _, _ = _inputs(30, 72, torch.bfloat16, 15)
    x.requires_grad_(True)
    plain = torch.autograd.grad(m(x), (m.gamma, m.beta), dy)
    ready = []
    for p in (m.gamma, m.beta):
        p.main_grad = torch.full((72,), 3.0, device="cuda")
        p._grad_filled, p._grad_ready_cb = False, ready.append
    m(x).backward(dy)
    assert m.gamma.grad is None and m.beta.grad is None and len(ready) == 2
    assert torch.equal(m.gamma.main_grad, plain[0]) and torch.equal(m.beta.main_grad, plain[1])
    m(x).backward(dy)   # a second use in the same step adds up, and is reported once
    assert torch.equal(m.gamma.main_grad, 2 * plain[0]) and len(ready) == 2


def test_refusals():
    x = torch.zeros(4, 64, device="cuda")
    v = torch.ones(64, device="cuda")
    for bad in [lambda: F.layer_norm(x.double(), v, v), lambda: F.layer_norm(x.int(), v, v),
                lambda: F.layer_norm(x, v.bfloat16(), v), lambda: F.layer_norm(x, v[:63], v),
                lambda: F.layer_norm(x, v, v.view(8, 8)), lambda: F.layer_norm(x, v.cpu(), v),
                lambda: F.layer_norm(x[:, :0]), lambda: F.layer_norm(x, torch.ones(128, device="cuda")[::2], v),
                lambda: K.layer_norm_bwd(x.bfloat16(), x, v, torch.zeros(2, 4, device="cuda")),
                lambda: K.layer_norm_bwd(x[:3], x, v, torch.zeros(2, 4, device="cuda")),
                lambda: K.layer_norm_bwd(x, x, v, torch.zeros(2, 3, device="cuda")), lambda: K.layer_norm_fwd(x.cpu(), None, None, 1e-5)]:
        with pytest.raises(ValueError):
            bad()
    xg = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(F.layer_norm(xg, v, v).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):   # differentiable once
        g.sum().backward()
