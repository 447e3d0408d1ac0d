"""Newton-Schulz kernels and the Muon step against the definition in 64 bits.

How far a result may be off: the iteration multiplies an early rounding error by up to 3.44 per step, in the kernels as
in any fp32 computation, so the yardstick is the error that plain fp32 arithmetic makes on the same matrix (``ref`` on
the CPU, blocked sums).  A kernel's operand carries 22 bits where fp32 has 24, so each of its roundings is at most 4
times one of fp32's, with as much again for the dropped lo * lo products; and a product over K elements is 3 K / 16
sequential fp32 additions, whose rounding errors add up like a random walk.  Hence, in the Frobenius norm,
``error <= (8 + sqrt(3 K / 16)) * error of fp32 + one fp32 rounding``; losing one of the three partial products makes
the error a thousand times larger.  The result is then rounded to its type, by at most ``eps / 2``.
"""
import math

import pytest
import torch

from distributed_tensorflow_amd.models import build_model
from distributed_tensorflow_amd.ops import functional as F
from distributed_tensorflow_amd.ops import newton_schulz as ns
from distributed_tensorflow_amd.ops import ref
from distributed_tensorflow_amd.optim import OptRegion, make_optimizer
from distributed_tensorflow_amd.parallel.engine import DataParallelEngine

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _exact(g, steps=5):
    return ref.newton_schulz(g.double().cpu(), steps)


def _allowed(g, want, steps=5):
    """Error allowed before the rounding to the output's type, Frobenius norm."""
    base = (ref.newton_schulz(g.float().cpu(), steps).double() - want).norm().item()
    return (8 + math.sqrt(3 * max(g.shape) / 16)) * base + 2.0 ** -23 * want.norm().item()


def _check(got, g, steps=5):
    want = _exact(g, steps)
    off = (got.double().cpu() - want).norm().item()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    allowed = _allowed(g, want, steps) + half * want.norm().item() * (1 + 1e-3) + 1e-30
    assert off <= allowed, "%.3g against %.3g" % (off, allowed)


def _matrix(rows, cols, dtype, seed, kind="noise"):
    gen = torch.Generator().manual_seed(seed)
    g = torch.randn(rows, cols, generator=gen)
    if kind == "directions":   # a few strong directions over noise, as averaged gradients have
        r = max(1, min(rows, cols) // 8)
        g = g + (torch.randn(rows, r, generator=gen) * torch.arange(1, r + 1) ** -0.5) @ torch.randn(r, cols, generator=gen)
    return (g * 1e-3).to(dtype).cuda()


SIZES = [(1, 1), (1, 7), (7, 1), (3, 3), (8, 1024), (32, 72), (64, 64), (65, 63), (64, 576), (63, 300), (300, 63), (129, 1000),
         (512, 512), (515, 513), (512, 1030), (1000, 515), (640, 2049), (2049, 640), (64, 8192), (8200, 64), (40, 1500), (1500, 17), (1, 4000), (64, 8300)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_against_the_definition(rows, cols, dtype):
    g = _matrix(rows, cols, dtype, rows + 3 * cols)
    before = g.clone()
    o = F.orthogonalize(g)
    assert o.dtype == dtype and o.shape == g.shape and torch.equal(g, before)
    _check(o, g)


@pytest.mark.parametrize("rows,cols", [(64, 576), (300, 200), (1024, 600), (512, 4608)])
def test_directions_over_noise(rows, cols):
    g = _matrix(rows, cols, torch.float32, rows * cols, "directions")
    _check(F.orthogonalize(g), g)


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_number_of_steps(steps):
    g = _matrix(100, 260, torch.float32, steps)
    _check(F.orthogonalize(g, steps=steps), g, steps)


def test_singular_values_come_out_near_one():
    g = _matrix(96, 200, torch.float32, 9)
    s = torch.linalg.svdvals(F.orthogonalize(g).double().cpu())
    assert 0.65 < s.min().item() and s.max().item() < 1.25   # f^5 of 0.03 .. 0.2 lies in 0.68 .. 1.21


@pytest.mark.parametrize("scale", [1e-25, 1e-12, 1e12, 1e30])
def test_any_scale(scale):
    # squares of these overflow or vanish in fp32; at 1e-25 the 1e-7 next to the norm makes the result the scaled input
    g = _matrix(70, 130, torch.float32, 10) * scale
    _check(F.orthogonalize(g), g)


def test_batches_and_layouts():
    g = torch.stack([_matrix(40, 90, torch.float32, s) for s in range(6)])
    each = torch.stack([F.orthogonalize(m) for m in g])
    assert torch.equal(F.orthogonalize(g), each)
    assert torch.equal(F.orthogonalize(g.view(2, 3, 40, 90)), each.view(2, 3, 40, 90))
    t = F.orthogonalize(g.transpose(1, 2))
    assert t.is_contiguous() and t.shape == (6, 90, 40)
    _check(t[1], g[1].t())
    assert torch.equal(F.orthogonalize(g[:, 3:, 5:]), F.orthogonalize(g[:, 3:, 5:].contiguous()))
    assert torch.equal(F.orthogonalize(g[:1].expand(4, 40, 90))[3], each[0])
    assert F.orthogonalize(g[:0]).shape == (0, 40, 90)


def test_a_matrix_of_extremes_leaves_the_others_alone():
    g = torch.stack([_matrix(80, 200, torch.float32, s) for s in range(5)])
    want = F.orthogonalize(g)
    g[1, 3, 4], g[2, 0, 199], g[3] = float("nan"), float("inf"), 0.0
    got = F.orthogonalize(g)
    assert torch.equal(got[0], want[0]) and torch.equal(got[4], want[4])
    assert got[1].isnan().all() and got[2].isnan().all() and not got[3].any()


@pytest.mark.parametrize("rows,cols", [(300, 700), (700, 300), (130, 64), (256, 256)])
@pytest.mark.parametrize("large_from,piece", [(128, 1), (128, 3), (1 << 30, 1), (1 << 30, 5), (128, 1 << 30), (1 << 30, 1 << 30)])
def test_any_cut_of_the_work(monkeypatch, rows, cols, large_from, piece):
    # tile edges and pieces that the estimate would not take at these sizes
    monkeypatch.setattr(ns, "_choose", lambda dims, symmetric: (large_from, piece if symmetric else 1 << 30))
    g = torch.stack([_matrix(rows, cols, torch.float32, 50 + s) for s in range(2)])
    plan = ns.NsPlan([(0, rows, cols), (rows * cols, rows, cols)], g.device)
    out = torch.empty_like(g)
    plan.launch(inp=g, steps=5, out=out)
    for o, m in zip(out, g):
        _check(o, m)


@pytest.mark.parametrize("rows,cols", [(300, 340), (340, 300)])
def test_more_small_tiles_than_two_to_a_cu(monkeypatch, rows, cols):
    monkeypatch.setattr(ns, "_choose", lambda dims, symmetric: (1 << 30, 1 << 30))
    n = 40
    g = torch.stack([_matrix(rows, cols, torch.float32, 90 + s) for s in range(n)])
    plan = ns.NsPlan([(s * rows * cols, rows, cols) for s in range(n)], g.device)
    assert plan.counts[4] > 2 * ns.CUS and plan.counts[6] > 2 * ns.CUS   # tiles of A, of B
    out = torch.empty_like(g)
    plan.launch(inp=g, steps=5, out=out)
    for o, m in zip(out[::13], g[::13]):
        _check(o, m)


def test_leftover_tiles(monkeypatch):
    # a whole round of workgroups and a few tiles more, whose reductions are cut
    monkeypatch.setattr(ns, "_choose", lambda dims, symmetric: (1 << 30, 1 << 30))
    monkeypatch.setattr(ns, "SLOTS", 16)
    monkeypatch.setattr(ns, "MIN_STEPS", 1)
    g = _matrix(380, 1000, torch.float32, 60)
    plan = ns.NsPlan([(0, 380, 1000)], g.device)
    assert plan.slabs > 0
    out = torch.empty_like(g)
    plan.launch(inp=g, steps=5, out=out)
    _check(out, g)


def test_large_matrix():
    g = _matrix(4096, 4096, torch.float32, 61)
    want = ref.newton_schulz(g.double(), 2)
    base = (ref.newton_schulz(g, 2).double() - want).norm().item()
    off = (F.orthogonalize(g, steps=2).double() - want).norm().item()
    assert off <= (8 + math.sqrt(3 * 4096 / 16)) * base + 2.0 ** -23 * want.norm().item()


@pytest.mark.parametrize("rows,cols", [(100, 1 << 20), (1 << 20, 70)])
def test_longest_side(rows, cols):
    g = _matrix(rows, cols, torch.float32, 12)
    _check(F.orthogonalize(g, steps=1), g, 1)


def test_rank_one():
    u, v = _matrix(200, 1, torch.float32, 11), _matrix(1, 333, torch.float32, 12)
    g = (u @ v) * 1e6
    o = F.orthogonalize(g).double().cpu()
    s = 1.0
    for _ in range(5):
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    want = (u / u.norm()).double().cpu() @ (v / v.norm()).double().cpu() * s
    # the product u v is rounded to fp32 per entry: noise of 2^-25 |g| whose small singular values, up to
    # (sqrt(200) + sqrt(333)) / sqrt(200 * 333) = 0.13 of it, grow by 3.4445^5 = 485: 2e-6 each, 14 of them in the norm
    assert (o - want).norm().item() < 1e-4


def test_repeatable():
    g = _matrix(600, 1400, torch.float32, 13)
    first = F.orthogonalize(g)
    assert all(torch.equal(first, F.orthogonalize(g)) for _ in range(3))


def test_captured_and_replayed():
    g = _matrix(130, 260, torch.float32, 14)
    h = _matrix(64, 96, torch.bfloat16, 15)
    want = [F.orthogonalize(g), F.orthogonalize(h)]   # (uploads the plans)
    graphs = []
    for _ in range(2):   # two graphs of the same shapes
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = (F.orthogonalize(g), F.orthogonalize(h))
        graphs.append((graph, out))
    for seed in (20, 21, 22):
        g.copy_(_matrix(130, 260, torch.float32, seed))
        h.copy_(_matrix(64, 96, torch.bfloat16, seed))
        for graph, out in graphs:
            graph.replay()
        eager = (F.orthogonalize(g), F.orthogonalize(h))
        torch.cuda.synchronize()
        assert not torch.equal(eager[0], want[0])
        for _, out in graphs:
            assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_first_call_of_a_shape_cannot_be_captured():
    g = torch.zeros(37, 41, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = g + 1
        with pytest.raises(RuntimeError, match="capture"):
            F.orthogonalize(g)
    graph.replay()
    torch.cuda.synchronize()
    assert (kept == 1).all()


def test_two_streams_at_once():
    a, b = _matrix(256, 1152, torch.float32, 16), _matrix(256, 1152, torch.float32, 17)
    want = F.orthogonalize(a), F.orthogonalize(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(s1):
            x = F.orthogonalize(a)
        with torch.cuda.stream(s2):
            y = F.orthogonalize(b)
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    for bad in [lambda: F.orthogonalize(x.double()), lambda: F.orthogonalize(x[0]), lambda: F.orthogonalize(x, steps=0),
                lambda: F.orthogonalize(x[:, :0]), lambda: F.orthogonalize(x.clone().requires_grad_(True)),
                lambda: F.orthogonalize(x.int()), lambda: F.orthogonalize(x[:1, :1].expand(40000, 40000))]:
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------ the optimizer step
PLACES = [(0, 32, 72), (2304, 5, 7), (2368, 300, 64), (21568, 64, 300), (40768, 513, 600), (348608, 1, 64), (348672, 1000, 515)]
TOTAL = 863680


def _buffers(grad_dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    w, g, buf = torch.randn(TOTAL, generator=gen), torch.randn(TOTAL, generator=gen) * 1e-3, torch.randn(TOTAL, generator=gen) * 1e-2
    return w, g.to(grad_dtype), buf


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("nesterov", [True, False])
def test_step(grad_dtype, nesterov):
    w, g, buf = _buffers(grad_dtype, 30)
    region = OptRegion("r", w.cuda(), g.cuda(), w.bfloat16().cuda(), True, PLACES)
    opt = make_optimizer("muon", [region], 0.02, momentum=0.95, nesterov=nesterov, weight_decay=0.1)
    opt.buf["r"].copy_(buf)
    opt.step(grad_scale=0.5)
    gd = g.double() * 0.5
    m = 0.95 * buf.double() + gd
    u = gd + 0.95 * m if nesterov else m
    got_w, got_w16, got_buf = region.w.double().cpu(), region.w16.double().cpu(), opt.buf["r"].double().cpu()
    inside = torch.zeros(TOTAL, dtype=torch.bool)
    for at, r, c in PLACES:
        s = slice(at, at + r * c)
        inside[s] = True
        # buf: a product and a sum, three roundings
        assert ((got_buf[s] - m[s]).abs() <= 3 * 2.0 ** -24 * (0.95 * buf[s].double().abs() + gd[s].abs())).all()
        # the direction is rounded like buf: one more unit in the yardstick's input
        d = u[s].view(r, c)
        o = ref.newton_schulz(d, 5)
        rate = 0.02 * math.sqrt(max(1, r / c))
        want = w[s].double() * (1 - 0.02 * 0.1) - rate * o.view(-1)
        off = (got_w[s] - want).norm().item()
        allowed = rate * (_allowed(d, o) * 2) + 4 * 2.0 ** -24 * w[s].double().norm().item()
        assert off <= allowed, "%d x %d: %.3g against %.3g" % (r, c, off, allowed)
        # the bf16 copy is the rounded weight, whatever that is
        assert torch.equal(region.w16[s], region.w[s].bfloat16())
    assert torch.equal(got_w[~inside], w[~inside].double()) and torch.equal(got_buf[~inside], buf[~inside].double())
    assert torch.equal(got_w16[~inside], w.bfloat16()[~inside].double())


@pytest.mark.parametrize("nesterov", [True, False])
def test_step_over_short_matrices(nesterov):
    # all sides of at most 64: one launch an iteration
    places = [(0, 8, 1024), (8192, 64, 576), (45056, 500, 33), (61568, 7, 5), (61632, 64, 64)]
    total = 65792
    gen = torch.Generator().manual_seed(33)
    w, g, buf = (torch.randn(total, generator=gen) * s for s in (1.0, 1e-3, 1e-2))
    region = OptRegion("r", w.cuda(), g.cuda(), w.bfloat16().cuda(), True, places)
    opt = make_optimizer("muon", [region], 0.02, nesterov=nesterov, weight_decay=0.1)
    opt.buf["r"].copy_(buf)
    opt.step()
    m = 0.95 * buf.double() + g.double()
    u = g.double() + 0.95 * m if nesterov else m
    inside = torch.zeros(total, dtype=torch.bool)
    for at, r, c in places:
        s = slice(at, at + r * c)
        inside[s] = True
        d = u[s].view(r, c)
        o = ref.newton_schulz(d, 5)
        rate = 0.02 * math.sqrt(max(1, r / c))
        want = w[s].double() * (1 - 0.02 * 0.1) - rate * o.view(-1)
        off = (region.w[s].double().cpu() - want).norm().item()
        assert off <= rate * _allowed(d, o) * 2 + 4 * 2.0 ** -24 * w[s].double().norm().item(), (r, c)
        assert torch.equal(region.w16[s], region.w[s].bfloat16())
    assert torch.equal(region.w.cpu()[~inside], w[~inside])


def test_step_without_bf16_copy_and_with_vectors():
    w, g, _ = _buffers(torch.float32, 31)
    regions = [OptRegion("r", w.cuda(), g.cuda(), None, True, PLACES[:3], [(21568, 500)])]
    both = [make_optimizer("muon", [OptRegion("r", w.clone(), g.clone(), None, True, PLACES[:3], [(21568, 500)])], 0.02),
            make_optimizer("muon", regions, 0.02)]
    for opt in both:
        for _ in range(2):
            opt.step()
    a, b = both[0].regions[0].w, both[1].regions[0].w.cpu()
    # both sides fp32: matrices as far apart as the yardstick allows after two steps (rate 0.02, entries of about 0.1),
    # Adam's elementwise updates a few roundings
    assert (a[:21568] - b[:21568]).norm().item() <= 1e-5 * 0.02 * 30 + 8 * 2.0 ** -24 * w[:21568].norm().item()
    torch.testing.assert_close(a[21568:22068], b[21568:22068], rtol=1e-5, atol=1e-7)
    assert torch.equal(b[22068:], w[22068:])


def test_captured_step_replays():
    w, g, buf = _buffers(torch.float32, 32)

    def fresh():
        region = OptRegion("r", w.cuda(), g.cuda(), w.bfloat16().cuda(), True, PLACES)
        opt = make_optimizer("muon", [region], lambda t: 0.02 / (t + 1), weight_decay=0.01)
        opt.buf["r"].copy_(buf)
        return region, opt

    (ra, eager), (rb, opt) = fresh(), fresh()
    opt.prepare()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.launch()
    for k in range(3):
        new = torch.randn(TOTAL, generator=torch.Generator().manual_seed(40 + k)) * 1e-3
        ra.g.copy_(new)
        rb.g.copy_(new)
        eager.step()
        opt.prepare()
        graph.replay()
        opt.advance()
        torch.cuda.synchronize()
        assert torch.equal(ra.w, rb.w) and torch.equal(ra.w16, rb.w16) and torch.equal(eager.buf["r"], opt.buf["r"])


def test_muon_step_refusals():
    plan = ns.NsPlan([(0, 4, 8)], torch.device("cuda", 0))
    w = torch.zeros(32, device="cuda")
    hyper = torch.zeros(2, device="cuda")
    good = dict(w=w, buf=w.clone(), g=w.clone(), w16=None, hyper=hyper, mu=0.9, wd=0.0, nesterov=True, steps=5)
    for name, t in [("w", w.bfloat16()), ("buf", w[:16]), ("g", w.half()), ("g", w[::2]), ("w16", w), ("hyper", hyper[:1]),
                    ("w", w.cpu()), ("g", w.cpu()), ("steps", 0), ("steps", ns.MAX_STEPS + 1)]:
        with pytest.raises(ValueError):
            ns.muon_step(plan, **{**good, name: t})


@pytest.mark.parametrize("matrices", [[(0, 4, 8), (32, 1, 1)], [(1, 4, 8)], [(-1, 4, 8)]])
def test_a_plan_that_does_not_fit_its_buffers_is_refused(matrices):
    plan = ns.NsPlan(matrices, torch.device("cuda", 0))
    w = torch.zeros(32, device="cuda")
    with pytest.raises(ValueError, match="plan"):
        ns.muon_step(plan, w, w.clone(), w.clone(), None, torch.zeros(2, device="cuda"), 0.9, 0.0, True, 5)


def test_model_trains_with_muon_and_matches_the_cpu():
    # one step of the head alone in both: features and labels are the same, the head's gradients agree to bf16 accuracy,
    # but an orthogonalised update turns every singular direction to size 1, noise included -- so what is compared are the
    # properties the update must have: its singular values and its alignment with the momentum
    torch.manual_seed(1)
    model = build_model("flower_cnn", 5, device="cuda", dropout_rate=0.0).train()
    engine = DataParallelEngine(model, mode="sync_dp", optimizer="muon", lr=0.02, opt_kwargs={"momentum": 0.9, "nesterov": False})
    x = torch.zeros(16, 64, 64, 8)
    x[..., :3] = torch.randn(16, 64, 64, 3, generator=torch.Generator().manual_seed(2))
    x, y = x.cuda().bfloat16(), torch.arange(16, device="cuda", dtype=torch.int32) % 5
    before = {g.name: g.master.clone() for g in engine.flat.groups}
    engine.begin_step()
    logits, reg = model(x)
    loss, _, _, _ = F.softmax_xent(logits, y, 5)
    (loss + reg).backward()
    engine.finish_step()
    torch.cuda.synchronize()
    for region in engine.optimizer.regions:
        moved = (before[region.name] - region.w).double().cpu()
        for at, r, c in region.matrices:
            s = slice(at, at + r * c)
            rate = 0.02 * math.sqrt(max(1, r / c))
            got = moved[s].view(r, c) / rate
            u = engine.optimizer.buf[region.name][s].view(r, c)
            want = ref.newton_schulz(u.double().cpu(), 5)
            # the weights' own rounding, 2^-24 of values below 1, divided by the rate
            slack = 2.0 ** -24 * math.sqrt(r * c) / rate * 2
            assert (got - want).norm().item() <= _allowed(u, want) + slack, (r, c)
        for at, n in region.vectors:
            assert moved[at:at + n].abs().max().item() > 0


@pytest.mark.parametrize("mode,kw", [("sync_dp", {}), ("async_ssp", {"staleness": 1})])
def test_step_graph_with_a_normalised_head_matches_eager(mode, kw):
    # layer normalisation, its gradients into the flat buffers and the Muon step together, eager and replayed
    from distributed_tensorflow_amd.train.session import TrainingSession

    def run(hip_graph):
        torch.manual_seed(9)
        model = build_model("flower_cnn", 5, device="cuda", dropout_rate=0.0, head_norm="layer")
        eng = DataParallelEngine(model, mode=mode, optimizer="muon", lr=lambda t: 0.02 / (1 + t), opt_kwargs={"weight_decay": 0.01},
                                 **kw)
        sess = TrainingSession(model, eng, num_classes=5, hip_graph=hip_graph, graph_warmup_steps=2)
        gen = torch.Generator().manual_seed(4)
        losses = []
        for _ in range(6):
            x = torch.zeros(8, 64, 64, 8)
            x[..., :3] = torch.rand(8, 64, 64, 3, generator=gen) * 2 - 1
            y = torch.randint(0, 5, (8,), generator=gen, dtype=torch.int32)
            losses.append(sess.run_step(x.cuda().bfloat16(), y.cuda()).loss)
        assert (sess._graph is not None) == (hip_graph and eng.graph_capturable)
        assert not torch.equal(model.head.feature_norm.gamma, torch.ones_like(model.head.feature_norm.gamma))
        return losses, [g.master.clone() for g in eng.flat.groups]

    (l0, w0), (l1, w1) = run(False), run(True)
    assert l0 == l1 and all(math.isfinite(l) for l in l0)
    for a, b in zip(w0, w1):
        assert torch.equal(a, b)
