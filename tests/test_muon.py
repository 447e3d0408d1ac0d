"""Orthogonalisation and the Muon optimizer on the CPU: oracle, plans, regions, engines, checkpoints, refusals."""
import math

import numpy as np
import pytest
import torch
import torch.nn as nn

from distributed_tensorflow_amd.io.saver import Saver
from distributed_tensorflow_amd.models import build_model
from distributed_tensorflow_amd.ops import functional as F
from distributed_tensorflow_amd.ops import newton_schulz as ns
from distributed_tensorflow_amd.optim import FusedMuon, OptRegion, make_optimizer, regions_from_flat
from distributed_tensorflow_amd.parallel.engine import DataParallelEngine
from distributed_tensorflow_amd.parallel.flat import FlatParams


def _by_singular_values(g, steps=5):
    u, s, vt = torch.linalg.svd(g, full_matrices=False)
    s = s / (s.square().sum().sqrt() + 1e-7)
    for _ in range(steps):
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    return (u * s) @ vt


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 9), (9, 1), (6, 6), (5, 40), (40, 5)])
def test_oracle_maps_the_singular_values(rows, cols):
    g = torch.randn(2, rows, cols, dtype=torch.float64, generator=torch.Generator().manual_seed(rows + 7 * cols))
    got = F.orthogonalize(g)
    for a, b in zip(got, g):
        torch.testing.assert_close(a, _by_singular_values(b), rtol=1e-9, atol=1e-9)


def test_result_does_not_depend_on_scale_and_zero_stays_zero():
    g = torch.randn(12, 30, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    torch.testing.assert_close(F.orthogonalize(g * 1e6), F.orthogonalize(g), rtol=1e-6, atol=1e-6)
    assert not F.orthogonalize(torch.zeros(4, 4)).any()
    assert F.orthogonalize(torch.zeros(0, 4, 4)).shape == (0, 4, 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dtype_and_layout_are_kept(dtype):
    g = torch.randn(30, 8, generator=torch.Generator().manual_seed(2)).to(dtype)
    o = F.orthogonalize(g.t())
    assert o.dtype == dtype and o.shape == (8, 30) and o.is_contiguous()
    # one rounding of values of at most 1.21, and 1e-4 for fp32 arithmetic amplified over five iterations
    torch.testing.assert_close(o.double(), _by_singular_values(g.t().double()), rtol=torch.finfo(dtype).eps / 2 + 1e-4,
                               atol=1e-4)


def test_refusals():
    x = torch.randn(4, 8)
    for bad in [lambda: F.orthogonalize(x[0]), lambda: F.orthogonalize(x, steps=0), lambda: F.orthogonalize(x, steps=2.0),
                lambda: F.orthogonalize(x, steps=65), lambda: F.orthogonalize(x, steps=True),
                lambda: F.orthogonalize(x[:, :0]), lambda: F.orthogonalize(x[:0]), lambda: F.orthogonalize(x.int()),
                lambda: F.orthogonalize(torch.nn.Parameter(x)), lambda: ns.orthogonalize(x, 5),
                lambda: F.orthogonalize(torch.empty(1, 1).expand(1, (1 << 20) + 1)),
                lambda: F.orthogonalize(torch.empty(1, 1).expand(40000, 40000))]:
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        F.orthogonalize(torch.nn.Parameter(x))


@pytest.mark.parametrize("shapes", [[(64, 64), (65, 80)], [(5, 700), (700, 5), (513, 2000), (1031, 600)],
                                    [(2048, 512), (64, 64), (1000, 2048)], [(4096, 4096)], [(4700, 3900)],
                                    [(256, 2304)] * 6])
def test_plan_covers_every_tile_once_and_stays_inside(shapes):
    places, at = [], 0
    for r, c in shapes:
        places.append((at, r, c))
        at += r * c + 3
    plan = ns.NsPlan(places, "cpu")
    table, base = plan.table.numpy(), plan.table.data_ptr()
    mats = table[:len(shapes) * ns._MAT.itemsize].view(ns._MAT)
    lists = []
    counts = plan.counts[2:] + plan.counts[:1]
    for start, count, width in zip(plan.places[1:], counts, (4, 4, 8, 8, 8, 8, 8, 8)):
        assert (start - base) % 32 == 0 and start - base + 4 * width * count <= table.size
        lists.append(table[start - base:start - base + 4 * width * count].view(np.int32).reshape(-1, width))
    chunks, packs, gram, gram_joins, poly, poly_joins, full, small = lists
    assert not len(small)
    end = part = 0
    slabs = {id(gram): [], id(poly): [], id(full): []}   # (first, length) of every tile's slabs
    for k, (m, (at, r, c)) in enumerate(zip(mats, places)):
        edge = 128 if any((t[t[:, 0] == k][:, 3] == 128).any() for t in (gram, poly, full)) else 64
        assert (m["at"], m["rows"], m["cols"], m["tall"]) == (at, r, c, r > c)
        for padded, size in ((m["rp"], r), (m["cp"], c), (m["mp"], min(r, c))):
            assert size <= padded < size + edge and padded % edge == 0
        # planes follow one another without overlap
        assert m["x"] == end and m["a"] == end + 4 * m["rp"] * m["cp"] and m["x"] % 8 == 0 and m["a"] % 8 == 0
        end = m["a"] + 4 * m["mp"] * m["mp"]
        assert m["part"] == part and m["parts"] == -(-r * c // m["chunk"]) <= ns.MAX_PARTS
        part += m["parts"]
        assert sorted(map(tuple, chunks[chunks[:, 0] == k][:, 1:2])) == [(i,) for i in range(m["parts"])]
        assert {tuple(t) for t in packs[packs[:, 0] == k][:, 1:3]} == \
            {(i, j) for i in range(m["rp"] // 64) for j in range(m["cp"] // 64)}
        for jobs, longest, lower in ((gram, max(m["rp"], m["cp"]), True), (poly, m["mp"], True), (full, m["mp"], False)):
            seen = np.zeros((m["mp"], m["mp"]) if lower else (m["rp"], m["cp"]), dtype=np.int64)
            pieces = {}
            for _, ti, tj, e, k0, k1, slab, _ in jobs[jobs[:, 0] == k]:
                assert e in (64, edge) and 0 <= k0 < k1 <= longest and k0 % 32 == k1 % 32 == 0
                assert e * (ti + 1) <= seen.shape[0] and e * (tj + 1) <= seen.shape[1] and ti >= 0 <= tj
                seen[e * ti:e * (ti + 1), e * tj:e * (tj + 1)] += k1 - k0
                if lower and ti != tj:   # the mirror image
                    seen[e * tj:e * (tj + 1), e * ti:e * (ti + 1)] += k1 - k0
                assert (slab >= 0) == (k1 - k0 < longest)
                pieces.setdefault((ti, tj, e), []).append((k0, k1, slab))
            joins = {tuple(t[1:4]): (t[4], t[6]) for t in (gram_joins if jobs is gram else poly_joins) if t[0] == k} \
                if lower else {}
            assert set(joins) == {t for t, v in pieces.items() if len(v) > 1}
            for tile, v in pieces.items():   # the pieces follow one another, and so do their slabs
                v.sort()
                assert v[0][0] == 0 and v[-1][1] == longest and all(a[1] == b[0] for a, b in zip(v, v[1:]))
                if len(v) > 1:
                    unit = (tile[2] // 64) ** 2
                    assert joins[tile] == (len(v), v[0][2])
                    assert [s for _, _, s in v] == [v[0][2] + i * unit for i in range(len(v))]
                    slabs[id(jobs)] += [v[0][2], len(v) * unit]
            assert (seen == longest).all()
        # the scale: a power of two, no entry of X (at most 1.21) above fp16's range
        assert math.log2(m["scale"]) == int(math.log2(m["scale"])) and 1.21 * m["scale"] < 65504
        assert m["scale"] <= math.sqrt(r * c) < 2 * m["scale"] or m["scale"] == 2 ** 15
    assert plan.ws_elems == end and plan.parts == part
    for v in slabs.values():
        places = sorted(zip(v[::2], v[1::2]))
        assert all(a + n == b for (a, n), (b, _) in zip(places, places[1:])) and (not places or places[0][0] == 0)
        assert not places or sum(places[-1]) <= plan.slabs


@pytest.mark.parametrize("shapes", [[(1, 1)], [(64, 576)] * 3, [(5, 700), (700, 5), (64, 64), (33, 8192)]])
def test_short_sides_are_sliced_completely(shapes):
    places, at = [], 0
    for r, c in shapes:
        places.append((at, r, c))
        at += r * c
    plan = ns.NsPlan(places, "cpu")
    table, base = plan.table.numpy(), plan.table.data_ptr()
    mats = table[:len(shapes) * ns._MAT.itemsize].view(ns._MAT)
    nsmall, slices = plan.counts[:2]
    assert nsmall == slices and plan.counts[3:] == [0] * 6 and plan.slabs == 2 * slices
    start = plan.places[8] - base
    jobs = table[start:start + 32 * nsmall].view(np.int32).reshape(-1, 8)
    slab = 0
    for k, m in enumerate(mats):
        mine = jobs[jobs[:, 0] == k]
        blocks = max(m["rp"], m["cp"]) // 64
        assert min(m["rp"], m["cp"]) == m["mp"] == 64
        # {matrix, slice, first block, blocks, slices, -, first slab, -}: slice after slice, block after block
        assert list(mine[:, 1]) == list(range(len(mine))) and (mine[:, 3] >= 1).all() and (mine[:, 4] == len(mine)).all()
        assert mine[0, 2] == 0 and (mine[1:, 2] == mine[:-1, 2] + mine[:-1, 3]).all() and mine[-1, 2] + mine[-1, 3] == blocks
        assert (mine[:, 6] == slab).all()
        slab += len(mine)
    assert slab == slices


def _model():
    torch.manual_seed(3)
    return build_model("flower_cnn", 5, widths=(8, 8, 16, 16, 24), dropout_rate=0.0)


def test_regions_of_a_model_say_where_its_matrices_are():
    model = _model()
    flat = FlatParams(model)
    (region,) = regions_from_flat(flat)
    inside = torch.zeros(region.w.numel(), dtype=torch.int64)
    for at, r, c in region.matrices:
        inside[at:at + r * c] += 1
    for at, n in region.vectors:
        inside[at:at + n] += 2
    for seg in flat.groups[0].segments:
        want = 1 if seg.param.dim() > 1 else 2
        assert (inside[seg.offset:seg.offset + seg.numel] == want).all()
        if want == 1:
            assert (seg.offset, seg.param.shape[0], seg.numel // seg.param.shape[0]) in region.matrices
    assert not region.w[inside == 0].any() and inside.max() == 2


@pytest.mark.parametrize("nesterov", [True, False])
def test_step_follows_the_formulas(nesterov):
    gen = torch.Generator().manual_seed(4)
    w = torch.randn(400, generator=gen)
    g = torch.randn(400, generator=gen)
    places, vectors = [(0, 6, 20), (128, 20, 4)], [(256, 30)]
    opt = make_optimizer("muon", [OptRegion("r", w.clone(), g.clone(), None, True, places, vectors)], 0.02, momentum=0.9,
                         nesterov=nesterov, weight_decay=0.1, vector_lr_scale=0.5)
    assert isinstance(opt, FusedMuon)
    ref, buf = w.double().clone(), torch.zeros(400, dtype=torch.float64)
    m = v = torch.zeros(30, dtype=torch.float64)
    for t in range(1, 4):
        opt.step(grad_scale=0.5)
        gd = g.double() * 0.5
        buf = 0.9 * buf + gd
        u = gd + 0.9 * buf if nesterov else buf
        for at, r, c in places:
            s = slice(at, at + r * c)
            ref[s] = ref[s] * (1 - 0.02 * 0.1) - 0.02 * max(1, r / c) ** 0.5 * _by_singular_values(u[s].view(r, c)).view(-1)
        m, v = 0.9 * m + 0.1 * gd[256:286], 0.999 * v + 0.001 * gd[256:286] ** 2
        ref[256:286] -= 0.01 * math.sqrt(1 - 0.999 ** t) / (1 - 0.9 ** t) * m / (v.sqrt() + 1e-8)
    got = opt.regions[0].w.double()
    torch.testing.assert_close(got, ref, rtol=1e-5, atol=1e-5)
    assert torch.equal(got[286:], w[286:].double()) and torch.equal(got[120:128], w[120:128].double())


def test_optimizer_refusals():
    w, g = torch.zeros(100), torch.zeros(100)
    for kw in [dict(matrices=None), dict(matrices=[(0, 10, 11)]), dict(matrices=[(0, 5, 10), (49, 2, 2)]),
               dict(matrices=[(0, 5, 10)], vectors=[(40, 20)]), dict(matrices=[(-1, 2, 2)]), dict(matrices=[(0, 0, 4)]),
               dict(matrices=[], vectors=[(99, 2)])]:
        with pytest.raises(ValueError):
            make_optimizer("muon", [OptRegion("r", w, g, None, True, **kw)], 0.02)
    with pytest.raises(ValueError):
        make_optimizer("muon", [OptRegion("r", w, g, None, True, [(0, 10, 10)])], 0.02, ns_steps=0)
    with pytest.raises(ValueError):
        DataParallelEngine(_model(), mode="sharded_ps", optimizer="muon", lr=0.02)


@pytest.mark.parametrize("mode,kw", [("sync_dp", {}), ("async_ssp", {"staleness": 1})])
def test_training_steps_update_every_parameter(mode, kw):
    model = _model().train()
    engine = DataParallelEngine(model, mode=mode, optimizer="muon", lr=0.02, opt_kwargs={"weight_decay": 0.01}, **kw)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    x = torch.zeros(4, 32, 32, 8)
    x[..., :3] = torch.randn(4, 32, 32, 3, generator=torch.Generator().manual_seed(5))
    y = torch.tensor([0, 1, 2, 3])
    for _ in range(3):
        engine.begin_step()
        logits, reg = model(x)
        loss, _, _, _ = F.softmax_xent(logits, y, 5)
        (loss + reg).backward()
        engine.finish_step()
    engine.drain()
    for n, p in model.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n
    # padding rows and channels have no gradient and stay what they were
    assert not model.head.flower_logits.weight[5:].any() and not model.conv1.weight[..., 3:].any()


def test_checkpoint_round_trip(tmp_path):
    def run(seed, restore=None):
        torch.manual_seed(seed)
        model = build_model("flower_cnn", 5, widths=(8, 8, 16, 16, 24), dropout_rate=0.0).train()
        engine = DataParallelEngine(model, mode="sync_dp", optimizer="muon", lr=0.02)
        saver = Saver(model, engine)
        if restore:
            assert saver.restore(restore) == 2
        return model, engine, saver

    def train(model, engine, n):
        x = torch.zeros(2, 32, 32, 8)   # the channels behind the three colours are zeros, as everywhere
        x[..., :3] = torch.randn(2, 32, 32, 3, generator=torch.Generator().manual_seed(6))
        for _ in range(n):
            engine.begin_step()
            loss, _, _, _ = F.softmax_xent(model(x)[0], torch.tensor([1, 2]), 5)
            loss.backward()
            engine.finish_step()

    model, engine, saver = run(1)
    train(model, engine, 2)
    prefix = saver.save(str(tmp_path), 2)
    names = saver.variables()
    assert "FlowerCNN/conv2/weights/Momentum" in names and "FlowerCNN/conv2/BatchNorm/beta/Adam_1" in names
    other, engine2, _ = run(2, restore=prefix)
    for a, b in zip(engine.optimizer.slots().values(), engine2.optimizer.slots().values()):
        assert torch.equal(a, b)
    train(model, engine, 1)
    train(other, engine2, 1)
    for (n, p), q in zip(model.named_parameters(), other.parameters()):
        assert torch.equal(p, q), n


def test_head_with_feature_norm_trains_and_exports_under_its_own_names(tmp_path):
    from distributed_tensorflow_amd.io.export import Servable, export_servable

    torch.manual_seed(7)
    kw = dict(widths=(8, 8, 16, 16, 24), dropout_rate=0.0, head_norm="layer")
    model = build_model("flower_cnn", 5, **kw).train()
    engine = DataParallelEngine(model, mode="sync_dp", optimizer="muon", lr=0.02)
    saver = Saver(model, engine)
    x = torch.zeros(4, 32, 32, 8)
    x[..., :3] = torch.randn(4, 32, 32, 3, generator=torch.Generator().manual_seed(8))
    for _ in range(2):
        engine.begin_step()
        logits, reg = model(x)
        (F.softmax_xent(logits, torch.tensor([0, 1, 2, 3]), 5)[0] + reg).backward()
        engine.finish_step()
    assert not torch.equal(model.head.feature_norm.gamma, torch.ones(24))
    names = saver.variables()
    assert {"fc_trainable/feature_norm/gamma", "fc_trainable/feature_norm/beta/Adam",
            "fc_trainable/dense_prelogit1/kernel/Momentum"} <= set(names)
    path = export_servable(model, list("abcde"), str(tmp_path), 1, model_name="flower_cnn", image_size=32, model_kwargs=kw,
                           engine=engine)
    served = Servable(path, device="cpu").model
    model.eval()
    with torch.no_grad():
        torch.testing.assert_close(served(x)[0], model(x)[0], rtol=1e-5, atol=1e-5)
    with pytest.raises(ValueError):
        build_model("flower_cnn", 5, head_norm="batch")


def test_parameter_servers_refuse_muon():
    from distributed_tensorflow_amd.parallel.ps import PSWorkerEngine

    with pytest.raises(ValueError, match="muon"):
        PSWorkerEngine(_model(), [("127.0.0.1", 1)], 0, True, optimizer="muon")
