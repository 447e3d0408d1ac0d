"""Large batches of orthogonalisations: bounded workspaces, plans by shape and not matrix by matrix."""
import pytest
import torch

from distributed_tensorflow_amd.ops import functional as F
from distributed_tensorflow_amd.ops import newton_schulz as ns
from distributed_tensorflow_amd.ops import ref

SHAPES = [(8, 8), (64, 64), (64, 8192), (8192, 64), (65, 65), (100, 20000), (70, 100000), (256, 2304), (300, 300), (1000, 1000),
          (2000, 2000), (64, 9000)]


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_a_group_stays_within_its_bytes(rows, cols):
    many = ns._group(rows, cols)
    plan = ns.NsPlan([(i * rows * cols, rows, cols) for i in range(many)], "cpu")
    assert many >= 2 and plan.ws_elems * 2 + plan.slabs * 4096 * 4 <= 1.1 * ns.GROUP_BYTES


def test_a_matrix_larger_than_a_group_goes_by_itself():
    assert ns._group(20000, 20000) == 1 and ns._group(1 << 20, 1 << 15) == 1


@pytest.mark.parametrize("shapes", [[(8, 8)] * 40, [(70, 90)] * 7, [(70, 90), (300, 200), (70, 90), (70, 90)], [(640, 9000)] * 3])
def test_a_run_of_one_shape_is_its_matrices_one_by_one(shapes):
    # the run's places and chunks against those of matrices told apart by a shape in between
    places, at = [], 0
    for r, c in shapes:
        places.append((at, r, c))
        at += r * c + 5
    plan = ns.NsPlan(places, "cpu")
    mats = plan.table.numpy()[:len(shapes) * ns._MAT.itemsize].view(ns._MAT)
    ws = part = 0
    for m, (at, r, c) in zip(mats, places):
        assert (m["at"], m["rows"], m["cols"], m["x"], m["part"]) == (at, r, c, ws, part)
        assert m["a"] == ws + 4 * m["rp"] * m["cp"]
        ws = m["a"] + 4 * m["mp"] * m["mp"]
        part += m["parts"]
    assert (plan.ws_elems, plan.parts) == (ws, part)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols", [(20000, 8, 8), (6000, 16, 40), (900, 70, 90), (40, 64, 8192), (30, 700, 1000)])
def test_more_than_a_group(monkeypatch, batch, rows, cols):
    monkeypatch.setattr(ns, "GROUP_BYTES", 256 << 20)
    assert batch > ns._group(rows, cols)
    g = torch.randn(batch, rows, cols, generator=torch.Generator(device="cuda").manual_seed(batch), device="cuda")
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = F.orthogonalize(g)
    torch.cuda.synchronize()
    # the workspace of one group next to the result, and what the allocator rounds up
    assert torch.cuda.max_memory_allocated() - before <= out.numel() * 4 + 1.2 * ns.GROUP_BYTES + (16 << 20)
    groups = -(-batch // ns._group(rows, cols))
    edges = [k * batch // groups for k in range(groups)]
    picked = sorted({0, 1, edges[1] - 1, edges[1], edges[1] + 1, edges[-1] - 1, edges[-1], batch - 1})
    for k in picked:
        want = ref.newton_schulz(g[k].double().cpu())
        fp32 = (ref.newton_schulz(g[k].cpu()).double() - want).norm().item()
        off = (out[k].cpu().double() - want).norm().item()
        # as for single matrices: three times fp32's error and the roundings of the last two iterations
        assert off <= 3 * fp32 + 5 * 2.0 ** -23 * want.norm().item(), k
    # every matrix has singular values near one, so none was left out or written twice over another
    want = ref.newton_schulz(g)
    off = (out - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
    assert off.max().item() < 1e-3   # (two fp32 iterations may part by their errors, amplified: some 1e-5 at worst)


@pytest.mark.gpu
def test_groups_are_captured_and_replayed(monkeypatch):
    monkeypatch.setattr(ns, "GROUP_BYTES", 1 << 20)
    assert 1 <= ns._group(70, 90) < 7
    g = torch.randn(7, 70, 90, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    assert -(-7 // ns._group(70, 90)) > 1
    F.orthogonalize(g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.orthogonalize(g)
    for seed in (2, 3, 4):
        g.copy_(torch.randn(7, 70, 90, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
        graph.replay()
        eager = F.orthogonalize(g)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
