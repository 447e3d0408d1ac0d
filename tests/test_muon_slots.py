"""Which optimizer slots a checkpoint of a Muon run holds."""
import pytest
import torch

from distributed_tensorflow_amd.io import bundle
from distributed_tensorflow_amd.io.saver import Saver
from distributed_tensorflow_amd.models import build_model
from distributed_tensorflow_amd.ops import functional as F
from distributed_tensorflow_amd.parallel.engine import DataParallelEngine

MATRICES = ["FlowerCNN/conv%d/weights" % k for k in range(1, 6)] + ["fc_trainable/dense_prelogit1/kernel",
                                                                    "fc_trainable/flower_logits/kernel"]


def _run(optimizer, seed, device="cpu"):
    torch.manual_seed(seed)
    model = build_model("flower_cnn", 5, device=torch.device(device), widths=(8, 8, 16, 16, 24), dropout_rate=0.0).train()
    engine = DataParallelEngine(model, mode="sync_dp", optimizer=optimizer, lr=0.02)
    return model, engine, Saver(model, engine)


def _train(model, engine, device="cpu", steps=2):
    x = torch.zeros(2, 32, 32, 8)
    x[..., :3] = torch.randn(2, 32, 32, 3, generator=torch.Generator().manual_seed(6))
    x = x.to(device=device, dtype=torch.bfloat16 if device == "cuda" else torch.float32)
    for _ in range(steps):
        engine.begin_step()
        loss, _, _, _ = F.softmax_xent(model(x)[0], torch.tensor([1, 2], dtype=torch.int32, device=device), 5)
        loss.backward()
        engine.finish_step()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_kernels_have_momentum_and_vectors_have_adam(device):
    # (one flat buffer for everything on the CPU, one for the bf16 kernels and one for the rest on the GPU)
    model, engine, saver = _run("muon", 1, device)
    _train(model, engine, device)
    names = set(saver.variables())
    plain = set(saver.variables(include_slots=False))
    trained = {v.name for v in saver.specs if v.trainable}
    want = {n + "/Momentum" for n in MATRICES} | {n + s for n in trained - set(MATRICES) for s in ("/Adam", "/Adam_1")}
    assert set(MATRICES) <= trained and names - plain == want


def test_what_was_saved_comes_back(tmp_path):
    model, engine, saver = _run("muon", 1)
    _train(model, engine)
    prefix = saver.save(str(tmp_path), 2)
    other, engine2, saver2 = _run("muon", 2)
    assert saver2.restore(prefix) == 2
    for (k, a), b in zip(engine.optimizer.slots().items(), engine2.optimizer.slots().values()):
        assert torch.equal(a, b), k
    _train(model, engine, steps=1)
    _train(other, engine2, steps=1)
    for p, q in zip(model.parameters(), other.parameters()):
        assert torch.equal(p, q)


def test_moments_of_another_optimizer_are_not_taken_for_kernels(tmp_path):
    model, engine, saver = _run("adam", 1)
    _train(model, engine)
    prefix = saver.save(str(tmp_path), 2)
    assert "FlowerCNN/conv2/weights/Adam" in bundle.read_bundle(prefix)
    other, engine2, saver2 = _run("muon", 2)
    saver2.restore(prefix)
    (m,) = engine2.optimizer.m.values()
    (region,) = engine2.optimizer.regions
    assert m.any() and not any(m[at:at + r * c].any() for at, r, c in region.matrices)
