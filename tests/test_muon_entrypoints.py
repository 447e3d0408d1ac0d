"""The distributed trainer with the Muon optimizer and the layer-normalised head: two ranks, checkpoint, export."""
import glob
import json
import os
import socket
import subprocess
import sys

import numpy as np

from distributed_tensorflow_amd.io import bundle
from distributed_tensorflow_amd.io.export import Servable

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DIST = os.path.join(ROOT, "recognition_flower", "distributed")


def _port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def test_two_workers_train_with_muon_and_the_export_knows_its_head(tmp_path):
    cluster = {"worker": ["localhost:%d" % _port(), "localhost:%d" % _port()]}
    cmd = ["train_dataset.py", "--synthetic", "--mode=sync_dp", "--optimizer=muon", "--learning_rate=0.02", "--momentum=0.95",
           "--weight_decay=0.01", "--head_norm=layer", "--model=flower_cnn", "--train_steps=4", "--batch_size=4", "--image_size=32",
           "--checkpoint_dir=%s/ckpt/" % tmp_path, "--summaries_dir=%s/events/" % tmp_path, "--device=cpu"]
    procs = []
    for i in range(2):
        env = dict(os.environ, TF_CONFIG=json.dumps({"cluster": cluster, "task": {"type": "worker", "index": i}}))
        procs.append(subprocess.Popen([sys.executable] + cmd, cwd=DIST, env=env, stdout=subprocess.PIPE,
                                      stderr=subprocess.STDOUT, text=True))
    outs = [p.communicate(timeout=240)[0] for p in procs]
    assert [p.returncode for p in procs] == [0, 0], outs
    saved = bundle.read_bundle(bundle.latest_checkpoint(str(tmp_path / "ckpt")))
    assert int(saved["global_step"]) == 4 and "fc_trainable/feature_norm/gamma/Adam" in saved
    assert np.abs(saved["FlowerCNN/conv3/weights/Momentum"]).max() > 0
    labels = tmp_path / "labels.json"   # the trainer's synthetic input has five classes
    labels.write_text(json.dumps({"classes": list("abcde")}))
    env = dict(os.environ)
    env.pop("TF_CONFIG", None)
    r = subprocess.run([sys.executable, "save_model.py", "--model=flower_cnn", "--image_size=32", "--device=cpu",
                        "--dataset_path=%s/none" % tmp_path, "--labels_json=%s" % labels, "--checkpoint_dir=%s/ckpt/" % tmp_path, "--output_dir=%s/models" % tmp_path],
                       cwd=DIST, env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=240)
    assert r.returncode == 0, r.stdout
    (path,) = glob.glob(str(tmp_path / "models" / "*"))
    served = Servable(path, device="cpu").model
    assert np.array_equal(served.head.feature_norm.gamma.detach().numpy(), saved["fc_trainable/feature_norm/gamma"])


def test_modes_that_cut_matrices_end_at_once(tmp_path):
    for mode, task in (("async_ps", {"type": "ps", "index": 0}), ("sharded_ps", {"type": "worker", "index": 0})):
        cluster = {"ps": ["localhost:%d" % _port()], "worker": ["localhost:%d" % _port()]}
        env = dict(os.environ, TF_CONFIG=json.dumps({"cluster": cluster, "task": task}))
        r = subprocess.run([sys.executable, "train_dataset.py", "--synthetic", "--mode=" + mode, "--optimizer=muon",
                            "--checkpoint_dir=%s/ckpt/" % tmp_path, "--device=cpu"], cwd=DIST, env=env,
                           stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
        assert r.returncode != 0 and "whole matrices" in r.stdout, r.stdout


def test_an_unknown_head_norm_ends_every_task_at_once(tmp_path):
    cluster = {"ps": ["localhost:%d" % _port()], "worker": ["localhost:%d" % _port()]}
    for task in ("ps", "worker"):
        env = dict(os.environ, TF_CONFIG=json.dumps({"cluster": cluster, "task": {"type": task, "index": 0}}))
        r = subprocess.run([sys.executable, "train_dataset.py", "--synthetic", "--mode=async_ps", "--head_norm=batch",
                            "--checkpoint_dir=%s/ckpt/" % tmp_path, "--device=cpu"], cwd=DIST, env=env,
                           stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
        assert r.returncode != 0 and "head_norm" in r.stdout, r.stdout
