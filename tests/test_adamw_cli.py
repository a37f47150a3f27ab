"""main_moco.py with AdamW: pretraining, resuming, and what it refuses."""

import os
import subprocess
import sys

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, *more):
    return subprocess.run(
        [sys.executable, "main_moco.py", "synthetic", "-a", "resnet18",
         "--moco-k", "32", "--crop-size", "32", "--load-size", "40", "-b",
         "8", "-j", "0", "--max-steps-per-epoch", "2", "--synthetic-len",
         "16", "--device", "cpu", "--save-dir", str(tmp_path), "-p", "1",
         "--lr", "1e-3", *more],
        cwd=REPO, timeout=600, capture_output=True, text=True)


@pytest.mark.parametrize("kind", ["adamw", "adamw8bit"])
def test_pretrain_and_resume(tmp_path, kind):
    r = run(tmp_path, "--optimizer", kind, "--clip-grad", "1.0",
            "--epochs", "1")
    assert r.returncode == 0, r.stderr
    path = tmp_path / "checkpoint_0000.pth.tar"
    state = torch.load(path, map_location="cpu",
                       weights_only=True)["optimizer"]["state"]
    want = torch.float8_e4m3fn if kind == "adamw8bit" else torch.float32
    assert state and all(s["exp_avg"].dtype == want and s["step"] == 2
                         for s in state.values())
    r = run(tmp_path, "--optimizer", kind, "--epochs", "2", "--resume",
            str(path))
    assert r.returncode == 0, r.stderr
    state = torch.load(tmp_path / "checkpoint_0001.pth.tar",
                       map_location="cpu",
                       weights_only=True)["optimizer"]["state"]
    assert all(s["step"] == 4 for s in state.values())


def test_clip_needs_adamw(tmp_path):
    r = run(tmp_path, "--clip-grad", "1.0", "--epochs", "1")
    assert r.returncode == 2 and "--clip-grad" in r.stderr
