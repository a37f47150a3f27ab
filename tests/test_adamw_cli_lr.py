"""main_moco.py: the learning rate's default is SGD's, and AdamW says so."""

import os
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("options,warns", [
    (["--optimizer", "adamw"], True), (["--optimizer", "adamw8bit"], True),
    (["--optimizer", "adamw", "--lr", "1e-3"], False), ([], False)])
def test_default_learning_rate(tmp_path, options, warns):
    r = subprocess.run(
        [sys.executable, "main_moco.py", "synthetic", "-a", "resnet18",
         "--moco-k", "32", "-b", "8", "-j", "0", "--epochs", "0",
         "--synthetic-len", "16", "--device", "cpu", "--save-dir",
         str(tmp_path), *options],
        cwd=REPO, timeout=600, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert ("--lr 0.03 is SGD's default" in r.stderr) == warns
