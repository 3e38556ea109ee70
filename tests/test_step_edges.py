"""What the training step's operators get wrong most easily (tests/step_edges.py): on the GPU, and on the CPU model of the
library under AddressSanitizer and UBSan (tests/test_kernel_model.py describes it)."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

import pytest

import step_edges

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "model")
sys.path.insert(0, HERE)
import run  # noqa: E402

EDGES = sorted(step_edges.EDGES)


@pytest.mark.gpu
@pytest.mark.parametrize("name", EDGES)
def test_on_the_gpu(name):
    step_edges.EDGES[name]("cuda")


@pytest.fixture(scope="module")
def model():
    return run.build()


@pytest.mark.skipif(not os.path.exists(run.CLANG) or shutil.which("make") is None,
                    reason="needs ROCm's clang++ (host build with AddressSanitizer)")
@pytest.mark.parametrize("name", EDGES)
def test_on_the_cpu_model(model, name):
    r = subprocess.run([sys.executable, os.path.join(HERE, "run_step_edges.py"), name], env=run.env(model), capture_output=True,
                       text=True, timeout=900)
    assert r.returncode == 0, (r.stdout[-2000:], r.stderr[-6000:])
    assert f"{name}: held" in r.stdout
