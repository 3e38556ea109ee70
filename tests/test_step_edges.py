"""What the training step's operators get wrong most easily (tests/step_edges.py): on the GPU, and on the CPU model of the
library under AddressSanitizer and UBSan (tests/test_kernel_model.py describes it)."""

from __future__ import annotations

import ctypes
import os
import shutil
import subprocess
import sys

import pytest

import step_edges
from crukx_sync import _native
from crukx_sync._native import AdamW, Logits, Policy, Positions

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


def test_the_c_interface_refuses_misaligned_data():
    """On any host: nothing is launched for these, whatever the addresses point to."""
    L, err = _native.lib(), _native.errbuf()
    buf = (ctypes.c_double * 64)()
    at = ctypes.addressof(buf)
    none, pos = Positions(None, 0, 0), Positions(at, 2, 1)
    x = Logits(at, 1, 2, 4, 8, 4, 2, 8, pos, none, 1.0)
    off = Positions(at + 2, 2, 1)

    def scores(logp=at, entropy=at, stats=at, scratch=at):
        return L.crx_token_logprobs(ctypes.byref(x), logp, entropy, stats, scratch, None, err, 512)

    def scores_grad(stats=at, entropy=at, up=pos, up_entropy=pos, grad=at):
        return L.crx_token_logprobs_grad(ctypes.byref(x), stats, entropy, ctypes.byref(up), ctypes.byref(up_entropy), grad, None, err, 512)

    def loss(old=pos, adv=pos, ref=pos, loss=at, kl=at, clipped=at, logp=at, stats=at, slope=at, grad=at, scratch=at):
        p = Policy(old, adv, ref, 0.2, 0.2, 0.0, 1.0, 0)
        return L.crx_policy_loss(ctypes.byref(x), ctypes.byref(p), loss, kl, clipped, logp, stats, slope, grad, scratch, None, err, 512)

    def loss_grad(stats=at, slope=at, upstream=at, grad=at):
        return L.crx_policy_loss_grad(ctypes.byref(x), stats, slope, upstream, 0, grad, None, err, 512)

    def norm(norm=at, scratch=at):
        return L.crx_grad_norm(0, None, None, None, norm, scratch, None, err, 512)

    for call, pairs, others in ((scores, ["stats"], ["logp", "entropy", "scratch"]), (scores_grad, ["stats"], ["entropy", "up", "up_entropy", "grad"]),
                                (loss, ["stats"], ["old", "adv", "ref", "loss", "kl", "clipped", "logp", "slope", "grad", "scratch"]),
                                (loss_grad, ["stats"], ["slope", "upstream", "grad"]), (norm, ["scratch"], ["norm"])):
        for name in pairs + others:
            bad = off if name in ("old", "adv", "ref", "up", "up_entropy") else at + (4 if name in pairs else 2)
            assert call(**{name: bad}) == _native.INVALID and b"aligned" in err.value, (call.__name__, name, err.value)
    numels, types, one = (ctypes.c_uint64 * 1)(8), (ctypes.c_int32 * 1)(2), (ctypes.c_void_p * 1)(at)
    assert L.crx_clip_grads(1, one, numels, types, at + 2, 1.0, None, err, 512) == _native.INVALID and b"aligned" in err.value
    a = AdamW(1e-3, 0.9, 0.99, 1e-8, 0.0, 1, at + 2, 1.0)
    rc = L.crx_adamw_step(1, one, one, one, one, one, numels, types, types, ctypes.byref(a), None, err, 512)
    assert rc == _native.INVALID and b"aligned" in err.value
