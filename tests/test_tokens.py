"""Argument checks of token statistics and distillation that need no GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

import gefen
from gefen.kernels import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GOOD = dict(logits=64, labels=64, rows=4, rows_per_batch=2, batch_stride=10, row_stride=5, vocab=5, dtype=0, n_seq=2)
BAD = [({"dtype": 3}, -2), ({"vocab": 0}, -1), ({"rows": -1}, -1), ({"rows_per_batch": 0}, -1), ({"logits": None}, -1),
       ({"rows": 1 << 31}, -1), ({"rows": 1 << 30}, -1), ({"n_seq": -1}, -1), ({"n_seq": 1 << 30}, -1)]
TEACHER = dict(ids=64, logps=64, temperature=1.0, hard_weight=0.0, top=3, ids64=1, rest=0, by_sequence=0)


def logits(**change):
    return _native.Logits(**{**GOOD, **change})


def teacher(**change):
    return _native.Teacher(**{**TEACHER, **change})


def statistics(desc, temperature=1.0, top=3, logps=64, ids=64, ws=64, n=1 << 20):
    return _native.load().gefenx_token_statistics(ctypes.byref(desc), temperature, top, logps, 64, ids, 64, 64, ws, n, None)


def distill(desc, t, ws=64, n=1 << 20, loss=64):
    return _native.load().gefenx_distillation_loss(ctypes.byref(desc), None if t is None else ctypes.byref(t), loss, 64, 64, 64,
                                                   64, 64, ws, n, None)


def test_host_tensors_are_refused():
    x, y = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long)
    ids, lp = torch.zeros(2, 3, 2, dtype=torch.long), torch.zeros(2, 3, 2)
    with pytest.raises(ValueError, match="HIP device"):
        gefen.token_statistics(x, y, top=2)
    with pytest.raises(ValueError, match="HIP device"):
        gefen.token_statistics(x)
    for call in (gefen.distillation_loss, gefen.distillation_loss_and_grad):
        with pytest.raises(ValueError, match="HIP device"):
            call(x, y, ids, lp)


def test_other_things_than_tensors_are_refused():
    with pytest.raises(TypeError):
        gefen.token_statistics([[1.0]])
    with pytest.raises(TypeError):
        gefen.token_logps(torch.zeros(1, 3), None)
    with pytest.raises(TypeError):
        gefen.distillation_loss(torch.zeros(1, 3), None, None, None)


@pytest.mark.parametrize("change,status", BAD)
def test_bad_logits_are_refused_on_the_host(change, status):
    lib, t, bad = _native.load(), teacher(), logits(**change)
    assert lib.gefenx_token_statistics_workspace_bytes(ctypes.byref(logits()), 3) > 0
    assert lib.gefenx_token_statistics_workspace_bytes(ctypes.byref(bad), 3) == 0
    assert statistics(bad) == status
    assert lib.gefenx_token_statistics_grad(ctypes.byref(bad), 1.0, 3, 64, 64, 64, 64, 64, 64, None) == status
    assert lib.gefenx_distillation_workspace_bytes(ctypes.byref(logits()), ctypes.byref(t)) > 0
    assert lib.gefenx_distillation_workspace_bytes(ctypes.byref(bad), ctypes.byref(t)) == 0
    assert distill(bad, t) == status
    assert lib.gefenx_distillation_grad(ctypes.byref(bad), ctypes.byref(t), 64, 64, None, 1.0, 64, None) == status


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan"), float("inf"), 1e-5, 1e5])
def test_temperatures(temperature):
    assert statistics(logits(), temperature) == -1 and "temperature" in _native.last_error()
    assert distill(logits(), teacher(temperature=temperature)) == -1 and "temperature" in _native.last_error()
    assert _native.load().gefenx_token_statistics_grad(ctypes.byref(logits()), temperature, 3, 64, 64, 64, 64, 64, 64, None) == -1


@pytest.mark.parametrize("top", [-1, 6, 129, 1 << 20])
def test_bad_counts_of_tokens(top):
    assert statistics(logits(), top=top) == -1 and "top" in _native.last_error()
    assert _native.load().gefenx_token_statistics_workspace_bytes(ctypes.byref(logits()), top) == 0


@pytest.mark.parametrize("change", [{"top": 0}, {"top": 513}, {"rest": 3}, {"rest": -1}, {"hard_weight": -0.1}, {"hard_weight": 1.5},
                                    {"hard_weight": float("nan")}, {"ids": None}, {"logps": None}])
def test_bad_teachers(change):
    assert distill(logits(), teacher(**change)) == -1
    assert _native.load().gefenx_distillation_workspace_bytes(ctypes.byref(logits()), ctypes.byref(teacher(**change))) == 0


@pytest.mark.parametrize("top,rows,fits", [(128, 1 << 24, True), (128, (1 << 26) - 4, True), (129, (1 << 24) - 1, True),
                                          (129, 1 << 24, False), (512, (1 << 26) - 4, False)])
def test_rows_of_a_launch(top, rows, fits):
    """Short rows go to a wave each, with more than 128 tokens of the teacher to a workgroup each: a launch has 2^32 - 1
    threads at most."""
    desc, t = logits(rows=rows, rows_per_batch=rows, batch_stride=0, row_stride=600, vocab=600), teacher(top=top)
    assert (_native.load().gefenx_distillation_workspace_bytes(ctypes.byref(desc), ctypes.byref(t)) > 0) == fits
    if not fits:
        assert distill(desc, t, n=1 << 40) == -1 and "too many rows" in _native.last_error()
        grad = _native.load().gefenx_distillation_grad
        assert grad(ctypes.byref(desc), ctypes.byref(t), None, 64, None, 1.0, 64, None) == -1
        assert "too many rows" in _native.last_error()


def test_sequences_have_to_cover_the_rows():
    assert distill(logits(n_seq=3), teacher(by_sequence=1)) == -1
    assert distill(logits(n_seq=0), teacher(by_sequence=1)) == -1
    assert distill(logits(), None) == -1


def test_small_workspaces_and_missing_outputs():
    assert statistics(logits(), n=8) == -1 and "workspace" in _native.last_error()
    assert statistics(logits(), ws=None) == -1
    assert statistics(logits(), logps=None) == -1
    assert statistics(logits(labels=None)) == -1  # log-probabilities of no labels
    assert statistics(logits(), ids=None) == -1
    assert distill(logits(), teacher(), n=8) == -1 and "workspace" in _native.last_error()
    assert distill(logits(), teacher(), ws=None) == -1
    assert distill(logits(), teacher(), loss=None) == -1
    assert distill(logits(labels=None), teacher()) == -1
    lib = _native.load()
    grad = lambda *a: lib.gefenx_token_statistics_grad(ctypes.byref(a[0]), 1.0, 3, *a[1:], None)  # noqa: E731
    assert grad(logits(), None, 64, 64, 64, 64, 64) == -1
    assert grad(logits(), 64, None, 64, 64, 64, 64) == -1
    assert grad(logits(), 64, 64, 64, 64, 64, None) == -1
    assert grad(logits(labels=None), 64, 64, 64, 64, 64, 64) == -1
    t = teacher()
    for slopes, weights, out in ((None, 64, 64), (64, None, 64), (64, 64, None)):
        assert lib.gefenx_distillation_grad(ctypes.byref(logits()), ctypes.byref(t), slopes, weights, None, 1.0, out, None) == -1


def test_last_splits_stay_within_shared_memory(tmp_path):
    """The launch's shared memory, sized by whole splits, holds what a shorter last split addresses."""
    exe = tmp_path / "hunt_layout"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "gefen-x_amd", "csrc"), "-o", str(exe),
                    os.path.join(ROOT, "tests", "c", "hunt_layout.cpp")], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True)
    bad, checked = map(int, out.stdout.split())
    assert checked > 10000 and bad == 0, out.stderr
