"""The example model trains: CPU path, GPU path against it, and under autocast."""

from __future__ import annotations

import importlib.util
import os

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("tabular_distillation",
                                                  os.path.join(REPO, "examples", "tabular_distillation.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_example_trains_on_cpu():
    losses = _example().train("cpu", steps=12, rows=1024, batch=256, report=lambda s: None)
    assert losses[-1] < 0.8 * losses[0]


@pytest.mark.gpu
def test_example_trains_on_gpu_as_on_cpu():
    ex = _example()
    cpu = ex.train("cpu", steps=3, rows=1024, batch=256, report=lambda s: None)
    gpu = ex.train("cuda", steps=3, rows=1024, batch=256, report=lambda s: None)
    # (the first loss is one forward in 32 bits; the next ones follow an optimizer that
    # divides by the gradient's size, which amplifies its rounding)
    assert abs(gpu[0] - cpu[0]) < 1e-4 * cpu[0]
    assert all(abs(g - c) < 0.02 * c for g, c in zip(gpu, cpu))


@pytest.mark.gpu
def test_example_trains_under_autocast():
    losses = _example().train("cuda", steps=25, rows=2048, batch=512, autocast=True, report=lambda s: None)
    assert losses[-1] < 0.7 * losses[0]
