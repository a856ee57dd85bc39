"""examples/gated_delta_mixer.py keeps nothing of a step behind its backward (the library's calls are stood in for: no GPU
is needed)."""
import gc
import os
import sys
import weakref

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture
def example(kmb, monkeypatch):
    import gated_delta_mixer as ex
    kept = []
    monkeypatch.setattr(ex, "_stream", lambda: None)
    monkeypatch.setattr(kmb, "delta_forward", lambda p, ws, **_: kept.append(weakref.ref(ws)))
    monkeypatch.setattr(kmb, "norm_forward", lambda p, **_: kept.append(weakref.ref(p._keep[6])))
    monkeypatch.setattr(kmb, "delta_backward", lambda *a, **_: None)
    monkeypatch.setattr(kmb, "norm_backward", lambda *a, **_: None)
    gc.collect()
    gc.disable()
    yield ex, kept
    gc.enable()


def test_the_mixer_frees_its_workspace(example):
    ex, kept = example
    r = lambda *s: torch.rand(s).requires_grad_(True)
    cu = torch.tensor([0, 3, 7], dtype=torch.int32)
    o, hT = ex.GatedDelta.apply(r(1, 7, 1, 8), r(1, 7, 1, 8), r(1, 7, 2, 4), r(1, 7, 2), r(1, 7, 2), cu, 0.5)
    assert kept[0]() is not None
    o.sum().backward()
    del o, hT
    assert kept[0]() is None


def test_the_norm_frees_its_statistics(example):
    ex, kept = example
    r = lambda *s: torch.rand(s).requires_grad_(True)
    y, s = ex.Norm.apply(r(5, 8), r(5, 8), r(8), r(8))
    assert kept[0]() is not None
    (y.sum() + s.sum()).backward()
    del y, s
    assert kept[0]() is None
