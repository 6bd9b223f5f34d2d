"""perf/operators.py mixes torch's memory with calls on the runtime's own stream, which no stream of torch's waits for:
the order of its waits, without a GPU."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("own", [False, True])
def test_prepare_waits_on_both_sides(monkeypatch, own):
    torch = pytest.importorskip("torch")
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    done = []

    class Made:
        def __init__(self, case, seed):
            done.append("tensors")

    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: done.append("wait"))
    monkeypatch.setattr(ops, "State", Made)
    monkeypatch.setattr(ops, "own", own)
    ops.prepare(ops.listed()[0], 1)
    assert done == ["wait", "tensors", "wait"]
