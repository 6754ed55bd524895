"""The cases of perf/: what their preparation leaves for the device's own
stream, which waits for none of torch's (it is made non-blocking)."""

from __future__ import annotations

import importlib
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

PERF = Path(__file__).resolve().parents[1] / "perf"


class Log(list):
    """A device, a buffer's view and a stream that write down what is asked of them."""

    def __getattr__(self, name):
        if name.startswith("_"):
            raise AttributeError(name)

        def call(*args, **kwargs):
            self.append(name)
            return self

        return call


def module(name):
    sys.path.insert(0, str(PERF))
    try:
        return importlib.import_module(name)
    finally:
        sys.path.remove(str(PERF))


@pytest.mark.parametrize("name,kind", [("operators", "norm"), ("operators", "silu"), ("operators", "rows"),
                                       ("cases", "matmul"), ("cases", "attention"), ("cases", "norm")])
def test_prepared_buffers_are_waited_for(name, kind, monkeypatch):
    """Every copy that torch queues into a buffer has been waited for when
    prepare() returns: the framework's first call would not wait for it."""
    m, log = module(name), Log()
    inputs = tuple(torch.zeros(2, 4) for _ in range(2)) + (torch.zeros(4, dtype=torch.bfloat16),)
    if kind == "matmul":
        inputs = torch.zeros((3, 4), dtype=torch.bfloat16), torch.zeros(2, 4)
    elif kind == "attention":
        inputs = torch.zeros(2, 4), torch.zeros(2, 4), torch.zeros(2, 4)
    elif kind == "rows":
        inputs = inputs[0], None, inputs[2]
    for f in ("_row_inputs", "_matmul_inputs", "_attention_inputs", "_norm_inputs"):
        monkeypatch.setattr(m, f, lambda case, seed: inputs, raising=False)
    monkeypatch.setattr(m, "own", True, raising=False)
    monkeypatch.setattr(m, "_hip", lambda: log)
    monkeypatch.setattr(m, "_view", lambda buf, *shape: log)
    monkeypatch.setattr(m.torch.cuda, "current_stream", lambda *a: SimpleNamespace(synchronize=lambda: log.append("wait")))
    monkeypatch.setattr(m.torch.cuda, "synchronize", lambda *a: log.append("wait"))
    m.prepare({"kind": kind, "n": 2, "rows": 2, "cols": 4, "dim": 4}, 1)
    copies = [i for i, what in enumerate(log) if what == "copy_"]
    assert copies and "wait" in log[copies[-1]:]
