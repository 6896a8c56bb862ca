"""The expert layer example's own checks, on the CPU: a context that keeps what it is asked for and computes nothing."""
import importlib.util
import os

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Array:
    ptr = 0

    def __init__(self, shape):
        self.shape = shape

    def to_host(self):
        return np.ones(self.shape, np.float32)


class Calls:
    """Stands in for a context: every call is listed by its name."""

    def __init__(self, *_):
        self.names = []

    def __enter__(self):
        return self

    def __exit__(self, *_):
        pass

    def empty(self, shape, dtype):
        return Array(shape)

    def upload(self, x):
        return Array(x.shape)

    def __getattr__(self, name):
        return lambda *_: self.names.append(name)


@pytest.fixture
def example():
    spec = importlib.util.spec_from_file_location("expert_layer", os.path.join(ROOT, "examples", "expert_layer.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_more_tokens_than_there_is_room_for_are_refused(example):
    """Nothing may be copied: it would go past the device buffers."""
    ctx = Calls()
    layer = example.ExpertLayer(ctx, np.zeros((2, 8, 16), np.float32), 10)
    served = example.ServedLayer(layer)
    del ctx.names[:]
    offsets = np.array([0, 4, 11])
    for call in (lambda: layer.forward(np.zeros((11, 16)), offsets), lambda: served.forward(np.zeros((11, 16)), offsets),
                 lambda: layer.backward(np.zeros((11, 8)))):
        with pytest.raises(ValueError, match="11 tokens"):
            call()
    assert ctx.names == []
    layer.forward(np.zeros((10, 16)), np.array([0, 4, 10]))
    assert "gemm_grouped" in ctx.names


def test_each_line_gives_its_own_difference(example, monkeypatch):
    """Single tokens and the prompt have their own figures; the largest is what main returns."""
    differences = {1: 0.5, 3: 0.25, 200: 0.375}
    monkeypatch.setattr(example, "Context", Calls)
    monkeypatch.setattr(example.ExpertLayer, "forward", lambda self, x, offsets: np.ones((len(x), 4)))
    monkeypatch.setattr(example.ServedLayer, "forward", lambda self, x, offsets: np.full((len(x), 4), 1 + differences[len(x)]))
    lines = []
    worst = example.main(steps=1, out=4, tokens=200, log=lines.append)[2]
    assert [line.split()[-1] for line in lines[1:]] == ["0.500", "0.250", "0.375"]
    assert worst == 0.5
