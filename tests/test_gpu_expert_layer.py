"""The expert layer example end to end: training steps through the grouped
products lower the loss, the 4-bit layer answers as 4-bit rounding allows."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_expert_layer_trains_and_serves():
    spec = importlib.util.spec_from_file_location("expert_layer", os.path.join(ROOT, "examples", "expert_layer.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    first, last, difference = example.main(steps=40, log=lambda *_: None)
    # the loss of zero weights is about 1 (unit-variance targets); gradient steps of 0.7 on about 250 tokens an expert
    # and 192 inputs contract the error by a constant factor
    assert 0.8 < first < 1.2
    assert last < 0.1 * first
    # an E2M1 code's rounding error is at most a sixth of its value and uniform below that: about 0.1 of a value's
    # size in each operand, so about 0.14 of the product's
    assert 0.02 < difference < 0.3
