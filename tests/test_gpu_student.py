"""The example that trains a linear-attention student on a teacher's top logits and generates with it: its loss falls, and
prompt and single tokens give the logits of the whole text.  Both paths round the same activations to bf16, in other
orders of summation; a unit in the last place of a layer's activations (2^-8) is carried on through the layers that follow, so
the logits may differ by a few of them: 2^-4 of their rms at most, over 10^5 and more of them."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_distillation_example_learns_and_generates():
    spec = importlib.util.spec_from_file_location("distill_example", os.path.join(ROOT, "examples", "distill.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, off = example.main(["--steps", "12"])
    assert all(0 < v < 100 for v in losses)
    assert min(losses[-3:]) < 0.9 * losses[0]
    assert off <= 2.0 ** -4
