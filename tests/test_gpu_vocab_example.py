"""The operators over a vocabulary together, as examples/distill_text_tower.py
uses them: the losses fall and the student comes to choose as its teacher."""
import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_student_learns_from_its_teacher():
    spec = importlib.util.spec_from_file_location("distill_text_tower",
                                                  os.path.join(ROOT, "examples", "distill_text_tower.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.main(["--steps", "150", "--texts", "128", "--vocab", "1000", "--dim", "64"])
    assert all(math.isfinite(v) for v in r["first"] + r["last"])
    assert r["last"][0] < 0.5 * r["first"][0] and r["last"][1] < r["first"][1]
    assert r["agreement"] > 0.5
