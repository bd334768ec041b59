"""examples/verify_step.py: the step operators between the quantized matmuls."""
from __future__ import annotations

import os
import runpy

import pytest

pytestmark = pytest.mark.gpu


def test_verify_step(capsys):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "verify_step.py")
    runpy.run_path(path)["main"]()
    out = capsys.readouterr().out
    assert out.count("accepted") == 2 and "one by one" in out
