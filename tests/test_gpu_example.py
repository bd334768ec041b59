"""examples/verify_step.py: the step operators between the quantized matmuls."""
from __future__ import annotations

import os
import runpy

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_verify_step(capsys):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "verify_step.py")
    runpy.run_path(path)["main"]()
    out = capsys.readouterr().out
    assert out.count("accepted") == 2 and "one by one" in out


def test_sample_drafts_alike():
    """Drafted steps over several moves of branches, against steps of one token."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "sample_drafts.py")
    results = runpy.run_path(path)["main"]()
    for cache, (alike, most, worst) in results.items():
        # (12 drafted steps: one token each and one more where a branch was taken)
        assert min(most) > 13, cache
        assert cache != torch.float16 or alike == most
