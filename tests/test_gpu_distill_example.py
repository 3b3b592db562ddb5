"""The distillation example end to end: the loss falls, the student writes what the teacher finds
likely, every token operator ran on its kernels, and a second run gives the same bits."""
import importlib.util
from pathlib import Path

import pytest
import torch

import xdna_train

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location(
        "distill_student", Path(__file__).resolve().parent.parent / "examples" / "distill_student.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_student_learns_and_repeats():
    main = _example().main
    xdna_train.reset_mapped_cpu_stats()
    first = main(steps=60, batch=4, length=64, report=20)
    stats = xdna_train.mapped_cpu_stats()
    for counter in ("embed.fwd", "embed.bwd", "gated.fwd", "gated.bwd", "distill.fwd", "distill.bwd", "logprobs.fwd"):
        assert stats.get(f"hip_tokens.{counter}.run", {}).get("calls", 0) > 0, counter
    # 60 steps on a fixed teacher: the loss at least halves, and the texts' tokens are at least
    # e times as likely to the teacher as tokens picked without looking
    assert first["losses"][-1] < 0.5 * first["losses"][0]
    assert first["written"] > first["chance"] + 1.0
    second = main(steps=60, batch=4, length=64, report=20)
    assert first["losses"] == second["losses"] and torch.equal(first["text"], second["text"])
