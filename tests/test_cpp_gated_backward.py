"""Builds tests/cpp/test_gated_backward.cu against the C++ API and
libchoreo_b200.so and runs its CPU cases here and its GPU cases on a B200."""
from __future__ import annotations

import pytest

import test_cpp_feed_forward as cpp


@pytest.fixture
def program(monkeypatch):
    monkeypatch.setattr(cpp, "SRC", cpp.ROOT / "tests" / "cpp" / "test_gated_backward.cu")
    monkeypatch.setattr(cpp, "OUT", cpp.ROOT / "tests" / "cpp" / "_build" / "test_gated_backward")
    return cpp.run


def test_cpp_gated_backward_cpu_cases(program):
    assert " 0 failures" in program("cpu")


@pytest.mark.gpu
def test_cpp_gated_backward_gpu_cases(program):
    assert " 0 failures" in program("gpu")
