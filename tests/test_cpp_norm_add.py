"""Runs tests/cpp/test_rms_norm_add.cpp, the residual norm through the C++ operator surface."""
import pytest

from test_cpp_programs import run


@pytest.mark.gpu
def test_cpp_rms_norm_add():
    assert run("test_rms_norm_add").strip().endswith("ok")
