"""Runs tests/cpp/test_norm_refusals.cpp: what the C++ surface's norms refuse, on the CPU."""
from test_cpp_programs import run


def test_cpp_norm_refusals():
    assert run("test_norm_refusals").strip().endswith("ok")
