"""Shared pytest setup: the `gpu` marker, import paths and fixtures.

Tests marked `gpu` need a B200 (sm_100) and call the product library
libx100gemm_b200.so through its C ABI; everything else runs on CPU.
"""
import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for sub in ("oracle", "x100-gemm_b200"):
    p = os.path.join(REPO, sub)
    if p not in sys.path:
        sys.path.insert(0, p)
GOLDEN = os.path.join(REPO, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 GPU (sm_100a) and the CUDA library")


def pytest_collection_modifyitems(items):
    """What is built from the reference's own sources (oracle/_ref) fails where those are not at hand: the tests of it come last, so
    that a run that stops at the first failure has run everything else."""
    items.sort(key=lambda item: item.path.name == "test_dropin_gpu.py" or item.name == "test_i8_8192_cubed_equals_reference_gemm_ref_i8")


@pytest.fixture(scope="session")
def golden_dir():
    return GOLDEN
