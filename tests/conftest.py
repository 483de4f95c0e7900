"""Pytest configuration: the ``gpu`` marker and shared fixtures.

``-m "not gpu"`` runs the CPU suite (oracle vs golden vectors, C-ABI symbol
checks, host logic, gloo multi-process tests). ``-m gpu`` runs the parity tests
of the CUDA kernels against the CPU oracle on a B200.
"""

import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200) and the built library")


# Tests that hold a wrong value: they run, and have to fail. test_muon_optimizer decays the weights by the learning rate
# times the factor of the matrix's shape, where the factor is the update's alone; tests/test_muon_rules.py and
# tests/test_gpu_muon_rules.py hold the right values, next to torch.optim.Muon's.
WRONG = {
    "tests/test_gpu_orthogonalize.py::test_muon_optimizer": "expects a weight decay scaled by the matrix's shape",
}


def pytest_collection_modifyitems(config, items):
    for item in items:
        if item.nodeid in WRONG:
            item.add_marker(pytest.mark.xfail(reason=WRONG[item.nodeid], raises=AssertionError, strict=True))
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(42)
    yield
