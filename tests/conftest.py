import os
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))                       # oracle/
sys.path.insert(0, str(ROOT / "4bit-forge_amd"))    # forge/


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP kernels through the C ABI)")


@pytest.fixture(scope="session")
def hip():
    """The operator table; GPU tests fail loudly if the HIP library did not load."""
    import torch
    from forge.backend.hip import kernels
    assert torch.cuda.is_available(), "GPU test collected without a GPU"
    kernels.build_group_meta_packed  # raises RuntimeError if libforge_hip.so is missing
    return kernels


# Tests whose expected value is wrong; they run, and have to fail where the code is right.
WRONG_VALUES = {
    "test_gpu_linear_int4.py::test_follows_the_solve[False]":
        "expects (nibble - 8) * scale of a record with zero points, whose nibbles are code - zero + 8 modulo 16: with "
        "code 15 and zero 5 that is the weight -6 instead of 10; test_gpu_linear_int4_zeros.py has the layer's product",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, why in WRONG_VALUES.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(raises=AssertionError, strict=True, reason=why))
