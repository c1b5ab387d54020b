"""Shared pytest setup: markers, import paths, golden fixtures."""
import json
import os
import sys

import numpy as np
import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG_DIR = os.path.join(REPO, "llama-efficient-inference_b200")
GOLDEN_DIR = os.path.join(REPO, "tests", "golden")
for p in (REPO, PKG_DIR, GOLDEN_DIR):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200 / sm_100a)")


@pytest.fixture(scope="session")
def golden():
    with open(os.path.join(GOLDEN_DIR, "golden.json")) as f:
        meta = json.load(f)
    arrays = dict(np.load(os.path.join(GOLDEN_DIR, "golden.npz")))
    return meta, arrays


@pytest.fixture(scope="session")
def cuda_device():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def paged_device_errors(request):
    """A GPU test of the paged operators (tests/test_paged_*_gpu.py) that leaves a bit in the device error words fails,
    whatever its outputs are."""
    if not os.path.basename(str(request.node.fspath)).startswith("test_paged") or \
            request.node.get_closest_marker("gpu") is None:
        yield
        return
    from llama import _native

    _native.device_errors()
    yield
    assert _native.device_errors() == 0, "the test left a device error (a wait that ran out, a bad position or slot)"
