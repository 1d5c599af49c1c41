import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on a B200)")


def pytest_collection_modifyitems(config, items):
    try:
        import torch
        has_gpu = torch.cuda.is_available()
    except Exception:
        has_gpu = False
    if has_gpu:
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(scope="session", autouse=True)
def cublas_workspace():
    """The workspace that cuBLAS keeps from its first product on, taken before the first test, when it has a segment of torch's
    memory to itself. Taken in some test it stays in whatever large segment was cached then, and the rest of that is free to a test
    that means to leave no room."""
    import torch
    if torch.cuda.is_available():
        x = torch.ones(8, 8, device="cuda")
        (x @ x).sum().item()


@pytest.fixture(scope="session")
def golden_dir():
    return os.path.join(ROOT, "tests", "golden")
