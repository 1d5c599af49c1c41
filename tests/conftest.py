import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on a B200)")
    config.addinivalue_line("markers", "cpu_only: hands made-up addresses to calls that a device would take; only where there is none")


# (as if marked cpu_only)
CPU_ONLY = {"test_strides_of_one_row_or_head_do_not_count"}


def pytest_collection_modifyitems(config, items):
    try:
        import torch
        has_gpu = torch.cuda.is_available()
    except Exception:
        has_gpu = False
    skip = pytest.mark.skip(reason="made-up addresses, and a CUDA device" if has_gpu else "no CUDA device")
    for item in items:
        cpu_only = "cpu_only" in item.keywords or getattr(item, "originalname", None) in CPU_ONLY
        if cpu_only if has_gpu else "gpu" in item.keywords:
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
