import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a)")


def pytest_collection_modifyitems(items):
    """The tests of the reference's own front-end, whose build needs its source
    tree, come last: where that is missing, a run that stops at the first
    failure has been through everything else."""
    items.sort(key=lambda item: item.path.name == "test_lamp3_front_gpu.py")


@pytest.fixture(scope="session")
def cuda():
    """torch with a CUDA device; GPU tests fail loudly if the kernels are missing."""
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from rushlite_b200 import capi

    capi.lib()  # raises if liblmpb.so is missing
    return torch
