import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (a B200); runs the CUDA kernels")


# Suites that run code compiled from the reference's own sources.
REFERENCE_SIDE = {
    "test_program_gpu": ("integration", "libcharlotte_program.so"),
    "test_encoder_program_gpu": ("integration", "libcharlotte_program.so"),
    "test_oracle_pins_gpu": ("oracle", "_ref", "libcharlotte_ref.so"),
}


def pytest_collection_modifyitems(items):
    """Skips the suites whose reference-side library was not built because
    there were no sources to build it from. Where there are, they run, and a
    missing library fails them."""
    import oracle
    for item in items:
        library = REFERENCE_SIDE.get(item.module.__name__)
        if library and not os.path.exists(os.path.join(ROOT, *library)) and oracle.reference_root() is None:
            item.add_marker(pytest.mark.skip(reason="the reference sources were absent when its side would have been built"))


@pytest.fixture(scope="session")
def cuda():
    """The CUDA device for GPU tests. A GPU test never skips: without a device
    it fails, so a run on a box whose CUDA is broken cannot pass silently."""
    import torch
    assert torch.cuda.is_available(), "GPU test without a CUDA device"
    torch.cuda.init()
    return torch.device("cuda:0")
