import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if REPO not in sys.path:
    sys.path.insert(0, REPO)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200, sm_100a)")


def _reference_unavailable():
    """Why the reference project's own kernels cannot run here, or None: the library is built from a checkout of it, which
    is not part of this repository.  Where there is a checkout the library has to be there too."""
    from oracle import build_oracle

    if os.path.exists(build_oracle.REF_LIB) or os.path.isdir(os.path.join(build_oracle.DEFAULT_REFERENCE, "src", "impl")):
        return None
    return "no checkout of the reference project to build its kernels from; tests/golden holds their recorded outputs"


def pytest_collection_modifyitems(config, items):
    """GPU tests fail (not skip) where they are asked for and CUDA is missing; elsewhere -m deselects them.  Only the
    comparisons with the reference project's kernels are skipped, where these cannot be had."""
    why = _reference_unavailable()
    if why:
        for item in items:
            if item.path.name == "test_reference_gpu.py":
                item.add_marker(pytest.mark.skip(reason=why))


@pytest.fixture(scope="session")
def cuda():
    import torch

    assert torch.cuda.is_available(), "this test needs a CUDA device"
    return torch.device("cuda:0")
