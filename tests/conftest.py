import os
import sys
import time

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
GOLDEN = os.path.join(ROOT, "tests", "golden")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on a B200)")


_rested = False


def pytest_runtest_setup(item):
    """Before the tests that count the memory in use: the autograd engine's thread lets go of the last gradients a moment after a
    backward pass has returned."""
    global _rested
    if item.module.__name__ == "test_zz_no_alloc" and not _rested:
        _rested = True
        time.sleep(0.5)


@pytest.fixture(scope="session")
def golden_dir():
    return GOLDEN
