import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")
    config.addinivalue_line("markers", "timeout: per-test limit (pytest-timeout; registered here too so that the marker is known without the plugin)")


# Tests that hold a value which is shown to be wrong: they run as they are and have to fail.
HOLDS_A_WRONG_VALUE = {
    "test_adapted_search_gpu.py::test_distill_step[":
        "repeats the loss and gradient of the query as the bank gives it, while every search is made with that query at unit length; "
        "test_distill_step_gpu.py holds the served score's against 64-bit autograd and against differences",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, why in HOLDS_A_WRONG_VALUE.items():
            if name in item.nodeid:
                item.add_marker(pytest.mark.xfail(strict=True, reason=why))


@pytest.fixture(scope="session")
def engine():
    """The initialised HIP library; GPU tests fail (not skip) when it is missing."""
    from rag_system_amd import _lib
    return _lib.engine()
