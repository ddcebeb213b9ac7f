import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a HIP GPU (MI355X) and the built library")


# Tests that hold a wrong value: they run, as they are, and are expected to fail.
WRONG_VALUES = {
    # Its third sequence says 1000 tokens in a table of 48, of which the last 20 are the call's. They stand at positions 980 to
    # 999 (lengths[b] - n + i), where there is no page; the test wants them over tokens 28 to 47, which are other ones.
    # tests/test_gpu_attention_limits.py has the same batch with the value that is right, under the same name.
    "tests/test_gpu_attention.py::test_append_leaves_what_is_not_its_own": "rows past the table written over earlier tokens",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, reason in WRONG_VALUES.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.xfail(reason=reason, strict=True))


@pytest.fixture(scope="session")
def gpu():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("GPU test collected without a GPU")
    from trifuse_amd import _lib

    _lib.load()
    return torch.device("cuda:0")
