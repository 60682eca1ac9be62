import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


def pytest_collection_modifyitems(items):
    # Streams share a few hardware queues in the order in which they are first used.  These tests hold one stream while another goes on,
    # so the two have to be on different queues: they come before files that use streams.
    items.sort(key=lambda item: os.path.basename(str(item.fspath)) != "test_gpu_pinned_context.py")


@pytest.fixture(scope="session")
def corc():
    """The C oracle (oracle/bdh_oracle.c) through ctypes; built on demand."""
    from oracle.bdh_oracle import COracle

    return COracle()
