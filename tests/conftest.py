import os
import sys

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests", "golden"))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (sm_100a) GPU")


def pytest_collection_modifyitems(items):
    """Tests that need the reference's own library run last where it was not built (its sources
    are needed for that): they fail there, and a run that stops at a failure has run all others."""
    if not os.path.exists(os.path.join(ROOT, "integration", "_build", "libttref_cuda.so")):
        items.sort(key=lambda i: i.path.name == "test_gpu_integration.py")  # (stable)


@pytest.fixture(scope="session")
def cache_dir(tmp_path_factory):
    return str(tmp_path_factory.mktemp("tt_cuda_cache"))
