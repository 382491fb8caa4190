import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


# Tests that hold a wrong value, and what replaces them; each has to fail.
SUPERSEDED = {
    "test_layer_follows_its_definition": "its oracle counts the arriving frame, which has no token in the cache yet, among the "
                                         "keep_frames protected ones, so that keep_frames = 1 protects nothing; see "
                                         "test_layer_protects_the_last_frames in test_gpu_frame_attention_edges.py",
}


def pytest_collection_modifyitems(config, items):
    import torch
    for item in items:
        if item.name in SUPERSEDED:
            item.add_marker(pytest.mark.xfail(reason=SUPERSEDED[item.name], strict=True))
    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no GPU in this environment")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(scope="session")
def lib():
    """The built C-ABI library; builds it only if nothing has been built yet."""
    from deltacnn_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from deltacnn_amd.csrc import build as _b  # noqa: F401
        _b.build()
    return _lib.load()
