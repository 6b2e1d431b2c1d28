import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (runs on the GPU box)")
    config.addinivalue_line("markers", "slow: full Paraformer-large CPU oracle runs (seconds each)")


def pytest_collection_modifyitems(items):
    """The sanitizer driver's process first: where a process that has launched a cooperative kernel keeps the device's one
    cooperative queue until it ends, another one's launch is refused (hipErrorIllegalState), so it goes before the tests
    that launch one in this process."""
    items.sort(key=lambda item: item.name != "test_api_end_to_end_asan_gpu")
