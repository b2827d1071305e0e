import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu)")


@pytest.fixture(autouse=True)
def _random_numbers():
    """What a test draws without a seed of its own is the same in every run (which rows of a sink-protecting cache are protected hangs on it)."""
    torch.manual_seed(0)


@pytest.fixture
def d() -> int:
    return 128


@pytest.fixture
def seed() -> int:
    return 42
