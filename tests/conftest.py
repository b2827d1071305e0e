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
def _seeded_draw(request):
    """``test_protected_rows_of_an_emptied_cache_are_forgotten`` draws its keys without a seed and expects side rows, which are there only if one of the two
    tokens of the largest mean norm lies below the packed boundary (32 of 70): 38 * 37 / (70 * 69), three draws in ten, have none. It draws the
    same keys in every run; no other test's numbers are touched."""
    if request.node.name.startswith("test_protected_rows_of_an_emptied_cache_are_forgotten"):
        with torch.random.fork_rng(devices=[]):
            torch.random.default_generator.manual_seed(0)
            yield
    else:
        yield


@pytest.fixture
def d() -> int:
    return 128


@pytest.fixture
def seed() -> int:
    return 42
