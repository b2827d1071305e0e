"""Chunks of length zero in a cache behind a shared prefix."""

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests.test_gpu_shared_prefix_cache import _cache, _check

pytestmark = gpu


@pytest.mark.parametrize("D,H", [(128, 2), (64, 3), (256, 1)])
def test_chunks_without_tokens(D, H):
    require_gpu()
    g = torch.Generator(device="cuda").manual_seed(D)
    rows = lambda B, h, S: torch.randn((B, h, S, D), generator=g, device="cuda").half()
    cache = _cache(D)
    cache.update_and_fetch(rows(1, H, 100), rows(1, H, 100))
    shared = cache.share()
    for S in (0, 3, 0, 70, 0):
        k, _ = shared.update_and_fetch(rows(4, H, S), rows(4, H, S))
        assert k.shape == (4, H, shared.offset, D)
        q = rows(4, 2 * H, 1)
        _check(shared, q, shared.fused_sdpa(q, 0.1), 0.1, H)
    assert shared.offset == 173
