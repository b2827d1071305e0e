"""Caches behind a shared prefix: chunks of length zero, prefixes restored from a state alone."""

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


@pytest.mark.parametrize("H", [2, 3, 4, 5])
def test_a_prefix_restored_without_its_meta_state(H):
    """Heads of 64 channels are kept in pairs, and the arrays do not show whether the last one is whole: queries and keys do."""
    require_gpu()
    D = 64
    g = torch.Generator(device="cuda").manual_seed(H)
    rows = lambda B, h, S: torch.randn((B, h, S, D), generator=g, device="cuda").half()
    cache = _cache(D)
    cache.update_and_fetch(rows(1, H, 100), rows(1, H, 100))
    again = type(cache).from_state(cache._config, cache.state)
    one, two = cache.share(), again.share()
    q, k, v = rows(3, 2 * H, 1), rows(3, H, 5), rows(3, H, 5)
    assert torch.equal(one.fused_sdpa(q, 0.1), two.fused_sdpa(q, 0.1))
    for c in (one, two):
        assert c.update_and_fetch(k, v)[0].shape == (3, H, 105, D)
    got = two.fused_sdpa(q, 0.1)
    assert torch.equal(one.fused_sdpa(q, 0.1), got)
    _check(two, q, got, 0.1, H)
    with pytest.raises(ValueError, match="as the prefix is"):
        two.update_and_fetch(rows(3, H + 1, 1), rows(3, H + 1, 1))
    assert two.branch().fused_sdpa(q, 0.1).shape == q.shape
