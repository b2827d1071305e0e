"""Packed caches that are emptied and filled again with another batch, attended against the same slots in 64 bits."""

import math

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests._spans import attend, seen
from tests.test_gpu_shared_prefix_cache import _cache, _check, _slots

pytestmark = gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("D,H,dtype", [(128, 2, F16), (64, 3, BF16), (256, 2, F16)])
def test_batches_of_a_shared_cache_one_after_the_other(D, H, dtype):
    """Larger and smaller batches on one prefix, each past a flush, whose tokens the one before left room for or not."""
    require_gpu()
    g = torch.Generator(device="cuda").manual_seed(D)
    rows = lambda B, h, S: torch.randn((B, h, S, D), generator=g, device="cuda").to(dtype)
    cache, scale = _cache(D), 1 / math.sqrt(D)
    cache.update_and_fetch(rows(1, H, 200), rows(1, H, 200))
    shared = cache.share()
    for B in (5, 9, 2, 33):
        for S in (40, 1, 60, 1):
            shared.update_and_fetch(rows(B, H, S), rows(B, H, S))
            q = rows(B, 2 * H, S)
            _check(shared, q, shared.fused_sdpa(q, scale), scale, H)
        assert shared._own._n_quantized == 64
        assert shared.trim(1000) == 102 and shared.offset == 200


@pytest.mark.parametrize("method", ["kivi", "kivi_sink"])
def test_batches_of_a_cache_one_after_the_other(method):
    require_gpu()
    D, H, scale = 128, 2, 1 / math.sqrt(128)
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = lambda B, h, S: torch.randn((B, h, S, D), generator=g, device="cuda").half()
    cache = _cache(D, method=method)
    for B in (3, 7, 1):
        fresh = _cache(D, method=method)
        for S in (100, 1, 1):
            k, v, q = rows(B, H, S), rows(B, H, S), rows(B, 4, S)
            got = []
            for c in (cache, fresh):   # (one holds the other's tokens until its attention call)
                c.update_and_fetch(k.clone(), v.clone())
                got.append(c.fused_sdpa(q, scale, fixed_order=True))
            assert torch.equal(*got)
        ks, vs = _slots(cache._store_args())
        if method == "kivi":   # (the step holds a packed slot as code * scale + zero: one rounding to fp16 less)
            want, _ = attend(q, ks, vs, seen(B, 1, 0, 102, None, True, 0), scale, 2.0 ** -11)
            assert float((got[0].double() - want).abs().max()) <= 2e-3 * max(1.0, float(want.abs().max()))
        assert cache.trim(1000) == 102 and cache.offset == 0
