"""Prompt-cache files of caches that share a prefix (no GPU)."""

import pytest
import torch

from veloxquant_mlx_amd.cache import KVCacheConfig, KVCacheFactory, load_prompt_cache, save_prompt_cache


def _cache():
    return KVCacheFactory.create(KVCacheConfig(method="kivi", head_dim=128, bit_width_inlier=4, fused_sdpa=True, fused_sdpa_memory_bound=True))


def test_the_cache_that_was_shared_is_saved_and_not_the_sequences_behind_it(tmp_path):
    cache, path = _cache(), str(tmp_path / "prompt.safetensors")
    cache.state = tuple(torch.randn((1, 2, 9, 128)).half() for _ in range(2))
    shared = cache.share()
    with pytest.raises(ValueError, match="layer 1 is a SharedPrefixKIVICache, which has no state"):
        save_prompt_cache(path, [cache, shared])
    assert not (tmp_path / "prompt.safetensors").exists()
    save_prompt_cache(path, [cache])
    again = load_prompt_cache(path, lambda i, name: _cache(), device="cpu")[0].share()
    assert again.offset == shared.offset == 9
    for name in ("k_tail", "v_tail"):
        assert torch.equal(again._prefix_args[name], shared._prefix_args[name])
