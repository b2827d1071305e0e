"""Caches that share a prefix, and differential attention over a cache, as a model's layer uses them: rotary positions, append,
attend, against the same over the cache's own slots in 64 bits."""

import math

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests._spans import _rows, attend, close, seen
from tests.test_gpu_differential import reference
from veloxquant_mlx_amd.cache import KVCacheConfig, KVCacheFactory, SharedPrefixKIVICache
from veloxquant_mlx_amd.fused_sdpa import make_fused_dispatcher
from veloxquant_mlx_amd.rotary import RotaryPositions

pytestmark = gpu
F16, BF16 = torch.float16, torch.bfloat16


def _cache(D, **kw):
    cfg = dict(method="kivi", head_dim=D, bit_width_inlier=4, kivi_group_size=32, residual_length=32, fused_sdpa=True, fused_sdpa_memory_bound=True)
    return KVCacheFactory.create(KVCacheConfig(**{**cfg, **kw}))


def _slots(a):
    """Keys and values a cache's slots stand for, in 64 bits."""
    n, D = a["n_packed"], (a["k_scale"] if a["n_packed"] else a["k_tail"]).shape[3]
    ks, vs = [], []
    if n:
        ks.append(_rows(a["k_packed"][:, :, :n].transpose(2, 3), a["k_scale"], a["k_zero"], a["bits"], D, n, a["group_size"], "k"))
        vs.append(_rows(a["v_packed"], a["v_scale"], a["v_zero"], a["bits"], D, n, a["group_size"], a["v_layout"]))
    if a["n_tail"]:
        ks.append(a["k_tail"][:, :, : a["n_tail"]].double())
        vs.append(a["v_tail"][:, :, : a["n_tail"]].double())
    return torch.cat(ks, 2), torch.cat(vs, 2)


def _unpair(x, H):
    """[B, P, n, 2 D] of paired heads -> [B, H, n, D]"""
    B, P, n, D2 = x.shape
    return x.view(B, P, n, 2, D2 // 2).transpose(2, 3).reshape(B, 2 * P, n, D2 // 2)[:, :H]


def _check(shared, q, got, scale, H, lens=None, window=0):
    pk, pv = _slots(shared._prefix_args)
    B, _, Sq, D = q.shape
    if shared._own.offset:
        ok, ov = _slots(shared._own._store_args())
    else:
        ok = ov = pk.new_zeros((B, pk.shape[1], 0, pk.shape[3]))
    k, v = torch.cat([pk.expand(B, -1, -1, -1), ok], 2), torch.cat([pv.expand(B, -1, -1, -1), ov], 2)
    if k.shape[3] != D:
        k, v = _unpair(k, H), _unpair(v, H)
    own_lens = None if lens is None else torch.as_tensor(lens, device="cuda") - shared.prefix_length
    packed = shared._prefix._n_quantized + shared._own._n_quantized > 0
    want, far = attend(q, k, v, seen(B, Sq, shared.prefix_length, ok.shape[2], own_lens, True, window), scale,
                       torch.finfo(F16 if packed else q.dtype).eps / 2)
    close(got, want, far)


@pytest.mark.parametrize("kw", [dict(D=128, Hq=8, H=2), dict(D=64, Hq=6, H=3, bit_width_inlier=2), dict(D=64, Hq=6, H=2, kivi_pair_heads=False),
                                dict(D=256, Hq=4, H=2, dtype=BF16), dict(D=128, Hq=8, H=4, dtype=BF16, prompt=9), dict(D=128, Hq=4, H=2, bit_width_inlier=3)])
def test_a_prompt_shared_by_sequences(kw):
    """Prefill of the prompt, then chunks and single tokens of five sequences behind it, past flushes of their own, every step attended
    through the dispatcher; then tokens taken back, and a second batch on the same prefix."""
    require_gpu()
    kw = dict(kw)
    D, Hq, H, dtype, prompt = kw.pop("D"), kw.pop("Hq"), kw.pop("H"), kw.pop("dtype", F16), kw.pop("prompt", 333)
    cache, rope, scale = _cache(D, **kw), RotaryPositions(D, base=500000.0), 1 / math.sqrt(D)
    g = torch.Generator(device="cuda").manual_seed(D + Hq)
    fresh = lambda B, S: [torch.randn((B, h, S, D), generator=g, device="cuda").to(dtype) for h in (Hq, H, H)]
    sdpa = make_fused_dispatcher(lambda *a, **k: pytest.fail("fell through to dense attention"))
    q, k, v = fresh(1, prompt)
    q, k = rope(q, k, offset=0)
    sdpa(q, *cache.update_and_fetch(k, v), cache=cache, scale=scale, mask="causal")
    shared = cache.share()
    assert isinstance(shared, SharedPrefixKIVICache) and shared.offset == shared.prefix_length == prompt
    q = fresh(3, 1)[0]
    _check(shared, q, shared.fused_sdpa(q, scale), scale, H)   # before any token of their own
    cache.update_and_fetch(k[:, :, :40], v[:, :, :40])         # (the prefix is a copy: the cache goes on by itself)

    def step(c, B, S, **opts):
        q, k, v = fresh(B, S)
        q, k = rope(q, k, offset=c.offset)
        keys, values = c.update_and_fetch(k, v)
        assert keys.shape == (B, H, c.offset, D) and values.shape == keys.shape
        got = c.fused_sdpa(q, scale, **opts) if opts else sdpa(q, keys, values, cache=c, scale=scale, mask="causal" if S > 1 else None)
        _check(c, q, got, scale, H, opts.get("lengths"), opts.get("sliding_window", 0))

    for S in (7, 1, 1, 60, 1, 1):
        step(shared, 5, S)
    assert shared.offset == prompt + 71 and shared._own._n_quantized == 32
    step(shared, 5, 1, sliding_window=50)
    step(shared, 5, 1, sliding_window=prompt)
    own = torch.tensor([3, 40, 0, 73, 74])
    step(shared, 5, 1, lengths=own[[0, 1, 2, 4, 3]] + prompt)
    step(shared, 5, 1, lengths=(own + prompt).cuda())
    assert shared.trim(20) == 20 and shared.offset == prompt + 55
    step(shared, 5, 1)
    other = shared.branch()
    step(other, 2, 4)
    step(shared, 5, 1)
    assert other.offset == prompt + 4 and shared.offset == prompt + 57
    assert shared.trim(1000) == 57 and shared.offset == prompt
    step(shared, 5, 40)
    step(shared, 5, 1)
    assert shared.trim(39) == 39 and shared.offset == prompt + 2 and shared._own._n_quantized == 0
    step(shared, 5, 1)


def test_one_sequence_is_a_cache():
    """A batch of one behind a prefix agrees with one cache that holds prompt and tokens (quantised at other boundaries: residual longer
    than the tokens, so that both hold them as they are)."""
    require_gpu()
    D, scale = 128, 1 / math.sqrt(128)
    cache = _cache(D, residual_length=96)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((1, 2, 300, D), generator=g, device="cuda").half() for _ in range(2))
    cache.update_and_fetch(k, v)
    shared = cache.share()
    k, v = (torch.randn((1, 2, 3, D), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((1, 8, 3, D), generator=g, device="cuda").half()
    cache.update_and_fetch(k, v)
    shared.update_and_fetch(k, v)
    one, other = cache.fused_sdpa(q, scale), shared.fused_sdpa(q, scale)
    assert cache._n_quantized == shared._prefix._n_quantized
    assert float((one.float() - other.float()).abs().max()) <= 2e-3 * max(1.0, float(one.abs().max()))


def test_the_context_limit_counts_the_prefix():
    require_gpu()
    cache = _cache(128, fused_sdpa_max_ctx=512)
    k = torch.randn((1, 2, 300, 128), device="cuda").half()
    cache.update_and_fetch(k, k)
    shared = cache.share()
    rows = lambda n: torch.randn((3, 2, n, 128), device="cuda").half()
    x = rows(200)
    shared.update_and_fetch(x, x)
    assert shared.offset == 500 and shared._own._packed_cap == 224     # 212 left, in whole groups
    q = torch.randn((3, 4, 1, 128), device="cuda").half()
    before = shared.fused_sdpa(q, 0.1)
    with pytest.raises(RuntimeError, match="fused_sdpa_max_ctx"):
        x = rows(100)
        shared.update_and_fetch(x, x)
    assert shared.offset == 500 and torch.equal(shared.fused_sdpa(q, 0.1), before)


def test_shared_refusals():
    require_gpu()
    k = torch.zeros((2, 2, 5, 128), dtype=F16, device="cuda")
    cache = _cache(128)
    with pytest.raises(ValueError, match="batch of one"):
        cache.share()
    cache.update_and_fetch(k, k)
    with pytest.raises(ValueError, match="batch of one"):
        cache.share()
    stash = _cache(128, fused_sdpa_memory_bound=False)
    stash.update_and_fetch(k[:1], k[:1])
    with pytest.raises(ValueError, match="memory_bound"):
        stash.share()
    cache = _cache(128)
    cache.update_and_fetch(k[:1], k[:1])
    shared = cache.share()
    for bad in (k[:, :1], k[..., :64].contiguous(), k.bfloat16(), k[0]):
        with pytest.raises(ValueError, match="as the prefix is"):
            shared.update_and_fetch(bad, bad)
    shared.update_and_fetch(k, k)
    with pytest.raises(ValueError, match="this cache holds 2"):
        shared.update_and_fetch(k[:1], k[:1])
    q = torch.zeros((2, 4, 1, 128), dtype=F16, device="cuda")
    for bad, what in ((dict(lengths=[5, 4]), "count the prefix"), (dict(lengths=[9, 9, 9]), "3 entries"), (dict(sliding_window=-1), "sliding window")):
        with pytest.raises(ValueError, match=what):
            shared.fused_sdpa(q, 0.1, **bad)
    with pytest.raises(ValueError):
        shared.fused_sdpa(q[:1], 0.1)
    assert shared.offset == 10


@pytest.mark.parametrize("kw", [dict(D=128), dict(D=128, fused_sdpa_memory_bound=False), dict(D=64, kivi_pair_heads=False, bit_width_inlier=2),
                                dict(D=256, dtype=BF16), dict(D=64, fused_sdpa_memory_bound=False)])
def test_differential_attention_over_a_cache(kw):
    """Halves turned by rotary positions each, prefill in two chunks and single tokens past a flush, the head norm behind."""
    require_gpu()
    kw = dict(kw)
    D, dtype, Hq, H, B = kw.pop("D"), kw.pop("dtype", F16), 8, 2, 3
    cache, rope, scale = _cache(D, **kw), RotaryPositions(D // 2), 1 / math.sqrt(D // 2)
    g = torch.Generator(device="cuda").manual_seed(D)
    lam = torch.rand(Hq, generator=g, device="cuda") * 0.5 + 0.2
    weight = torch.rand(D, generator=g, device="cuda") + 0.5
    for i, S in enumerate((70, 33, 1, 1, 1, 40, 1)):
        q, k, v = (torch.randn((B, h, S, D), generator=g, device="cuda").to(dtype) for h in (Hq, H, H))
        # a head's halves are heads of half the channels to the rotation
        halves = lambda x: x.view(B, -1, S, 2, D // 2).transpose(2, 3).reshape(B, -1, S, D // 2)
        whole = lambda x: x.view(B, -1, 2, S, D // 2).transpose(2, 3).reshape(B, -1, S, D)
        q, k = (whole(x) for x in rope(halves(q), halves(k), offset=cache.offset))
        cache.update_and_fetch(k, v)
        lengths = None if i != 4 else [cache.offset, 50, 7]
        opts = dict(norm_weight=weight, gain=0.8) if i % 2 else {}
        got = cache.fused_differential_sdpa(q, lam, scale, lengths=lengths, **opts)
        ks, vs = _slots(cache._store_args())
        mask = seen(B, S, 0, cache.offset, None if lengths is None else torch.tensor(lengths, device="cuda"), True, 0)
        want, far = reference(q, ks, vs, lam, mask, scale, torch.finfo(F16 if cache._n_quantized else dtype).eps / 2, opts.get("norm_weight"), 1e-5,
                              opts.get("gain", 1.0))
        close(got, want, far)
    assert cache._n_quantized > 0


def test_differential_refusals():
    require_gpu()
    q = torch.zeros((1, 4, 1, 64), dtype=F16, device="cuda")
    k = torch.zeros((1, 2, 5, 64), dtype=F16, device="cuda")
    cache = _cache(64)
    with pytest.raises(RuntimeError, match="before any tokens"):
        cache.fused_differential_sdpa(q, 0.1, 0.1)
    cache.update_and_fetch(k, k)
    with pytest.raises(ValueError, match="kivi_pair_heads"):
        cache.fused_differential_sdpa(q, 0.1, 0.1)
    plain = _cache(64, fused_sdpa=False, fused_sdpa_memory_bound=False)
    plain.update_and_fetch(k, k)
    with pytest.raises(RuntimeError, match="not enabled"):
        plain.fused_differential_sdpa(q, 0.1, 0.1)
    sink = _cache(64, method="kivi_sink", n_sink_tokens=2, kivi_pair_heads=False)
    sink.update_and_fetch(torch.randn_like(k).repeat(1, 1, 40, 1), torch.randn_like(k).repeat(1, 1, 40, 1))
    if sink._extra_attend_args():
        with pytest.raises(ValueError, match="outside its packed store"):
            sink.fused_differential_sdpa(q, 0.1, 0.1)
    good = _cache(64, kivi_pair_heads=False)
    good.update_and_fetch(k, k)
    for bad in (dict(lengths=[1, 2]), dict(sliding_window=-3)):
        with pytest.raises(ValueError):
            good.fused_differential_sdpa(q, 0.1, 0.1, **bad)
