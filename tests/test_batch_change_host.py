"""Packed caches that are emptied and filled again with other rows, on the host: buffers are those of the rows that are written to them
(the kernels take their addresses and cannot tell)."""

import pytest
import torch

from veloxquant_mlx_amd import kernels as K
from veloxquant_mlx_amd.cache import KVCacheConfig, KVCacheFactory

F16, BF16 = torch.float16, torch.bfloat16


def _cache(**kw):
    return KVCacheFactory.create(KVCacheConfig(**{**dict(method="kivi", head_dim=128, bit_width_inlier=4, kivi_group_size=32, residual_length=32,
                                                         fused_sdpa=True, fused_sdpa_memory_bound=True), **kw}))


def _rows(B, H, S, D, dtype=F16):
    return torch.zeros((B, H, S, D), dtype=dtype)


@pytest.fixture
def writes(monkeypatch):
    """The kernels' place is taken by checks of what they would write; the calls that passed."""
    calls = []

    def append(k, v, k_tail, v_tail, n_tail, n_flush, packed, tok0, spare, **kw):
        B, H, S, D = k.shape
        buffers = [k_tail, v_tail] + (list(packed) + list(spare) if n_flush else [])
        assert all(t.shape[:2] == (B, H) for t in buffers), [tuple(t.shape) for t in buffers]
        assert k_tail.shape[3] == v_tail.shape[3] == D and n_tail + S <= k_tail.shape[2] and k_tail.dtype == k.dtype
        if n_flush:
            assert packed[1].shape[3] == D and tok0 + n_flush <= packed[0].shape[2] and spare[0].shape[3] == D
        calls.append((tuple(k.shape), n_flush))
        return kw.get("args")

    def pack(x, axis, group, bits, *, out, dst_tok0, **kw):
        assert all(t.shape[:2] == x.shape[:2] for t in out) and (axis == -1 or out[1].shape[3] == x.shape[3])
        calls.append((tuple(x.shape), x.shape[2]))

    monkeypatch.setattr(K, "kivi_cache_append", append)
    monkeypatch.setattr(K, "kivi_quant_pack", pack)
    return calls


@pytest.mark.parametrize("S", [70, 5])
@pytest.mark.parametrize("first,then", [
    ((5, 2, 128, F16), (9, 2, 128, F16)), ((5, 2, 128, F16), (2, 2, 128, F16)), ((3, 2, 128, F16), (3, 4, 128, F16)), ((3, 2, 128, F16), (3, 2, 128, BF16)),
    ((1, 8, 128, F16), (8, 1, 128, F16)), ((2, 2, 128, F16), (2, 2, 64, F16))])
@pytest.mark.parametrize("method", ["kivi", "kivi_sink"])
def test_an_emptied_cache_takes_other_rows(writes, method, first, then, S):
    c = _cache(method=method)
    for B, H, D, dtype in (first, then, first):
        x = _rows(B, H, S, D, dtype)
        c.update_and_fetch(x, x)
        c.update_and_fetch(x, x)
        assert c.offset == 2 * S and c._tail_k.shape[:2] == (B, H) and c._tail_k.dtype == dtype
        assert (c._n_quantized > 0) == (S == 70) and (S != 70 or c._ks.shape[:2] == (B, H))
        c.offset = c._n_quantized = 0   # (what trimming all of it leaves)
    assert len(writes) >= (6 if method == "kivi" else 0)


@pytest.mark.parametrize("first,then", [((4, 4, 64), (7, 4, 64)), ((4, 4, 64), (4, 3, 64)), ((4, 3, 64), (2, 5, 64)), ((4, 4, 64), (4, 1, 64))])
def test_an_emptied_cache_of_paired_heads(writes, first, then):
    c = _cache(head_dim=64)
    for B, H, D in (first, then):
        x = _rows(B, H, 70, D)
        c.update_and_fetch(x, x)
        pairs = (H + 1) // 2 if H > 1 else 1
        assert c._pair == (H > 1) and c._tail_k.shape[:2] == (B, pairs) and c._ks.shape[3] == (128 if H > 1 else 64)
        c.offset = c._n_quantized = 0


@pytest.mark.parametrize("method", ["kivi", "kivi_sink"])
@pytest.mark.parametrize("S", [70, 1])
def test_a_cache_with_tokens_refuses_other_rows(writes, method, S):
    c = _cache(method=method)
    x = _rows(3, 2, 70, 128)
    c.update_and_fetch(x, x)
    seen, shape = len(writes), c._shape_bhd
    for B, H, D in ((4, 2, 128), (2, 2, 128), (3, 4, 128), (3, 2, 64), (6, 1, 128)):
        x = _rows(B, H, S, D)
        with pytest.raises(ValueError, match="holds 3 sequences, 2 heads and 128 channels"):
            c.update_and_fetch(x, x)
    assert c.offset == 70 and c._shape_bhd == shape and len(writes) == seen and c._pending is None


def test_protected_rows_of_an_emptied_cache_are_forgotten(writes):
    c = _cache(method="kivi_sink", n_sink_tokens=2)
    x = torch.rand((3, 2, 70, 128)).half()
    c.update_and_fetch(x, x)
    assert c._side_k.shape[0] == 3
    c.trim(70)
    y = torch.rand((5, 2, 70, 128)).half()
    c.update_and_fetch(y, y)
    assert c._side_k.shape[0] == 5 and len(c._side_pos) == 5 and c._extra_attend_args()["sinks"][2].shape[0] == 5
    c.trim(70)
    c.update_and_fetch(x[:1], x[:1])
    assert c._side_k.shape[0] == 1 and len(c._side_pos) == 1


@pytest.mark.parametrize("prompt", [300, 9])
def test_a_shared_cache_takes_another_batch_once_it_is_empty(writes, prompt):
    cache = _cache()
    packed = prompt // 32 * 32 if prompt > 64 else 0
    state = [_rows(1, 2, prompt - packed, 128) for _ in range(2)]
    if packed:
        meta = [torch.zeros((1, 2, packed // 32, 128), dtype=F16)] * 2
        state = [torch.zeros((1, 2, packed, 16), dtype=torch.int32), *meta, torch.zeros((1, 2, packed // 8, 128), dtype=torch.int32),
                 *[torch.zeros((1, 2, 4, packed), dtype=F16)] * 2] + state
    cache.state = tuple(state)
    shared = cache.share()
    assert shared.offset == prompt
    for B in (5, 9, 2):
        x = _rows(B, 2, 70, 128)
        shared.update_and_fetch(x, x)
        x = _rows(B, 2, 1, 128)
        shared.update_and_fetch(x, x)
        assert shared.offset == prompt + 71 and shared._own._n_quantized == 32 and shared._own._tail_k.shape[0] == shared._own._kp.shape[0] == B
        with pytest.raises(ValueError, match=f"this cache holds {B}"):
            x = _rows(B + 1, 2, 1, 128)
            shared.update_and_fetch(x, x)
        shared._own.offset = shared._own._n_quantized = 0
    assert writes[-2:] == [((2, 2, 70, 128), 32), ((2, 2, 1, 128), 0)]


def test_the_append_refuses_buffers_of_other_rows():
    new = _rows(9, 2, 40, 128)
    tails = lambda B=9, H=2, D=128, n=128: tuple(_rows(B, H, n, D) for _ in range(2))

    def packed(B=9, H=2, D=128, cap=64, layout="token"):
        k = [torch.zeros((B, H, cap, D // 8), dtype=torch.int32)] + [torch.zeros((B, H, cap // 32, D), dtype=F16) for _ in range(2)]
        if layout == "token":
            return k + [torch.zeros((B, H, cap // 8, D), dtype=torch.int32)] + [torch.zeros((B, H, D // 32, cap), dtype=F16) for _ in range(2)]
        return k + [torch.zeros((B, H, cap, D // 8), dtype=torch.int32)] + [torch.zeros((B, H, cap, D // 32), dtype=F16) for _ in range(2)]

    def call(tail, n_flush=0, store=None, spare=None):
        K.kivi_cache_append(new, new, *tail, 0, n_flush, store, 0, spare, bits=4, group_size=32, levels=15, eps=1e-8, v_layout="token")

    for tail in (tails(B=5), tails(H=1), tails(D=64)):
        with pytest.raises(ValueError, match="tails .* do not fit"):
            call(tail)
    for store in (packed(B=5), packed(H=4), packed(D=64), packed(layout="channel"), packed()[:5] + packed(cap=96)[5:], packed(cap=96)[:3] + packed()[3:]):
        with pytest.raises(ValueError, match="packed store .* does not fit"):
            call(tails(), 32, store, tails())
    for spare in (tails(B=5), tails(D=256), (tails()[0], tails(n=64)[0])):
        with pytest.raises(ValueError, match="spare tails .* do not fit"):
            call(tails(), 32, packed(), spare)
    with pytest.raises(RuntimeError, match="no CPU path"):   # (buffers that fit)
        call(tails(), 32, packed(), tails())


def test_a_shared_cache_refuses_values_unlike_the_keys(writes):
    """Before anything is counted: the cache goes on as it was."""
    cache = _cache()
    cache.state = (_rows(1, 2, 9, 128), _rows(1, 2, 9, 128))
    shared = cache.share()
    good = _rows(3, 2, 5, 128)
    shared.update_and_fetch(good, good)
    for S in (5, 1):
        k = _rows(3, 2, S, 128)
        for v in (_rows(3, 2, S + 1, 128), _rows(1, 2, S, 128), _rows(3, 1, S, 128), _rows(3, 2, S, 64), k[0], k.bfloat16()):
            with pytest.raises(ValueError, match="as the prefix is"):
                shared.update_and_fetch(k, v)
    assert shared.offset == 14 and len(writes) == 1
    shared.update_and_fetch(good, good)
    assert shared.offset == 19


def test_no_tokens_are_appended_to_a_shared_cache(writes):
    """A chunk of length zero, before any own token and behind some."""
    cache = _cache()
    cache.state = (_rows(1, 2, 9, 128), _rows(1, 2, 9, 128))
    shared = cache.share()
    none, some = _rows(3, 2, 0, 128), _rows(3, 2, 5, 128)
    for x, n in ((none, 0), (some, 5), (none, 5), (some, 10)):
        k, v = shared.update_and_fetch(x, x)
        assert k.shape == v.shape == (3, 2, 9 + n, 128) and shared.offset == 9 + n


def test_a_restored_prefix_of_paired_heads_takes_its_keys(writes):
    """Restored without its meta_state it holds 5 or 6 heads; keys of neither leave it as it is."""
    cache = _cache(head_dim=64)
    cache.state = (_rows(1, 3, 9, 128), _rows(1, 3, 9, 128))      # three pairs
    for H in (5, 6):
        shared = cache.share()
        for bad in (10, 4, 12, 3):
            with pytest.raises(ValueError, match="as the prefix is"):
                shared.update_and_fetch(_rows(2, bad, 1, 64), _rows(2, bad, 1, 64))
        assert shared.update_and_fetch(_rows(2, H, 4, 64), _rows(2, H, 4, 64))[0].shape == (2, H, 13, 64)
        with pytest.raises(ValueError, match="as the prefix is"):
            shared.update_and_fetch(_rows(2, 11 - H, 1, 64), _rows(2, 11 - H, 1, 64))
