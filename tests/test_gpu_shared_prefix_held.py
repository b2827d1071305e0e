"""What a shared prefix keeps, and that calls repeat themselves."""

import math

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests.test_gpu_differential import _case as _two_maps
from tests.test_gpu_shared_prefix import _case
from tests.test_gpu_shared_prefix_cache import _cache
from veloxquant_mlx_amd import kernels as K

pytestmark = gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("D,prompt", [(128, 333), (64, 100), (256, 64), (128, 9)])
def test_the_prefix_is_a_copy(D, prompt):
    """The cache that was shared goes on, past a flush, is trimmed into the prompt, overwritten and filled again with other batches: what the
    shared cache holds and answers stays, bit for bit."""
    require_gpu()
    g = torch.Generator(device="cuda").manual_seed(D + prompt)
    rows = lambda B, h, S: torch.randn((B, h, S, D), generator=g, device="cuda").half()
    cache, scale = _cache(D), 1 / math.sqrt(D)
    k, v = rows(1, 2, prompt), rows(1, 2, prompt)
    cache.update_and_fetch(k, v)
    shared = cache.share()
    shared.update_and_fetch(rows(4, 2, 3), rows(4, 2, 3))
    q = rows(4, 4, 1)
    held = {n: t.clone() for n, t in shared._prefix_args.items() if isinstance(t, torch.Tensor)}
    live = dict(k_packed=2, k_scale=2, k_zero=2, v_packed=2, v_scale=3, v_zero=3, k_tail=2, v_tail=2)
    assert held and set(held) <= set(live)
    want = shared.fused_sdpa(q, scale)

    def same():
        assert torch.equal(shared.fused_sdpa(q, scale), want)
        for n, t in held.items():
            assert torch.equal(shared._prefix_args[n], t)

    k.zero_(), v.zero_()                                                   # the caller's rows
    same()
    cache.update_and_fetch(rows(1, 2, 150), rows(1, 2, 150))               # past a flush
    same()
    cache.trim(150 + prompt // 2)                                          # back into the prompt ...
    cache.update_and_fetch(rows(1, 2, 200), rows(1, 2, 200))               # ... and over it
    same()
    other = shared.branch()
    other.update_and_fetch(rows(7, 2, 100), rows(7, 2, 100))               # another batch on the same prefix
    other.fused_sdpa(rows(7, 4, 1), scale)
    other.trim(100)
    same()
    cache.trim(10 ** 6)
    cache.update_and_fetch(rows(3, 2, 50), rows(3, 2, 50))
    same()


def test_differential_attention_refuses_rows_outside_the_packed_store():
    require_gpu()
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn((1, 2, 200, 128), generator=g, device="cuda").half()
    sink = _cache(128, method="kivi_sink", n_sink_tokens=2)
    sink.update_and_fetch(x, x)
    assert sink._extra_attend_args()
    with pytest.raises(ValueError, match="outside its packed store"):
        sink.fused_differential_sdpa(torch.zeros((1, 4, 1, 128), dtype=F16, device="cuda"), 0.1, 0.1)
    with pytest.raises(ValueError, match="must be a KIVIKVCache"):
        sink.share()


@pytest.mark.parametrize("kw", [
    dict(B=4, Hq=8, Hkv=2, D=128, prefix=(256, 7), own=(0, 33)), dict(B=21, Hq=8, Hkv=2, D=128, prefix=(4096, 7), own=(512, 33), lens=[26 * b for b in range(21)]),
    dict(B=60, Hq=8, Hkv=2, D=128, prefix=(4096, 7), own=(512, 33)), dict(B=70, Hq=8, Hkv=2, D=256, prefix=(1024, 7), own=(128, 33)),
    dict(B=12, Hq=8, Hkv=2, D=128, prefix=(0, 4000), own=(0, 260), Sq=5, dtype=BF16), dict(B=2, Hq=8, Hkv=2, D=64, prefix=(256, 7), own=(0, 300), Sq=300),
    dict(B=3, Hq=6, Hkv=2, D=80, prefix=(256, 7), own=(0, 300), bits=3, v_layout="channel")])
def test_a_prefix_call_repeats_itself(kw):
    require_gpu()
    q, p, o, got = _case(**kw)
    lens = kw.get("lens")
    call = dict(scale=q.shape[3] ** -0.5, causal=True, seq_lens=None if lens is None else torch.tensor(lens, device="cuda"))
    for _ in range(12):
        assert torch.equal(K.shared_prefix_attend(q, p, **o, **call), got)


@pytest.mark.parametrize("kw", [
    dict(B=1, Hq=32, Hkv=8, D=128, slots=(0, 1100), Sq=1100, dtype=BF16), dict(B=3, Hq=12, Hkv=4, D=256, slots=(0, 400), Sq=400),
    dict(B=1, Hq=8, Hkv=2, D=128, slots=(640, 65), bits=2), dict(B=6, Hq=32, Hkv=8, D=128, slots=(8192, 100)), dict(B=1, Hq=8, Hkv=2, D=128, slots=(512, 40), Sq=300)])
def test_a_differential_call_repeats_itself(kw):
    require_gpu()
    q, lam, s, w, got = _two_maps(**kw)
    for _ in range(12):
        assert torch.equal(K.differential_attend(q, lam, **s, scale=(q.shape[3] // 2) ** -0.5, causal=True, norm_weight=w, gain=0.2), got)
