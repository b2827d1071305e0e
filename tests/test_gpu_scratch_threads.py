"""Host threads that share a stream: every call's result is that of the call alone."""

import threading

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests._spans import store
from veloxquant_mlx_amd import kernels as K

pytestmark = gpu
F16, F32 = torch.float16, torch.float32


def _queries(shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").half()


def _select(seed):
    """Bounds, then choice."""
    s, _, _ = store(1, 4, 20000 + 3200 * seed, 7, 128, bits=4, seed=seed)
    q = _queries((1, 8, 40, 128), seed)
    return lambda: K.select_blocks(q, s["k_scale"], s["k_zero"], 30, levels=15, group_size=32, n_packed=s["n_packed"], n_tail=7, query_block=40, causal=True)


def _blocks(seed):
    """Parts over 8-bit slots, then their sum."""
    s, _, _ = store(2, 2, 2048 + 512 * seed, 9, 128, bits=8, seed=seed)
    q, blocks = _queries((2, 4, 1, 128), seed), torch.arange(40, dtype=torch.int32, device="cuda").expand(2, 2, 1, 40).contiguous()
    return lambda: K.block_sparse_attend(q, blocks, **s, block_size=32, scale=0.1)


def _spans(seed):
    s, _, _ = store(2, 2, 4096 + 1024 * seed, 9, 128, bits=4, seed=seed)
    q = _queries((2, 8, 1, 128), seed)
    return lambda: K.shared_prefix_attend(q, None, **s, scale=0.1)


def _packed(seed):
    s, _, _ = store(2, 2, 4096 + 1024 * seed, 64, 128, bits=4, seed=seed)
    q = _queries((2, 8, 1, 128), seed)
    return lambda: K.kivi_packed_attend(q, **s, scale=0.1, fixed_order=True, num_splits=7, _single_launch=False)


def _decode(seed):
    """One launch, with counters that the stream's calls share."""
    s, _, _ = store(2, 2, 4096 + 1024 * seed, 64, 128, bits=4, seed=seed)
    q = _queries((2, 8, 1, 128), seed)
    return lambda: K.kivi_packed_attend(q, **s, scale=0.1, fixed_order=True, num_splits=5)


def _indices(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = 3000 + 1000 * seed
    ki, vi = (torch.randint(0, 256, (1, 2, n, 16), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
    kc, vc = (torch.randn((256, 8), generator=g, device="cuda") for _ in range(2))
    q = torch.randn((1, 4, 1, 128), generator=g, device="cuda")
    return lambda: K.metal_fused_sdpa(q, ki, kc, vi, vc, 0.1, num_splits=6)


@pytest.mark.parametrize("kinds", [(_select, _select), (_blocks, _blocks), (_spans, _select), (_packed, _packed), (_decode, _blocks), (_indices, _spans)])
def test_two_threads_on_one_stream(kinds):
    require_gpu()
    calls = [kind(seed) for seed, kind in enumerate(kinds)]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    start, got = threading.Barrier(2, timeout=30), [[], []]

    def run(which):
        start.wait()
        for _ in range(60):
            got[which].append(calls[which]())

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads)
    torch.cuda.synchronize()
    for which in range(2):
        assert len(got[which]) == 60
        assert all(torch.equal(x, want[which]) for x in got[which])
