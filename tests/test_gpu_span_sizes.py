"""Sizes of attention over spans that other tests leave out."""

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests.test_gpu_differential import _case as _two_maps
from tests.test_gpu_shared_prefix import _case
from veloxquant_mlx_amd import kernels as K

pytestmark = gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [1, 3, 81, 129, 255])
@pytest.mark.parametrize("B,Hq,Hkv,n,own,Sq", [(1, 1, 1, 5, 12, 1), (3, 3, 1, 0, 40, 1), (1, 5, 5, 300, 7, 3), (1, 1, 1, 3000, 1, 1)])
def test_odd_heads(dtype, D, B, Hq, Hkv, n, own, Sq):
    """Odd numbers of records of odd size, in one part and in many."""
    require_gpu()
    _case(B, Hq, Hkv, D, (0, n), (0, own), Sq, dtype=dtype, seed=D)


@pytest.mark.parametrize("bits,v_layout", [(4, "channel"), (3, "channel"), (2, "token")])
def test_odd_heads_over_packed_slots(bits, v_layout):
    require_gpu()
    _case(3, 3, 1, 81, (96, 5), (32, 6), 1, bits=bits, v_layout=v_layout)


@pytest.mark.parametrize("kw", [
    dict(B=70, Hq=8, Hkv=2, prefix=(1024, 40), own=(128, 9)), dict(B=70, Hq=8, Hkv=2, prefix=(512, 0), own=(64, 33), bits=2, group=64),
    dict(B=70, Hq=8, Hkv=2, prefix=(768, 3), own=(128, 50), lens=[(37 * b) % 179 for b in range(70)]),
    dict(B=70, Hq=8, Hkv=2, prefix=(768, 70), own=(128, 9), bits=2, window=200), dict(B=65, Hq=4, Hkv=1, prefix=(256, 5), own=(0, 3), dtype=BF16, window=30),
    dict(B=40, Hq=16, Hkv=2, prefix=(512, 9), own=(128, 20), Sq=5), dict(B=6, Hq=16, Hkv=2, prefix=(512, 9), own=(128, 20), Sq=6),
    dict(B=6, Hq=16, Hkv=2, prefix=(512, 9), own=(128, 20), Sq=6, bits=2, lens=[0, 1, 148, 130, 5, 64], window=300),
    dict(B=5, Hq=16, Hkv=2, prefix=(1280, 1), own=(64, 64), Sq=8, dtype=BF16, group=128), dict(B=100, Hq=6, Hkv=2, prefix=(256, 0), own=(0, 0), causal=False)])
def test_prefixes_in_tiles_with_heads_of_256(kw):
    """More than 256 rows over the prefix with at most 64 a sequence: prefix tiles and own slots are two launches that fill one set of parts."""
    require_gpu()
    _case(D=256, **kw)


@pytest.mark.parametrize("kw", [
    # the prefix by the kernel for few rows, own slots in tiles
    dict(B=2, Hq=8, Hkv=8, D=64, prefix=(1024, 0), own=(66560, 9), Sq=48, bits=2),
    # more than 64 rows a sequence: prefix and own slots walked by the same tiles
    dict(B=2, Hq=8, Hkv=2, D=128, prefix=(512, 9), own=(256, 40), Sq=150), dict(B=3, Hq=4, Hkv=2, D=256, prefix=(256, 70), own=(128, 60), Sq=90, bits=2),
    dict(B=2, Hq=8, Hkv=2, D=64, prefix=(384, 0), own=(128, 70), Sq=198, bits=2, lens=[198, 77]), dict(B=2, Hq=8, Hkv=2, D=128, prefix=(256, 33), own=(0, 300), Sq=300, dtype=BF16, window=90),
    dict(B=2, Hq=4, Hkv=1, D=256, prefix=(128, 5), own=(256, 9), Sq=40, dtype=BF16, lens=[265, 3]),
    # bfloat16 rows beside packed slots, few of them and many
    dict(B=5, Hq=8, Hkv=2, D=128, prefix=(640, 70), own=(128, 45), dtype=BF16), dict(B=48, Hq=8, Hkv=2, D=128, prefix=(640, 70), own=(128, 45), dtype=BF16, bits=2),
    dict(B=9, Hq=8, Hkv=2, D=64, prefix=(320, 33), own=(64, 9), Sq=9, dtype=BF16)])
def test_other_cuts(kw):
    require_gpu()
    _case(**kw)


@pytest.mark.parametrize("kw", [
    dict(B=2, Hq=8, Hkv=2, D=128, slots=(512, 40), Sq=300), dict(B=1, Hq=8, Hkv=2, D=256, slots=(512, 40), Sq=130, bits=2), dict(B=2, Hq=4, Hkv=2, D=64, slots=(256, 9), Sq=265, bits=2),
    dict(B=2, Hq=8, Hkv=2, D=128, slots=(512, 40), Sq=300, dtype=BF16, lens=[552, 290]), dict(B=1, Hq=8, Hkv=2, D=256, slots=(384, 17), Sq=401, dtype=BF16, window=100),
    dict(B=3, Hq=8, Hkv=2, D=128, slots=(256, 100), Sq=20, dtype=BF16), dict(B=2, Hq=6, Hkv=2, D=66, slots=(0, 75), Sq=3), dict(B=1, Hq=3, Hkv=1, D=2, slots=(0, 9), Sq=2, norm=False)])
def test_two_maps(kw):
    """Prompts and chunks over packed slots, bfloat16 beside them, halves of odd size."""
    require_gpu()
    _two_maps(**kw)


def _rounded(x, u):
    return x if u is None else x.to(u).double()


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("D,n,G,Sq", [(64, 3, 1, 1), (128, 7, 4, 1), (256, 5, 2, 3), (80, 9, 1, 2), (128, 70, 1, 1)])
def test_float32_rows_keep_float32(maps, D, n, G, Sq):
    """Without packed slots nothing of a float32 call is held in 16 bits.  Scores, below 0.1, are off by D + 4 roundings of 2^-24, exponentials,
    references and the quotient by 2^-20 together, sums by n roundings, so a result by far less than weights or rows rounded to fp16 or
    bfloat16 are (which the same bound refuses, computed in 64 bits)."""
    require_gpu()
    B, H = 2, 3
    gen = torch.Generator(device="cuda").manual_seed(D + n)
    q, k, v = (torch.rand((B, h, m, D), generator=gen, device="cuda") + 0.5 for h, m in ((H * G, Sq), (H, n), (H, n)))
    v = v * torch.randn(v.shape, generator=gen, device="cuda").sign()
    scale, lam = 0.1 / (2.25 * D), 0.5
    if maps == 1:
        got = K.shared_prefix_attend(q, dict(k_tail=k[:1, :, :1], v_tail=v[:1, :, :1], n_tail=1), k_tail=k, v_tail=v, n_tail=n, scale=scale)
        one = lambda x: torch.cat([x[:1, :, :1].expand(B, -1, -1, -1), x], 2).repeat_interleave(G, 1).double()
    else:
        got = K.differential_attend(q, lam, k_tail=k, v_tail=v, n_tail=n, scale=scale)
        one = lambda x: x.repeat_interleave(G, 1).double()
    k, v = one(k), one(v)

    def formula(weights=None, rows=None):
        o = 0.0
        for i in range(maps):
            ch = slice(i * D // maps, (i + 1) * D // maps)
            p = torch.softmax((q[..., ch].double() @ k[..., ch].transpose(2, 3)) * scale, -1)
            o = o + (1.0 if i == 0 else -lam) * (_rounded(p, weights) @ _rounded(v, rows))
        return o

    want = formula()
    bound = (1 + lam) * v.abs().amax(2, keepdim=True) * (2 * 0.1 * (D + 4) * 2.0 ** -24 + 2.0 ** -20 + (n + 3) * 2.0 ** -24)
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())
    for mistake in (dict(weights=F16), dict(weights=BF16), dict(rows=F16), dict(rows=BF16)):
        assert bool(((formula(**mistake) - want).abs() > bound).any()), mistake


def test_out_may_be_the_queries():
    """``out`` may be the queries themselves: the same bits, one part a row and many, every kernel."""
    require_gpu()
    for kw in (dict(B=3, Hq=8, Hkv=2, D=128, prefix=(256, 7), own=(0, 33)), dict(B=21, Hq=8, Hkv=2, D=128, prefix=(4096, 7), own=(512, 33)),
               dict(B=60, Hq=8, Hkv=2, D=128, prefix=(4096, 7), own=(512, 33)), dict(B=2, Hq=8, Hkv=2, D=128, prefix=(0, 64), own=(0, 300), Sq=150),
               dict(B=2, Hq=6, Hkv=3, D=80, prefix=(0, 64), own=(0, 300), Sq=5, dtype=F32)):
        q, p, o, got = _case(**kw)
        again = q.clone()
        assert K.shared_prefix_attend(again, p, **o, scale=q.shape[3] ** -0.5, causal=True, out=again) is again and torch.equal(again, got)
    for kw in (dict(B=2, Hq=8, Hkv=2, D=128, slots=(4096, 30)), dict(B=2, Hq=8, Hkv=2, D=128, slots=(0, 300), Sq=300, dtype=BF16), dict(B=1, Hq=2, Hkv=1, D=66, slots=(0, 300), Sq=3)):
        q, lam, s, w, got = _two_maps(**kw)
        again = q.clone()
        K.differential_attend(again, lam, **s, scale=(q.shape[3] // 2) ** -0.5, causal=True, norm_weight=w, gain=0.2, out=again)
        assert torch.equal(again, got)
