"""bfloat16 queries and plain rows beside packed slots count as fp16 numbers: large magnitudes as 65504, what is not finite as it is."""

import math

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests._spans import attend, close, seen, store
from tests.test_gpu_differential import reference
from veloxquant_mlx_amd import kernels as K

pytestmark = gpu
BF16 = torch.bfloat16
CUTS = [   # few rows, tiles of a prefix beside few rows, tiles of everything
    dict(B=3, Sq=1, n=256), dict(B=64, Sq=1, n=1536), dict(B=2, Sq=70, n=256)]


def _setup(maps, D, B, Sq, n, bits=4, Hq=8, H=2):
    o, ok, ov = store(B, H, 0 if maps == 1 else n, 80, D, bits=bits, dtype=BF16, seed=2, spare=8)
    p, pk, pv = store(1, H, n, 9, D, bits=bits, dtype=BF16, seed=1) if maps == 1 else (None, ok[:1, :, :0], ov[:1, :, :0])
    q = torch.randn((B, Hq, Sq, D), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(BF16)
    return q, p, o, torch.cat([pk.expand(B, -1, -1, -1), ok], 2), torch.cat([pv.expand(B, -1, -1, -1), ov], 2)


def _call(maps, q, p, o):
    scale = 1 / math.sqrt(q.shape[3] // maps)
    if maps == 1:
        return K.shared_prefix_attend(q, p, **o, scale=scale, causal=True)
    return K.differential_attend(q, 0.4, **o, scale=scale, causal=True)


@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("maps,D", [(1, 128), (1, 64), (1, 256), (2, 128), (2, 256)])
@pytest.mark.parametrize("place", ["own values", "own keys", "prefix values", "prefix keys", "queries"])
def test_large_magnitudes_count_as_the_largest_fp16_number(cut, maps, D, place):
    require_gpu()
    if maps == 2 and "prefix" in place:
        pytest.skip("no prefix")
    q, p, o, k, v = _setup(maps, D, **cut)
    tail = k.shape[2] - 80                   # place of the own plain rows
    first = tail - 9                         # ... of the prefix's
    B, Sq = q.shape[0], q.shape[2]
    cap = 65504.0
    if place == "queries":
        q[1, 3, 0, 5], q[0, 2, -1, 7] = 1e5, -3e38
        for s in (p, o):      # (their channels of the keys are zeros: the others decide)
            for name in () if s is None else ("k_tail", "k_scale", "k_zero"):
                if name in s:
                    s[name][..., 5], s[name][..., 7] = 0.0, 0.0
        k[..., 5], k[..., 7] = 0.0, 0.0
        ref_q = q.double().clamp(-cap, cap)
    else:
        ref_q = q.double()
        side, which = place.split()
        s, at, b = (o, tail, B - 1) if side == "own" else (p, first, slice(None))
        rows, t = (s["v_tail"], v) if which == "values" else (s["k_tail"], k)
        rows[b if side == "own" else 0, 1, 4, 3], rows[b if side == "own" else 0, 0, 6, 9] = 1e5, -3e38
        t[b, 1, at + 4, 3], t[b, 0, at + 6, 9] = cap, -cap
    got = _call(maps, q, p, o)
    scale = 1 / math.sqrt(D // maps)
    mask = seen(B, Sq, 0, k.shape[2], None, True, 0)
    if maps == 1:
        want, far = attend(ref_q, k, v, mask, scale, 2.0 ** -11)
    else:
        want, far = reference(ref_q, k, v, 0.4, mask, scale, 2.0 ** -11)
    assert bool(got.isfinite().all())
    close(got, want, far)


@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("maps,D", [(1, 128), (1, 256), (2, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_stays_so(cut, maps, D, bad):
    """A value that every row of its kv head and sequence sees makes its channel of theirs not finite, a key's channel of NaN the rows NaN; others
    keep their bits."""
    require_gpu()
    q, p, o, _, _ = _setup(maps, D, **cut)
    Sq = q.shape[2]
    clean = _call(maps, q, p, o)
    o["v_tail"][1, 1, 0, 3] = bad
    got = _call(maps, q, p, o)
    sees = Sq <= 80   # slot 0 of the own rows lies before every query
    assert sees and not bool(got[1, 4:, :, 3].isfinite().any())
    got[1, 4:, :, 3] = clean[1, 4:, :, 3]
    assert torch.equal(got, clean)
    o["v_tail"][1, 1, 0, 3] = 0.0
    clean = _call(maps, q, p, o)
    o["k_tail"][1, 1, 0, 3] = float("nan")
    got = _call(maps, q, p, o)
    assert bool(got[1, 4:].isnan().all())
    got[1, 4:] = clean[1, 4:]
    assert torch.equal(got, clean)
