"""``norm_rotary_embed`` against the norm and the rotation in 64 bits."""

import pytest
import torch

from tests._gpu import gpu, require_gpu
from veloxquant_mlx_amd import kernels as K
from veloxquant_mlx_amd.rotary import RotaryPositions

pytestmark = gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _reference(x, weight, eps, at, inv_freq, traditional, factor):
    """x [B, H, S, D], at [B, S]: the normed rows, and those turned, in 64 bits."""
    x = x.double()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        n = n * (weight.double() if weight.ndim == 1 else weight.double()[:, None])
    r = 2 * inv_freq.numel()
    t = at.double()[:, None, :, None] * inv_freq.double()
    c, s = factor * t.cos(), factor * t.sin()
    y = n.clone()
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if traditional else (slice(0, r // 2), slice(r // 2, r))
    a, b = n[..., lo], n[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    return n, y


def _check(got, x, normed, ref, factor=1.0):
    """One rounding to the type (half a step) on top of the float32 arithmetic, in units u = 2^-24: of the norm, D additions of squares lose at
    most D u of the sum (half of it in the root), mean, eps, root and the products with it and the weight 8 more; the turn's angle, sine, cosine and
    products 10 (as for the turn alone) of |a| + |b|, at most twice the row's largest normed magnitude."""
    assert got.dtype == x.dtype and got.shape == x.shape
    D = x.shape[-1]
    half_step = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    bound = half_step * ref.abs() + 2 * (D / 2 + 18) * 2.0 ** -24 * max(1.0, factor) * normed.abs().amax(-1, keepdim=True) + tiny
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


def _rows(B, H, S, D, dtype, seed, view):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if view == "dense":
        x = torch.randn((B, H, S, D), generator=g, device="cuda")
    elif view == "projection":   # [B, S, H + 1, D] rows, heads 1 .. H
        return (torch.randn((B, S, H + 1, D), generator=g, device="cuda") * 3).to(dtype)[:, :, 1:].transpose(1, 2)
    elif view == "odd":          # rows that start at odd elements
        return torch.randn((B, H, S, D + 3), generator=g, device="cuda").to(dtype)[..., 1:D + 1]
    else:
        return torch.randn((B, H, S, D, 2), generator=g, device="cuda").to(dtype)[..., 0]   # channels apart
    return (x * torch.randn((B, H, S, 1), generator=g, device="cuda").exp()).to(dtype)


def _weight(shape, dtype, seed):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") + 1).to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("traditional", [False, True])
@pytest.mark.parametrize("B,Hq,Hk,S,D,dims,view,weights", [
    (1, 32, 8, 1, 128, 128, "projection", "row"), (2, 5, 1, 7, 64, 64, "dense", "row"), (3, 12, 4, 67, 256, 64, "projection", "heads"),
    (1, 2, 2, 300, 80, 80, "dense", "row"), (2, 3, 1, 33, 96, 24, "odd", "heads"), (1, 1, 1, 5, 7, 6, "dense", "row"),
    (1, 2, 1, 9, 16, 2, "apart", "none"), (4, 40, 10, 513, 128, 96, "projection", "row"), (1, 9, 3, 2000, 64, 32, "projection", "none"),
    (2, 3, 2, 11, 24, 16, "dense", "row"), (1, 2, 1, 3, 1024, 512, "dense", "heads"), (1, 1, 1, 2, 2048, 2048, "dense", "row"),
    (2, 4, 2, 65, 8, 8, "dense", "row"), (1, 3, 1, 17, 40, 16, "projection", "heads"), (5, 1, 1, 129, 16, 16, "dense", "heads")])
def test_rows(dtype, traditional, B, Hq, Hk, S, D, dims, view, weights):
    require_gpu()
    q, k = _rows(B, Hq, S, D, dtype, 1, view), _rows(B, Hk, S, D, dtype, 2, view)
    kept = q.clone(), k.clone()
    qw, kw = ((None, None) if weights == "none" else (_weight((D,), dtype, 3), _weight((D,), dtype, 4)) if weights == "row"
              else (_weight((Hq, D), dtype, 3), _weight((Hk, D), dtype, 4)))
    rope = RotaryPositions(dims, traditional=traditional)
    first = torch.arange(B, device="cuda") * 1000003 + 17      # far apart, past a million
    got = rope.normed(q, k, q_weight=qw, k_weight=kw, norm_eps=1e-5, offset=first)
    at = first[:, None] + torch.arange(S, device="cuda")
    for x, w, y in zip((q, k), (qw, kw), got):
        assert y.is_contiguous()
        _check(y, x, *_reference(x, w, 1e-5, at, rope.inv_freq, traditional, 1.0))
    assert torch.equal(q, kept[0]) and torch.equal(k, kept[1])
    # one position tensor a sequence, alone or with k, and a host offset: the same bits
    for positions in (at, at.int(), at[:, None, :].expand(B, 3, S)[:, 1]):
        assert torch.equal(rope.normed(q, q_weight=qw, norm_eps=1e-5, positions=positions), got[0])
    assert torch.equal(rope.normed(k, q_weight=kw, norm_eps=1e-5, positions=at), got[1])
    same = rope.normed(q, k, q_weight=qw, k_weight=kw, offset=23)
    assert torch.equal(same[0], rope.normed(q, q_weight=qw, positions=(torch.arange(S, device="cuda") + 23)))


@pytest.mark.parametrize("dtype,weight_dtype", [(F16, F32), (BF16, F32), (F32, BF16), (BF16, F16)])
@pytest.mark.parametrize("D,dims", [(128, 64), (100, 100)])
def test_weights_of_another_type_and_a_factor(dtype, weight_dtype, D, dims):
    require_gpu()
    q, k = _rows(2, 6, 19, D, dtype, 5, "projection"), _rows(2, 2, 19, D, dtype, 6, "projection")
    qw, kw = _weight((D,), weight_dtype, 7), _weight((2, D), weight_dtype, 8)
    rope = RotaryPositions(dims, scaling={"type": "yarn", "factor": 8, "original_max_position_embeddings": 4096})
    at = (torch.arange(19, device="cuda") * 37 - 400).expand(2, 19)      # positions below zero too
    got = rope.normed(q, k, q_weight=qw, k_weight=kw, positions=at)
    assert rope.attention_factor > 1
    for x, w, y in zip((q, k), (qw, kw), got):
        _check(y, x, *_reference(x, w, 1e-6, at, rope.inv_freq, False, rope.attention_factor), rope.attention_factor)
    # a weight for one of the two only, and a strided one
    one = rope.normed(q, k, k_weight=torch.stack((kw, kw), -1)[..., 0], positions=at)
    assert torch.equal(one[1], got[1])
    _check(one[0], q, *_reference(q, None, 1e-6, at, rope.inv_freq, False, rope.attention_factor), rope.attention_factor)


@pytest.mark.parametrize("traditional,D,dims", [(False, 128, 128), (True, 128, 64), (False, 20, 12), (False, 256, 64)])
def test_outputs_in_place_and_in_a_cache(traditional, D, dims):
    require_gpu()
    B, Hq, Hk, S = 2, 8, 2, 19
    rows = torch.randn((B, S, (Hq + 2 * Hk) * D), device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)).half()
    q = rows[..., : Hq * D].view(B, S, Hq, D).transpose(1, 2)
    k = rows[..., Hq * D: (Hq + Hk) * D].view(B, S, Hk, D).transpose(1, 2)
    v = rows[..., (Hq + Hk) * D:].clone()
    qw, kw = _weight((D,), F16, 1), _weight((Hk, D), F16, 2)
    rope = RotaryPositions(dims, traditional=traditional)
    want = rope.normed(q, k, q_weight=qw, k_weight=kw, offset=5)
    store = torch.full((B, Hk, 64, D), 7.0, dtype=F16, device="cuda")
    rope.normed(q, k, q_weight=qw, k_weight=kw, offset=5, k_out=store[:, :, 10: 10 + S])
    assert torch.equal(store[:, :, 10: 10 + S], want[1]) and bool((store[:, :, :10] == 7).all()) and bool((store[:, :, 10 + S:] == 7).all())
    got = rope.normed(q, k, q_weight=qw, k_weight=kw, offset=5, out=q, k_out=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(rows[..., (Hq + Hk) * D:], v)


@pytest.mark.parametrize("D,dims", [(128, 128), (128, 32), (12, 12)])
def test_values_that_are_not_finite_stay_in_their_row(D, dims):
    require_gpu()
    x = _rows(1, 3, 40, D, F32, 11, "dense")
    clean = RotaryPositions(dims).normed(x, offset=3)
    x[0, 1, 7, D - 1], x[0, 2, 9, 0], x[0, 0, 0] = float("nan"), float("inf"), 0.0
    got = RotaryPositions(dims).normed(x, offset=3)
    assert bool(got[0, 1, 7].isnan().all()) and bool(got[0, 2, 9, 0].isnan()) and bool((got[0, 0, 0] == 0).all())
    hit = torch.zeros(x.shape[:3], dtype=torch.bool, device="cuda")
    hit[0, 1, 7] = hit[0, 2, 9] = hit[0, 0, 0] = True
    assert torch.equal(got[~hit], clean[~hit])
    # rows below the normal numbers, eps 0: as large ones, rows of zeros are 0 / 0
    small = torch.full((1, 1, 1, D), 2.0 ** -70, device="cuda")
    y = RotaryPositions(dims).normed(small, norm_eps=0.0, positions=torch.zeros(1, dtype=torch.int64, device="cuda"))
    assert float((y - 1).abs().max()) < (D / 2 + 18) * 2.0 ** -23
    assert bool(RotaryPositions(dims).normed(torch.zeros((1, 1, 1, D), device="cuda"), norm_eps=0.0).isnan().all())


def test_other_stream_and_graph():
    require_gpu()
    q, k = _rows(2, 8, 33, 128, BF16, 12, "projection"), _rows(2, 2, 33, 128, BF16, 13, "projection")
    w = _weight((128,), BF16, 14)
    rope = RotaryPositions(128)
    at = torch.zeros(2, dtype=torch.int64, device="cuda")
    want = [rope.normed(q, k, q_weight=w, k_weight=w, offset=n) for n in (0, 5, 900000)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rope.normed(q, k, q_weight=w, k_weight=w, offset=5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[0], want[1][0]) and torch.equal(other[1], want[1][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rope.normed(q, k, q_weight=w, k_weight=w, offset=at)
    for n, ref in zip((0, 5, 900000, 5), (*want, want[1])):
        at.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_empty_calls():
    require_gpu()
    rope = RotaryPositions(64)
    for shape in ((0, 4, 3, 64), (2, 0, 3, 64), (2, 4, 0, 64)):
        q = torch.zeros(shape, dtype=F16, device="cuda")
        assert rope.normed(q).shape == shape
    q, k = torch.zeros((2, 0, 3, 64), dtype=F16, device="cuda"), _rows(2, 2, 3, 64, F16, 15, "dense")
    assert torch.equal(rope.normed(q, k)[1], rope.normed(k))
