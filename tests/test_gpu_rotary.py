"""``rotary_embed`` against the rotation in 64 bits."""

import pytest
import torch

from tests._gpu import gpu, require_gpu
from veloxquant_mlx_amd import kernels as K
from veloxquant_mlx_amd.rotary import RotaryPositions

pytestmark = gpu


def _reference(x, at, inv_freq, traditional, factor, inverse):
    """x [B, H, S, D], at [B, S]: the turned rows in 64 bits."""
    r = 2 * inv_freq.numel()
    t = at.double()[:, None, :, None] * inv_freq.double()
    c, s = factor * t.cos(), factor * t.sin() * (-1 if inverse else 1)
    y = x.double().clone()
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if traditional else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., lo].double(), x[..., hi].double()
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    return y


def _check(got, x, ref, factor=1.0):
    """One rounding to the type (half a step), on top of the float32 turn: the angle is off by at most pi 2^-25, its sine
    and cosine by 2 units of 2^-24, and four more float32 roundings of the two products follow: 6e-7 (|a| + |b|), with |a| + |b|
    at most twice the row's largest magnitude."""
    assert got.dtype == x.dtype and got.shape == x.shape
    half_step = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    bound = half_step * ref.abs() + 2 * 6e-7 * max(1.0, factor) * x.double().abs().amax(-1, keepdim=True) + tiny
    assert bool(((got.double() - ref).abs() <= bound).all()), float(((got.double() - ref).abs() - bound).max())


def _rows(B, H, S, D, dtype, seed, view):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if view == "dense":
        return torch.randn((B, H, S, D), generator=g, device="cuda").to(dtype)
    if view == "projection":   # [B, S, H + 1, D] rows, heads 1 .. H
        return torch.randn((B, S, H + 1, D), generator=g, device="cuda").to(dtype)[:, :, 1:].transpose(1, 2)
    if view == "odd":          # rows that start at odd elements
        return torch.randn((B, H, S, D + 3), generator=g, device="cuda").to(dtype)[..., 1:D + 1]
    return torch.randn((B, H, S, D, 2), generator=g, device="cuda").to(dtype)[..., 0]   # channels apart


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("traditional", [False, True])
@pytest.mark.parametrize("B,Hq,Hk,S,D,dims,view", [
    (1, 32, 8, 1, 128, 128, "projection"), (2, 5, 1, 7, 64, 64, "dense"), (3, 12, 4, 67, 256, 64, "projection"), (1, 2, 2, 300, 80, 80, "dense"),
    (2, 3, 1, 33, 96, 24, "odd"), (1, 1, 1, 5, 7, 6, "dense"), (1, 2, 1, 9, 16, 2, "apart"), (4, 40, 10, 513, 128, 96, "projection"),
    (1, 9, 3, 2000, 64, 32, "projection")])
def test_rows(dtype, traditional, B, Hq, Hk, S, D, dims, view):
    require_gpu()
    q, k = _rows(B, Hq, S, D, dtype, 1, view), _rows(B, Hk, S, D, dtype, 2, view)
    kept = q.clone(), k.clone()
    rope = RotaryPositions(dims, traditional=traditional)
    first = torch.arange(B, device="cuda") * 1000003 + 17      # far apart, past a million
    got = rope(q, k, offset=first)
    at = first[:, None] + torch.arange(S, device="cuda")
    for x, y in zip((q, k), got):
        assert y.is_contiguous()
        _check(y, x, _reference(x, at, rope.inv_freq, traditional, 1.0, False))
    assert torch.equal(q, kept[0]) and torch.equal(k, kept[1])
    # one position tensor a sequence or for all, 32 or 64 bits, alone or with k, and a host offset: the same bits
    for positions in (at, at.int(), at[:, None, :].expand(B, 3, S)[:, 1]):
        assert torch.equal(rope(q, positions=positions), got[0])
    same = rope(q, k, offset=23)
    assert torch.equal(same[0], rope(q, positions=(torch.arange(S, device="cuda") + 23)))
    assert torch.equal(same[1], rope(k, offset=torch.full((1,), 23, dtype=torch.int32, device="cuda")))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("traditional", [False, True])
def test_inverse_and_factor(dtype, traditional):
    require_gpu()
    B, H, S, D = 2, 3, 50, 64
    x = _rows(B, H, S, D, dtype, 3, "dense")
    rope = RotaryPositions(48, traditional=traditional, scaling={"type": "yarn", "factor": 8, "original_max_position_embeddings": 4096})
    at = (torch.arange(S, device="cuda") * 37 - 400).expand(B, S)      # positions below zero too
    y = rope(x, positions=at)
    f = rope.attention_factor
    assert f > 1
    _check(y, x, _reference(x, at, rope.inv_freq, traditional, f, False), f)
    back = rope(y, positions=at, inverse=True)
    _check(back, y, _reference(y, at, rope.inv_freq, traditional, 1 / f, True), f)
    # the transposed map is the gradient: <R x, u> = <x, R^T u>
    u = _rows(B, H, S, D, dtype, 4, "dense")
    ru = K.rotary_embed(u, inv_freq=rope.inv_freq, positions=at, traditional=traditional, attention_factor=f, inverse=True)
    xx = x.double().requires_grad_()
    t = at.double()[:, None, :, None] * rope.inv_freq
    c, s = f * t.cos(), f * t.sin()
    lo, hi = (slice(0, 48, 2), slice(1, 48, 2)) if traditional else (slice(0, 24), slice(24, 48))
    a, b = xx[..., lo], xx[..., hi]
    ((a * c - b * s) * u[..., lo].double() + (b * c + a * s) * u[..., hi].double()).sum().add((xx[..., 48:] * u[..., 48:].double()).sum()).backward()
    _check(ru, u, xx.grad, f)


@pytest.mark.parametrize("traditional,D,dims", [(False, 128, 128), (True, 128, 64), (False, 20, 12)])
def test_outputs_in_place_and_in_a_cache(traditional, D, dims):
    require_gpu()
    B, Hq, Hk, S = 2, 8, 2, 19
    rows = torch.randn((B, S, (Hq + 2 * Hk) * D), device="cuda", dtype=torch.float32).half()
    q = rows[..., : Hq * D].view(B, S, Hq, D).transpose(1, 2)
    k = rows[..., Hq * D: (Hq + Hk) * D].view(B, S, Hk, D).transpose(1, 2)
    v = rows[..., (Hq + Hk) * D:].clone()
    rope = RotaryPositions(dims, traditional=traditional)
    want = rope(q, k, offset=5)
    buf = torch.full((B, Hk, 64, D), 7.0, device="cuda", dtype=torch.float16)
    q2, k2 = rope(q, k, offset=5, k_out=buf[:, :, 11:11 + S])      # rows of a cache
    assert torch.equal(q2, want[0]) and torch.equal(k2, want[1]) and k2.data_ptr() == buf[:, :, 11:].data_ptr()
    assert bool((buf[:, :, :11] == 7).all()) and bool((buf[:, :, 11 + S:] == 7).all())
    got = rope(q, k, offset=5, out=q, k_out=k)                    # views of one projection, turned where they are
    assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(rows[..., (Hq + Hk) * D:], v)


def test_empty_and_refusals():
    require_gpu()
    rope = RotaryPositions(8)
    x = torch.randn(2, 3, 4, 8, device="cuda")
    assert rope(x[:, :, :0]).shape == (2, 3, 0, 8) and rope(x[:, :0], x)[1].shape == x.shape
    assert torch.equal(rope(x[:, :0], x)[1], rope(x))
    f = rope.inv_freq
    buf = torch.zeros(2, 3, 8, 8, device="cuda")
    for kw, what in [
            (dict(q=x.double()), "dtype"), (dict(q=x, k=x.half()), "k must be"), (dict(q=x, k=x[:1]), "k must be"), (dict(q=x, inv_freq=f.half()), "inv_freq"),
            (dict(q=x, inv_freq=torch.ones(5, device="cuda")), "channels of 8"), (dict(q=x, inv_freq=f[:0]), "channels of 8"),
            (dict(q=x, offset=torch.zeros(3, dtype=torch.int64, device="cuda")), "offset must"), (dict(q=x, offset=torch.zeros(2, device="cuda")), "int32 or int64"),
            (dict(q=x, offset=torch.zeros(2, dtype=torch.int64)), "on cuda"), (dict(q=x, positions=torch.zeros(3, dtype=torch.int64, device="cuda")), "positions must"),
            (dict(q=x, positions=torch.zeros(4, dtype=torch.int64, device="cuda"), offset=torch.zeros(2, dtype=torch.int64, device="cuda")), "offset is an int"),
            (dict(q=x, out=x.half()), "output for q"), (dict(q=x, out=x[..., :0]), "output for q"), (dict(q=x, out=buf[:, :1, :4].expand(2, 3, 4, 8)), "share memory"),
            (dict(q=buf[:, :, :4], out=buf[:, :, 2:6]), "overlaps"), (dict(q=x, k=x.clone(), out=buf[:, :, :4], k_out=buf[:, :, :4]), "overlaps"),
            (dict(q=x, k=buf[:, :, :4], out=buf[:, :, :4]), "overlaps")]:
        with pytest.raises(ValueError, match=what):
            K.rotary_embed(**{"inv_freq": f, **kw})


def test_streams_and_graph():
    require_gpu()
    rope = RotaryPositions(128)
    q, k = _rows(1, 32, 1, 128, torch.bfloat16, 5, "dense"), _rows(1, 8, 1, 128, torch.bfloat16, 6, "dense")
    at = torch.tensor([41], device="cuda")
    out, k_out = torch.empty_like(q), torch.empty_like(k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rope(q, k, offset=at, out=out, k_out=k_out)
    torch.cuda.current_stream().wait_stream(side)
    want = rope(q, k, offset=41)
    assert torch.equal(out, want[0]) and torch.equal(k_out, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope(q, k, offset=at, out=out, k_out=k_out)
    for step in (42, 1000000, 7):      # the position is read when the graph runs
        at.fill_(step)
        graph.replay()
        want = rope(q, k, offset=step)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(k_out, want[1])
