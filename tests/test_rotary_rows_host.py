"""Which rows ``rotary_embed`` takes as outputs (no GPU): tensors that share no byte, however their rows lie between each other."""

import random

import pytest
import torch

from veloxquant_mlx_amd import _lib, kernels as K


def _bytes(t):
    at = torch.zeros(1, dtype=torch.int64)
    for n, st in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n) * st).reshape(-1)
    at = t.data_ptr() + at * t.element_size()
    return set((at[:, None] + torch.arange(t.element_size())).reshape(-1).tolist())


def test_tensors_that_are_found_apart_share_no_byte():
    """Any two strided views of one buffer, against the set of their bytes."""
    rng = random.Random(5)
    buf = torch.zeros(4096, dtype=torch.float16)
    found = shared = 0
    for _ in range(4000):
        views = []
        for _ in range(2):
            shape = [rng.choice((1, 2, 3, 4)) for _ in range(3)] + [rng.choice((1, 2, 4, 8))]
            strides = [rng.choice((0, 4, 8, 12, 16, 24, 32, 48, 64, 96)) for _ in range(3)] + [1]
            at = buf.as_strided(shape, strides, rng.randrange(0, 200))
            views.append(at.view(torch.int16) if rng.random() < 0.3 else at)
        apart, meet = K._apart(*views), bool(_bytes(views[0]) & _bytes(views[1]))
        assert not (apart and meet), views
        assert K._apart(*views[::-1]) in (apart, not meet)
        found, shared = found + apart, shared + meet
    assert found > 1000 and shared > 1000


def _projection(B, S, Hq, Hk, D):
    rows = torch.zeros((B, S, (Hq + 2 * Hk) * D), dtype=torch.float16)
    part = lambda lo, H: rows[..., lo * D:(lo + H) * D].view(B, S, H, D).transpose(1, 2)
    return part(0, Hq), part(Hq, Hk), part(Hq + Hk, Hk)


@pytest.mark.parametrize("B,S", [(1, 1), (2, 1), (1, 7), (2, 5), (3, 33)])
@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 16), (4, 4, 8), (1, 1, 64)])
def test_views_of_one_projection_are_apart(B, S, Hq, Hk, D):
    q, k, v = _projection(B, S, Hq, Hk, D)
    for a in (q, k, v):
        for b in (q, k, v):
            assert K._apart(a, b) == (a is not b)
    # heads of queries, keys and values one after the other; halves of a buffer of heads
    rows = torch.zeros((B, S, Hk, 3, D), dtype=torch.float16)
    a, b, c = (rows[..., i, :].transpose(1, 2) for i in range(3))
    assert K._apart(a, b) and K._apart(c, a) and not K._apart(b, b)
    heads = torch.zeros((B, Hq + Hk, S, D), dtype=torch.float16)
    assert K._apart(heads[:, :Hq], heads[:, Hq:]) and not K._apart(heads[:, :Hq], heads[:, Hq - 1:])


@pytest.fixture
def calls(monkeypatch):
    """Host tensors up to the library's call, which is counted."""
    seen = []

    class Library:
        @staticmethod
        def rotary_packed(args, stream):
            seen.append(args)
            return 0

    monkeypatch.setattr(K, "_need_gpu", lambda *a: None)
    monkeypatch.setattr(K, "_stream_of", lambda device: 0)
    monkeypatch.setattr(K, "_launch_on", lambda device, call: call())
    monkeypatch.setattr(_lib, "load", lambda: Library)
    return seen


@pytest.mark.parametrize("B,S", [(1, 1), (2, 1), (1, 9), (2, 9)])
def test_documented_outputs_are_taken(calls, B, S):
    D, Hq, Hk = 16, 4, 2
    f = torch.ones(D // 2)
    cache = torch.zeros((B, Hk, 40, D), dtype=torch.float16)[:, :, 11:11 + S]
    dense = torch.zeros((B, Hq, S, D), dtype=torch.float16)
    q, k, v = _projection(B, S, Hq, Hk, D)
    for out, k_out in ((q, k), (q, cache), (q, None), (None, k), (dense, k), (dense, cache), (None, v), (q, v)):
        got = K.rotary_embed(q, k, inv_freq=f, out=out, k_out=k_out)
        assert (out is None or got[0] is out) and (k_out is None or got[1] is k_out)
    K.rotary_embed(k, q, inv_freq=f, out=k, k_out=q)
    K.rotary_embed(q[:, :, :0], k[:, :, :0], inv_freq=f, out=q[:, :, :0], k_out=q[:, :2, :0])
    assert len(calls) == 9


def test_outputs_that_meet_other_rows_are_refused(calls):
    f = torch.ones(8)
    q, k, v = _projection(2, 9, 4, 2, 16)
    for kw in (dict(out=q, k_out=q[:, :2]), dict(k_out=q[:, 2:]), dict(out=q.clone(), k_out=q[:, 1:3])):
        with pytest.raises(ValueError, match="overlaps"):
            K.rotary_embed(q, k, inv_freq=f, **kw)
    x = torch.zeros((2, 4, 9, 16), dtype=torch.float16)
    for args in (dict(q=x, k=x, out=x, k_out=x), dict(q=x, k=x[:, 1:2], out=x, k_out=x[:, 1:2]), dict(q=x, k=x, out=x), dict(q=x, k=x, k_out=x),
                 dict(q=x[:, :, :8], out=x[:, :, 1:]), dict(q=x[:, :3], out=x[:, 1:]), dict(q=x, k=k.repeat(1, 2, 1, 1), out=q, k_out=q)):
        with pytest.raises(ValueError, match="overlaps"):
            K.rotary_embed(**args, inv_freq=f)
    assert not calls


def test_outputs_whose_rows_share_memory_are_refused(calls):
    f, buf = torch.ones(8), torch.zeros(8192)
    x = torch.zeros((2, 3, 5, 16))
    for strides in ((240, 80, 8, 1), (240, 80, 15, 1), (240, 0, 16, 1), (240, 79, 16, 1), (239, 80, 16, 1), (80, 80, 16, 1)):
        with pytest.raises(ValueError, match="share memory"):
            K.rotary_embed(x, inv_freq=f, out=buf.as_strided(x.shape, strides))
        with pytest.raises(ValueError, match="share memory"):
            K.rotary_embed(x, x.clone(), inv_freq=f, k_out=buf.as_strided(x.shape, strides))
    for strides in ((240, 80, 16, 1), (16, 32, 96, 1), (48, 16, 96, 1), (1000, 17, 60, 1), (16, 160, 32, 1)):
        K.rotary_embed(x, inv_freq=f, out=buf.as_strided(x.shape, strides))
    K.rotary_embed(x[:1, :1], inv_freq=f, out=buf.as_strided((1, 1, 5, 16), (0, 0, 16, 1)))   # strides that nothing walks
    assert len(calls) == 6
