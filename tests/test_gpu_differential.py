"""``differential_attend`` against the difference of two softmax maps in 64 bits."""

import math

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests._spans import attend, close, seen, store
from veloxquant_mlx_amd import kernels as K

pytestmark = gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def reference(q, k, v, lam, mask, scale, u, weight=None, eps=1e-5, gain=1.0):
    """The result in 64 bits and how far a kernel may be from it: both maps' distances, carried through the norm (its divisor moves by
    at most the root mean square of the distances)."""
    h = q.shape[3] // 2
    lam = (lam if isinstance(lam, torch.Tensor) else torch.tensor([float(lam)], device="cuda")).double().view(1, -1, 1, 1)
    (o1, f1), (o2, f2) = (attend(q[..., half], k[..., half], v, mask, scale, u) for half in (slice(0, h), slice(h, None)))
    o, far = o1 - lam * o2, f1 + lam.abs() * f2 + 2.0 ** -22 * (o1.abs() + lam.abs() * o2.abs())
    if weight is None:
        return o * gain, far * abs(gain)
    r = (o.square().mean(-1, keepdim=True) + eps).sqrt()
    dr = far.square().mean(-1, keepdim=True).sqrt() / r
    w = gain * weight.double()
    return o / r * w, (far / r + o.abs() / r * (dr + 2.0 ** -20)) * w.abs() / (1 - dr).clamp_min(0.5)


def _case(B, Hq, Hkv, D, slots, Sq=1, *, bits=4, group=32, v_layout="token", dtype=F16, meta=F16, causal=True, lens=None, window=0, norm=True,
          lam=None, spare=40, view=False, seed=0, norm_dtype=F32, gain=0.2):
    s, k, v = store(B, Hkv, *slots, D, bits=bits, group=group, v_layout=v_layout, dtype=dtype, meta=meta, spare=spare, view=view, seed=seed + 1)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn((B, Hq, Sq, D), generator=g, device="cuda").to(dtype)
    lam = torch.rand(Hq, generator=g, device="cuda") * 0.6 + 0.2 if lam is None else lam
    weight = (torch.rand(D, generator=g, device="cuda") + 0.5).to(norm_dtype) if norm else None
    scale = 1 / math.sqrt(D // 2)
    lens = None if lens is None else torch.tensor(lens, device="cuda")
    got = K.differential_attend(q, lam, **s, scale=scale, causal=causal, seq_lens=lens, sliding_window=window, norm_weight=weight, gain=gain)
    u = 0.0 if dtype == F32 else torch.finfo(F16 if slots[0] else dtype).eps / 2
    want, far = reference(q, k, v, lam, seen(B, Sq, 0, k.shape[2], lens, causal, window), scale, u, weight, 1e-5, gain)
    assert got.shape == q.shape and got.dtype == q.dtype
    close(got, want, far)
    return q, lam, s, weight, got


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("B,Hq,Hkv,D,n,Sq", [
    (1, 1, 1, 128, 1, 1), (2, 8, 2, 128, 65, 65), (1, 9, 3, 64, 200, 200), (3, 12, 4, 256, 130, 130), (2, 6, 2, 80, 40, 40), (1, 32, 8, 128, 500, 1),
    (2, 7, 7, 128, 300, 33), (1, 4, 1, 256, 257, 1), (1, 40, 10, 128, 127, 127), (1, 16, 1, 128, 96, 5)])
def test_plain_rows(dtype, norm, B, Hq, Hkv, D, n, Sq):
    require_gpu()
    _case(B, Hq, Hkv, D, (0, n), Sq, dtype=dtype, norm=norm, view=True)


@pytest.mark.parametrize("bits,group", [(2, 32), (4, 32), (4, 64), (2, 128)])
@pytest.mark.parametrize("B,Hq,Hkv,D,slots,Sq", [
    (1, 4, 4, 128, (128, 0), 1), (2, 32, 8, 128, (1152, 129), 1), (3, 12, 4, 256, (640, 60), 1), (2, 14, 2, 64, (384, 1), 2), (1, 8, 2, 128, (256, 100), 70)])
def test_packed(B, Hq, Hkv, D, slots, Sq, bits, group):
    require_gpu()
    if group > D:
        pytest.skip("value groups are at most a head")
    _case(B, Hq, Hkv, D, slots, Sq, bits=bits, group=group)


@pytest.mark.parametrize("kw", [
    dict(bits=3, v_layout="channel"), dict(bits=8), dict(bits=1), dict(bits=4, v_layout="channel"), dict(bits=4, meta=F32), dict(bits=4, group=16),
    dict(bits=4, dtype=F32), dict(bits=4, dtype=BF16), dict(lam=0.35), dict(lam=0.0), dict(norm_dtype=BF16), dict(norm=False, gain=3.0)])
def test_other_arguments(kw):
    require_gpu()
    _case(2, 8, 2, 128, (256, 29), 2, **kw)


@pytest.mark.parametrize("dtype,slots", [(F16, (256, 58)), (BF16, (0, 314)), (F32, (64, 250))])
@pytest.mark.parametrize("causal,window,lens,Sq", [
    (False, 0, None, 4), (True, 0, [314, 1, 157], 1), (True, 0, [314, 3, 257], 4), (True, 0, [0, 314, 64], 1), (True, 0, [2, 0, 63], 6),
    (False, 0, [0, 314, 65], 3), (True, 50, None, 300), (True, 200, [314, 1, 260], 2), (False, 100, [314, 20, 60], 2), (True, 1, None, 3)])
def test_masks(dtype, slots, causal, window, lens, Sq):
    require_gpu()
    q, lam, s, w, got = _case(3, 8, 2, 128, slots, Sq, dtype=dtype, causal=causal, window=window, lens=lens)
    if lens is not None:
        for b, n in enumerate(lens):
            empty = Sq - n if causal else Sq if n == 0 else 0      # the first queries of a short sequence see nothing
            if empty > 0:
                assert bool((got[b, :, :empty] == 0).all())


def test_one_tensor_lam_streams_and_graph():
    require_gpu()
    q, lam, s, w, _ = _case(2, 8, 2, 128, (256, 58), 1)
    one = torch.tensor([0.4], device="cuda")
    call = dict(scale=0.125, causal=True, norm_weight=w)
    assert torch.equal(K.differential_attend(q, one, **s, **call), K.differential_attend(q, 0.4, **s, **call))
    assert torch.equal(K.differential_attend(q, one, **s, **call), K.differential_attend(q, one.expand(8).contiguous(), **s, **call))
    out, lens = torch.empty_like(q), torch.full((2,), 314, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.differential_attend(q, lam, **s, **call, seq_lens=lens, out=out)
    for n in (314, 200, 1, 300):
        lens.fill_(n)
        g.replay()
        assert torch.equal(out, K.differential_attend(q, lam, **s, **call, seq_lens=lens))
        torch.cuda.synchronize()


def test_refusals():
    require_gpu()
    q, lam, s, w, _ = _case(2, 8, 2, 128, (256, 29), 2)
    for kw, what in [(dict(lam=lam.half()), "lam"), (dict(lam=lam[:5]), "lam"), (dict(lam=lam.cpu()), "lam"), (dict(norm_weight=w[:64]), "norm_weight"),
                     (dict(norm_weight=w.cpu()), "norm_weight"), (dict(norm_weight=w.double()), "dtype"), (dict(q=q[..., :63], n_packed=0, k_tail=s["k_tail"][..., :63], v_tail=s["v_tail"][..., :63]), "even"),
                     (dict(q=q[0]), "4D"), (dict(n_tail=500), "does not fit"), (dict(q=q[:1]), "batch"), (dict(sliding_window=-2), "window")]:
        args = {**dict(q=q, lam=lam, scale=0.1, norm_weight=w), **s, **kw}
        if args["q"].shape[-1] == 63:
            args["norm_weight"] = None
        with pytest.raises(ValueError, match=what):
            K.differential_attend(args.pop("q"), args.pop("lam"), **args)
