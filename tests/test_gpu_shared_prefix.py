"""``shared_prefix_attend`` against attention over the concatenated slots in 64 bits."""

import math

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests._spans import attend, close, seen, store
from veloxquant_mlx_amd import kernels as K

pytestmark = gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _weights_rounding(dtype, packed):
    """Weights are rounded to the type of the products: fp16 over packed slots, else that of the rows; float32 rows: not at all."""
    return 0.0 if dtype == F32 else torch.finfo(F16 if packed else dtype).eps / 2


def _case(B, Hq, Hkv, D, prefix, own, Sq=1, *, bits=4, group=32, v_layout="token", dtype=F16, meta=F16, causal=True, lens=None, window=0,
          spare=40, view=False, seed=0):
    kw = dict(bits=bits, group=group, v_layout=v_layout, dtype=dtype, meta=meta, spare=spare, view=view)
    p, pk, pv = store(1, Hkv, *prefix, D, seed=seed + 1, **kw)
    o, ok, ov = store(B, Hkv, *own, D, seed=seed + 2, **kw)
    q = torch.randn((B, Hq, Sq, D), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)
    scale = 1 / math.sqrt(D)
    lens = None if lens is None else torch.tensor(lens, device="cuda")
    got = K.shared_prefix_attend(q, p, **o, scale=scale, causal=causal, seq_lens=lens, sliding_window=window)
    mask = seen(B, Sq, pk.shape[2], ok.shape[2], lens, causal, window)
    want, far = attend(q, torch.cat([pk.expand(B, -1, -1, -1), ok], 2), torch.cat([pv.expand(B, -1, -1, -1), ov], 2), mask, scale,
                       _weights_rounding(dtype, prefix[0] + own[0] > 0))
    assert got.shape == q.shape and got.dtype == q.dtype
    close(got, want, far)
    return q, p, o, got


@pytest.mark.parametrize("bits,group", [(2, 32), (4, 32), (4, 64), (2, 128)])
@pytest.mark.parametrize("B,Hq,Hkv,D,prefix,own", [
    (1, 1, 1, 128, (128, 0), (0, 1)), (3, 8, 2, 128, (256, 7), (0, 33)), (5, 12, 4, 256, (640, 60), (128, 130)), (2, 14, 2, 64, (384, 1), (128, 5)),
    (7, 32, 8, 128, (1152, 129), (256, 64)), (2, 4, 4, 128, (128, 0), (128, 0)), (33, 7, 1, 128, (128, 63), (0, 2))])
def test_packed(B, Hq, Hkv, D, prefix, own, bits, group):
    require_gpu()
    if group > D:
        pytest.skip("value groups are at most a head")
    _case(B, Hq, Hkv, D, prefix, own, bits=bits, group=group)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("B,Hq,Hkv,D,n,own,Sq", [
    (1, 2, 1, 128, 1, 1, 1), (4, 8, 2, 64, 65, 31, 1), (2, 9, 3, 128, 257, 100, 5), (3, 12, 4, 256, 500, 64, 3), (2, 6, 3, 80, 70, 9, 2),
    (6, 40, 10, 128, 1000, 1, 1), (130, 4, 1, 64, 97, 3, 1), (2, 4, 2, 128, 300, 200, 200), (1, 64, 1, 128, 130, 40, 7)])
def test_plain_rows(dtype, B, Hq, Hkv, D, n, own, Sq):
    require_gpu()
    _case(B, Hq, Hkv, D, (0, n), (0, own), Sq, dtype=dtype, view=True)


@pytest.mark.parametrize("kw", [
    dict(Hq=8, D=128, own=(512, 70), bits=4), dict(Hq=8, D=64, own=(256, 33), bits=2), dict(Hq=4, D=256, own=(256, 40)), dict(Hq=40, D=128, own=(512, 40), Sq=3),
    dict(Hq=8, D=128, own=(0, 200), dtype=BF16), dict(Hq=8, D=128, own=(0, 200), dtype=BF16, Sq=70), dict(Hq=8, D=80, own=(256, 33)),
    dict(Hq=8, D=128, own=(128, 50), dtype=BF16), dict(Hq=8, D=128, own=(128, 50), v_layout="channel")])
@pytest.mark.parametrize("prefix", [(0, 0), (1536, 20)])
def test_nothing_behind_a_sequence_counts(kw, prefix):
    """Rows, scales and zeros behind a sequence's length may be NaN: the same bits, both operators."""
    require_gpu()
    kw = dict(bits=4, group=32, v_layout="token", dtype=F16, Sq=1) | kw
    Hq, D, own, Sq, dtype, Hkv = kw.pop("Hq"), kw.pop("D"), kw.pop("own"), kw.pop("Sq"), kw["dtype"], 2
    lens = [0, 1, 31, 32, 33, own[0], own[0] + 1, sum(own) - 1, sum(own), 100]
    B = len(lens)
    if D % kw["group"]:
        kw["group"] = 16
    o, _, _ = store(B, Hkv, *own, D, seed=2, **kw)
    p = store(1, Hkv, *prefix, D, seed=1, **kw)[0] if sum(prefix) else None
    q = torch.randn((B, Hq, Sq, D), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(dtype)
    dead = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in o.items()}
    for b, n in enumerate(lens):
        tail = max(0, n - own[0])
        if own[1]:
            dead["k_tail"][b, :, tail:], dead["v_tail"][b, :, tail:] = float("nan"), float("nan")
        if own[0]:
            group = -(-n // kw["group"])
            for name in ("k_scale", "k_zero"):
                dead[name][b, :, group:] = float("nan")
            for name in ("v_scale", "v_zero"):
                (dead[name][b, ..., n:] if kw["v_layout"] == "token" else dead[name][b, :, n:]).fill_(float("nan"))
    at = torch.tensor(lens, device="cuda")
    for causal in (False, True):
        call = dict(scale=0.1, causal=causal, seq_lens=at)
        if p is not None:
            one, two = (K.shared_prefix_attend(q, p, **x, **call) for x in (o, dead))
        else:
            one, two = (K.differential_attend(q, 0.4, **x, **call) for x in (o, dead))
        assert bool(one.isfinite().all()) and torch.equal(one, two)


def test_float32_scales_near_zero():
    """code * scale + zero of float32 scales is formed with one rounding to float32: a difference of near-equal numbers, seen alone through a
    window of one slot, is the fp16 number nearest to it."""
    require_gpu()
    _case(1, 6, 2, 200, (2192, 700), (48, 65), 130, group=16, v_layout="channel", dtype=BF16, meta=F32, window=1, spare=0, view=True, seed=253)


@pytest.mark.parametrize("kw", [
    dict(B=40, Hq=8, Hkv=2, D=128, prefix=(1024, 70), own=(256, 33), bits=4), dict(B=40, Hq=8, Hkv=2, D=64, prefix=(640, 3), own=(128, 1), bits=2),
    dict(B=24, Hq=12, Hkv=3, D=128, prefix=(2048, 0), own=(512, 9), bits=4, group=64, lens=[(b * 97) % 522 for b in range(24)]),
    dict(B=70, Hq=4, Hkv=4, D=128, prefix=(384, 5), own=(128, 20), bits=2, window=150), dict(B=20, Hq=6, Hkv=2, D=256, prefix=(512, 40), own=(128, 9)),
    dict(B=9, Hq=16, Hkv=2, D=128, prefix=(512, 1), own=(128, 30), Sq=5, dtype=BF16), dict(B=33, Hq=2, Hkv=2, D=128, prefix=(0, 90), own=(128, 30)),
    dict(B=3, Hq=16, Hkv=2, D=128, prefix=(4096, 0), own=(0, 140), Sq=7, group=128), dict(B=30, Hq=9, Hkv=3, D=128, prefix=(1536, 20), own=(256, 9)),
    dict(B=61, Hq=8, Hkv=2, D=256, prefix=(1280, 5), own=(128, 40), bits=2), dict(B=9, Hq=8, Hkv=2, D=64, prefix=(1280, 0), own=(640, 33), Sq=9, window=700)])
def test_prefixes_of_many_rows(kw):
    """The prefix under the rows of all sequences, next to own slots under few rows, with lengths and windows that leave runs empty."""
    require_gpu()
    _case(**kw)


@pytest.mark.parametrize("prefix,own,B", [((0, 90), (0, 40), 2), ((1024, 70), (256, 33), 40), ((4096, 0), (128, 3), 2), ((512, 0), (0, 9), 2)])
def test_a_query_of_nan_is_nan_and_alone(prefix, own, B):
    """Its row, however the slots are cut, and no other."""
    require_gpu()
    p, _, _ = store(1, 2, *prefix, 128, seed=1)
    o, _, _ = store(B, 2, *own, 128, seed=2)
    q = torch.randn((B, 8, 1, 128), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").half()
    clean = K.shared_prefix_attend(q, p, **o, scale=0.1)
    q[1, 3, 0, 5] = float("nan")
    got = K.shared_prefix_attend(q, p, **o, scale=0.1)
    assert bool(got[1, 3].isnan().all())
    got[1, 3] = clean[1, 3]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("kw", [
    dict(bits=3, group=32, v_layout="channel"), dict(bits=8, group=32), dict(bits=1, group=32), dict(bits=4, v_layout="channel"),
    dict(bits=4, meta=F32), dict(bits=4, group=16), dict(bits=4, dtype=F32), dict(bits=4, dtype=BF16), dict(bits=2, dtype=BF16, group=64)])
def test_other_stores(kw):
    require_gpu()
    _case(3, 8, 2, 128, (256, 9), (128, 20), 2, **kw)


@pytest.mark.parametrize("dtype,prefix,own", [(F16, (256, 10), (64, 50)), (BF16, (0, 300), (0, 114)), (F32, (64, 9), (32, 40))])
@pytest.mark.parametrize("causal,window,lens,Sq", [
    (False, 0, None, 4), (True, 0, [114, 1, 57], 1), (True, 0, [114, 3, 57], 4), (True, 0, [0, 114, 64], 1), (True, 0, [2, 0, 63], 6),
    (False, 0, [0, 114, 65], 3), (True, 50, None, 4), (True, 200, [114, 1, 60], 2), (False, 100, [114, 20, 60], 2), (True, 1, [0, 5, 114], 1),
    (True, 0, [-3, 500, 114], 1)])
def test_masks(dtype, prefix, own, causal, window, lens, Sq):
    require_gpu()
    if dtype == F32:
        lens = None if lens is None else [min(n, 72) for n in lens]
    _case(3, 8, 2, 128, prefix, own, Sq, dtype=dtype, causal=causal, window=window, lens=lens)


def test_without_own_slots_or_without_a_prefix():
    require_gpu()
    _case(3, 8, 2, 128, (256, 9), (0, 0), causal=False)
    _case(3, 8, 2, 128, (0, 0), (128, 9), 3)
    _case(2, 8, 2, 128, (0, 0), (0, 40), lens=[0, 40])       # a sequence that sees nothing: zero
    q, p, o, got = _case(2, 8, 2, 128, (0, 0), (0, 40), lens=[0, 40], seed=5)
    assert bool((got[0] == 0).all())


def test_far_scores_and_equal_ones():
    """Rows whose scores lie hundreds apart, and rows of equal scores."""
    require_gpu()
    B, H, D, n = 2, 4, 128, 400
    q = torch.randn((B, H, 1, D), device="cuda").half() * 30
    k, v = torch.randn((1, H, n, D), device="cuda").half() * 5, torch.randn((1, H, n, D), device="cuda").half()
    ok, ov = torch.randn((B, H, 50, D), device="cuda").half(), torch.randn((B, H, 50, D), device="cuda").half()
    got = K.shared_prefix_attend(q, dict(k_tail=k, v_tail=v, n_tail=n), k_tail=ok, v_tail=ov, n_tail=50, scale=1.0)
    mask = torch.ones((B, 1, n + 50), dtype=torch.bool, device="cuda")
    kk, vv = torch.cat([k.expand(B, -1, -1, -1), ok], 2).double(), torch.cat([v.expand(B, -1, -1, -1), ov], 2).double()
    close(got, *attend(q, kk, vv, mask, 1.0, 2.0 ** -11))
    got = K.shared_prefix_attend(q * 0, dict(k_tail=k, v_tail=v, n_tail=n), k_tail=ok, v_tail=ov, n_tail=50, scale=1.0)
    close(got, *attend(q * 0, kk, vv, mask, 1.0, 2.0 ** -11))


@pytest.mark.parametrize("packed,dtype,G", [(True, F16, 1), (True, F16, 40), (False, F16, 1), (False, F16, 40), (False, BF16, 1)])
def test_many_small_weights_count(packed, dtype, G):
    """One slot takes the maximum, 2^13 others weigh 2^-25.3 of it each, and are what the result is made of.  A weight of fp16 is off by at
    most half a step, 2^-11 of itself or 2^-32 of the largest.  (Enough sequences and heads that a row's slots are not cut into runs, of
    which each would have a maximum of its own.)"""
    require_gpu()
    B, H, D, n = 64, 8, 64, 1 << 13
    k, v = torch.zeros((B, H, n, D), dtype=dtype, device="cuda"), torch.ones((B, H, n, D), dtype=dtype, device="cuda")
    k[:, :, 70, 0], v[:, :, 70] = 1.0, 0.0
    scale = 25.3 * math.log(2.0) / 8
    q = torch.zeros((B, H * G, 1, D), dtype=dtype, device="cuda")
    q[..., 0] = 8.0
    peak = 1.0
    if packed:
        kq, vq = K.kivi_quant_pack(k, -2, 32, 4, meta_dtype=F16), K.kivi_quant_pack(v, -1, 32, 4, meta_dtype=F16, v_layout="token")
        own = dict(k_packed=kq[0], k_scale=kq[1], k_zero=kq[2], v_packed=vq[0], v_scale=vq[1], v_zero=vq[2], n_packed=n, bits=4, group_size=32, v_layout="token")
        peak = float((15 * kq[1][0, 0, 70 // 32, 0].double()).half())
    else:
        own = dict(k_tail=k, v_tail=v, n_tail=n)
    got = K.shared_prefix_attend(q, dict(n_tail=0), **own, scale=scale)
    small = math.exp(-8.0 * peak * scale)
    want = (n - 1) * small / (1 + (n - 1) * small)
    u = torch.finfo(dtype).eps / 2
    far = want * (2 * u + 16 * 2.0 ** -18) + (0 if dtype == BF16 else n * 2.0 ** -32) + u * want + torch.finfo(dtype).smallest_normal * u
    assert float((got.double() - want).abs().max()) <= far


@pytest.mark.parametrize("Sq", [1, 40])
@pytest.mark.parametrize("packed", [True, False])
def test_offsets_past_32_bits(packed, Sq):
    """The second kv head's slots lie more than 4 GiB behind the first's; a window over the last ones, behind which little is read."""
    require_gpu()
    Hq, Hkv, D, window, last = 4, 2, 128, 300, 1024
    p, k, v = store(1, Hkv, *((last, 0) if packed else (0, last)), D, bits=4, group=64, seed=5)
    room = 70_000_000 // 64 * 64 if packed else 17_000_000
    if packed:
        for name, axis, per in (("k_packed", 2, 1), ("k_scale", 2, 64), ("k_zero", 2, 64), ("v_packed", 2, 8), ("v_scale", 3, 1), ("v_zero", 3, 1)):
            shape = list(p[name].shape)
            shape[axis] = room // per
            big = torch.empty(shape, dtype=p[name].dtype, device="cuda")
            big.narrow(axis, (room - last) // per, last // per).copy_(p[name])
            p[name] = big
        p["n_packed"] = room
        assert p["k_packed"][:, :1].numel() * 4 > 1 << 32
    else:
        for name in ("k_tail", "v_tail"):
            big = torch.empty((1, Hkv, room, D), dtype=F16, device="cuda")
            big[:, :, -last:] = p[name]
            p[name] = big
        p["n_tail"] = room
        assert p["k_tail"][:, :1].numel() * 2 > 1 << 32
    o, ok, ov = store(2, Hkv, 0, 50, D, seed=6)
    q = torch.randn((2, Hq, Sq, D), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").half()
    got = K.shared_prefix_attend(q, p, **{**o, "bits": 4, "group_size": 64}, scale=0.1, causal=True, sliding_window=window)
    ks, vs = (torch.cat([x.expand(2, -1, -1, -1), y], 2) for x, y in ((k, ok), (v, ov)))
    want, far = attend(q, ks, vs, seen(2, Sq, last, 50, None, True, window), 0.1, torch.finfo(F16).eps / 2)
    close(got, want, far)


def test_agrees_with_the_cache_held_per_sequence():
    """The same slots, the prefix copied into every sequence, through the framework's own decode attention."""
    require_gpu()
    B, Hq, Hkv, D, nq = 4, 32, 8, 128, 512
    q, p, o, got = _case(B, Hq, Hkv, D, (nq, 0), (128, 40), spare=0)
    axis = dict(k_packed=2, k_scale=2, k_zero=2, v_packed=2, v_scale=3, v_zero=3)
    both = {n: torch.cat([p[n].expand(B, -1, -1, -1), o[n]], ax).contiguous() for n, ax in axis.items()}
    ref = K.kivi_packed_attend(q, **both, n_packed=nq + 128, bits=4, group_size=32, v_layout="token", k_tail=o["k_tail"], v_tail=o["v_tail"],
                               n_tail=40, scale=1 / math.sqrt(D))
    assert float((got.float() - ref.float()).abs().max()) <= 2e-3 * max(1.0, float(ref.abs().max()))


def test_streams_graphs_and_out():
    require_gpu()
    B, Hq, Hkv, D = 6, 32, 8, 128
    q, p, o, got = _case(B, Hq, Hkv, D, (512, 20), (128, 40))
    call = dict(scale=1 / math.sqrt(D), causal=True)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.shared_prefix_attend(q, p, **o, **call, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, got)
    # two graphs captured one after the other and replayed at once share no scratch, nor does an eager call between
    lens = torch.full((B,), 168, device="cuda")
    outs = [torch.empty_like(q), torch.empty_like(q)]
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.shared_prefix_attend(q if i == 0 else -q, p, **o, **call, seq_lens=lens, out=outs[i])
        graphs.append(g)
    for n in (168, 5, 130, 0):
        lens.fill_(n)
        torch.cuda.synchronize()
        for t in outs:
            t.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        eager = K.shared_prefix_attend(q, p, **o, **call, seq_lens=lens)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(outs[0], eager)
        assert torch.equal(outs[1], K.shared_prefix_attend(-q, p, **o, **call, seq_lens=lens))
        torch.cuda.synchronize()


def test_rows_of_sequences_do_not_depend_on_each_other():
    require_gpu()
    q, p, o, got = _case(9, 8, 2, 128, (512, 3), (128, 17))
    flip = {n: (t.flip(0) if isinstance(t, torch.Tensor) else t) for n, t in o.items()}
    again = K.shared_prefix_attend(q.flip(0), p, **flip, scale=1 / math.sqrt(128), causal=True)
    assert torch.equal(again.flip(0), got)


def test_refusals():
    require_gpu()
    q, p, o, _ = _case(2, 8, 2, 128, (256, 9), (128, 20))
    ok = dict(scale=0.1)
    bf = {n: (t.to(BF16) if n in ("k_tail", "v_tail") else t) for n, t in o.items()}
    for args, what in [
            ((q[0], p, o), "4D"), ((q.double(), p, o), "dtype"), ((q[..., :64], p, o), "channels"), ((q[:, :3], p, o), "kv heads"),
            ((q[:1], p, o), "batch"), ((q, {**p, "k_scale": None}, o), "must be given"), ((q, {**p, "group_size": 64}, o), "do not fit"),
            ((q, {**p, "n_packed": 9999}, o), "do not fit"), ((q, p, {**o, "n_tail": 9999}), "does not fit"), ((q, p, {**o, "v_layout": "x"}), "v_layout"),
            ((q, p, bf), "differ in plain rows"), ((q, {**p, "k_zero": p["k_zero"].float()}, o), "share one dtype"),
            ((q, o, o), "batch"), ((q, p, {**o, "v_tail": o["v_tail"][:, :1]}), "alike"), ((q, p, {**o, "k_packed": o["k_packed"].cpu()}), "must live"),
            ((q, {}, {}), "no key/value slots"), ((q, p, {**o, "n_tail": -1}), "negative")]:
        with pytest.raises(ValueError, match=what):
            K.shared_prefix_attend(args[0], args[1], **args[2], **ok)
    p2 = store(1, 2, 256, 9, 128, bits=2)[0]
    with pytest.raises(ValueError, match="differ in bits"):
        K.shared_prefix_attend(q, p2, **o, **ok)
    for extra, what in [(dict(seq_lens=torch.ones(3, dtype=torch.int64, device="cuda")), "seq_lens"), (dict(seq_lens=torch.ones(2, device="cuda")), "seq_lens"),
                        (dict(out=q[:, :, :, ::2]), "out must"), (dict(out=torch.empty_like(q, dtype=F32)), "out must"), (dict(sliding_window=-1), "window")]:
        with pytest.raises(ValueError, match=what):
            K.shared_prefix_attend(q, p, **o, **{**ok, **extra})
    long = torch.zeros((2, 8, 500, 128), dtype=F16, device="cuda")
    with pytest.raises(ValueError, match="exceeds"):
        K.shared_prefix_attend(long, p, **o, **ok, causal=True)
    assert K.shared_prefix_attend(q[:, :, :0], p, **o, **ok).shape == (2, 8, 0, 128)
