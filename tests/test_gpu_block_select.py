"""``select_blocks`` against the same choice by sorting bounds in 64 bits."""

import pytest
import torch

from tests._blocks import choose, group_bounds
from tests._gpu import gpu, require_gpu
from tests._spans import store
from veloxquant_mlx_amd import kernels as K

pytestmark = gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _inputs(B, Hq, Hkv, Sq, D, groups, *, dtype=F16, meta=F16, spare=2, seed=0, signed=False):
    """Queries, scales and zeros; groups past the live ones hold NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn((B, Hq, Sq, D), generator=g, device="cuda").to(dtype)
    factors = torch.randn(D, generator=g, device="cuda").mul(0.5).exp()
    zero = torch.full((B, Hkv, groups + spare, D), float("nan"), dtype=meta, device="cuda")
    scale = zero.clone()
    lo = torch.randn((B, Hkv, groups, D), generator=g, device="cuda") * factors
    width = torch.rand((B, Hkv, groups, D), generator=g, device="cuda") * factors
    if signed:
        width *= torch.randn((B, Hkv, groups, D), generator=g, device="cuda").sign()
    zero[:, :, :groups], scale[:, :, :groups] = lo.to(meta), (width / 4).to(meta)
    return q, scale, zero


def _same(q, scale, zero, n, **kw):
    got = K.select_blocks(q, scale, zero, n, **kw)
    want = choose(q, scale, zero, n, **kw)
    assert got.dtype == torch.int32 and got.shape == want.shape
    assert torch.equal(got, want), (got != want).nonzero()[:3].tolist()
    return got


@pytest.mark.parametrize("dtype,meta", [(F16, F16), (BF16, F16), (F32, F16), (F16, F32), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("B,Hq,Hkv,D,groups,group,block,n", [
    (1, 32, 8, 128, 129, 32, 32, 17), (2, 8, 2, 64, 70, 32, 64, 9), (1, 12, 4, 256, 33, 64, 128, 4), (3, 4, 4, 128, 300, 16, 16, 100),
    (1, 6, 2, 80, 41, 32, 96, 5), (1, 1, 1, 7, 20, 8, 8, 3), (2, 28, 4, 128, 65, 32, 64, 1), (1, 40, 1, 128, 90, 32, 32, 33),
    (1, 2, 1, 256, 700, 32, 32, 300)])
def test_one_query(dtype, meta, B, Hq, Hkv, D, groups, group, block, n):
    require_gpu()
    q, scale, zero = _inputs(B, Hq, Hkv, 1, D, groups, dtype=dtype, meta=meta, seed=groups)
    kw = dict(levels=15, group_size=group, n_packed=groups * group, block_size=block)
    _same(q, scale, zero, n, n_tail=37, causal=True, **kw)
    _same(q, scale, zero, max(n, 3), first=1, recent=2, **kw)


@pytest.mark.parametrize("signed", [False, True])
@pytest.mark.parametrize("levels", [1, 3, 255])
@pytest.mark.parametrize("Sq,query_block", [(5, 1), (5, 5), (13, 4), (64, 16), (3, 40), (70, 64)])
def test_tiles_of_queries(Sq, query_block, levels, signed):
    require_gpu()
    q, scale, zero = _inputs(2, 8, 2, Sq, 128, 60, seed=Sq, signed=signed, dtype=BF16)
    for block, n_tail, causal in ((32, 20, True), (64, 0, True), (64, 90, False), (160, 3, True)):
        _same(q, scale, zero, 6, levels=levels, group_size=32, n_packed=60 * 32, n_tail=n_tail, block_size=block, query_block=query_block, first=1,
              recent=1, causal=causal)


@pytest.mark.parametrize("query_block", [1, 3, 9])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(causal, query_block):
    require_gpu()
    q, scale, zero = _inputs(9, 4, 2, 9, 64, 50, seed=4)
    lens = torch.tensor([0, 1, 8, 9, 32, 33, 800, 1600, 5000], device="cuda")    # none, fewer than the queries, the whole, more than there is
    for first, recent in ((0, 0), (2, 3)):
        got = _same(q, scale, zero, 5, levels=15, group_size=32, n_packed=1600, n_tail=11, query_block=query_block, causal=causal, seq_lens=lens, first=first,
                    recent=recent)
        assert bool((got[0] == -1).all())


def test_a_store_that_ends_inside_a_block():
    require_gpu()
    q, scale, zero = _inputs(2, 8, 2, 3, 128, 21, seed=6)
    for n_packed in (21 * 32, 21 * 32 - 5, 1, 0):
        _same(q, scale, zero, 4, levels=15, group_size=32, n_packed=n_packed, n_tail=7, block_size=128, causal=True)
        _same(q, scale, zero, 4, levels=15, group_size=32, n_packed=n_packed, n_tail=7, block_size=32, causal=True, recent=1)


@pytest.mark.parametrize("n", [1, 7, 64, 255, 256, 257])
def test_equal_scores_go_to_the_lower_block(n):
    require_gpu()
    q, scale, zero = _inputs(1, 4, 2, 1, 64, 600, seed=8, spare=0)
    scale[:], zero[:] = scale[:, :, :1], zero[:, :, :1]
    got = _same(q, scale, zero, n, levels=3, group_size=32, n_packed=600 * 32)
    assert torch.equal(got[0, 0, 0], torch.arange(n, dtype=torch.int32, device="cuda"))
    scale[0, 0, 300:340] *= 2           # some above, the rest alike
    _same(q, scale, zero, n, levels=3, group_size=32, n_packed=600 * 32, first=min(1, n), recent=0)
    zero[:], scale[:] = 0, 0            # zeros of either sign
    zero[0, 0, ::3] = -0.0
    _same(q, scale, zero, n, levels=3, group_size=32, n_packed=600 * 32)


def test_scores_a_hair_apart():
    """Blocks that differ by the last bit of one channel's zero: float32 sums of the others would hide it."""
    require_gpu()
    q, scale, zero = _inputs(1, 4, 1, 1, 128, 256, seed=9, spare=0)
    scale[:], zero[:] = scale[:, :, :1], zero[:, :, :1]
    q[..., 5] = 2.0 ** -12
    zero[..., 5] = 0.25
    up = torch.randperm(256, generator=torch.Generator().manual_seed(1))[:40].cuda()
    zero[0, 0, up, 5] = 0.25 + 2.0 ** -12
    got = _same(q, scale, zero, 40, levels=15, group_size=32, n_packed=256 * 32)
    assert torch.equal(got.flatten().long(), up.sort().values)


@pytest.mark.parametrize("D", [128, 80])
def test_float32_scores_a_hair_apart(D):
    require_gpu()
    q, scale, zero = _inputs(1, 4, 1, 1, D, 256, seed=9, spare=0, dtype=F32, meta=F32)
    scale[:], zero[:] = scale[:, :, :1], zero[:, :, :1]
    q[..., 5] = 2.0 ** -12
    scale[..., 5], zero[..., 5] = 2.0 ** -6, 0.25
    up = torch.randperm(256, generator=torch.Generator().manual_seed(1))[:40].cuda()
    zero[0, 0, up, 5] = 0.25 + 2.0 ** -24      # 2^-36 of a score
    got = _same(q, scale, zero, 40, levels=15, group_size=32, n_packed=256 * 32)
    assert torch.equal(got.flatten().long(), up.sort().values)


@pytest.mark.parametrize("Sq,query_block", [(1, 1), (6, 6)])
def test_values_that_are_not_finite(Sq, query_block):
    require_gpu()
    q, scale, zero = _inputs(2, 4, 2, Sq, 128, 100, seed=10, meta=F32)
    zero[0, 0, 50, 3] = float("nan")
    scale[1, 1, 70, 9] = float("inf")
    zero[0, 1, 20, 100] = float("inf")
    kw = dict(levels=15, group_size=32, n_packed=3200, query_block=query_block)
    got = _same(q, scale, zero, 6, **kw)
    assert 50 in got[0, 0, 0].tolist()
    q[1, 0] = float("nan")          # every score of the kv head: the lowest blocks
    got = _same(q, scale, zero, 6, **kw)
    assert got[1, 0, 0].tolist() == [0, 1, 2, 3, 4, 5]


@pytest.mark.parametrize("what", ["ordinary", "signed", "close", "small", "past fp16", "odd"])
@pytest.mark.parametrize("dtype,D,Sq,query_block,groups", [(F16, 128, 48, 16, 2100), (BF16, 256, 24, 3, 2100), (BF16, 64, 100, 50, 2051)])
def test_many_rows_over_float32_stores(dtype, D, Sq, query_block, groups, what):
    """Sizes from which float32 scales and zeros are looked through rounded to fp16 first."""
    require_gpu()
    q, scale, zero = _inputs(1, 8, 2, Sq, D, groups, dtype=dtype, meta=F32, seed=D, signed=what == "signed")
    assert 8 * Sq * groups * D > 1e8
    if what == "close":         # far less apart than fp16 numbers are
        near = zero[:, :, :1] * (1 + 2.0 ** -16 * torch.rand((1, 2, groups, 1), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda"))
        zero[:, :, :groups], scale[:, :, :groups] = near, scale[:, :, :1].clone()
    elif what == "small":
        zero *= 2.0 ** -30
        scale *= 2.0 ** -30
        q = (q.float() * 2.0 ** -12).to(dtype)
    elif what == "past fp16":
        zero[:, 0] *= 1e6
        scale[0, 1, 77, 3] = 3e38
    elif what == "odd":
        zero[0, 0, 50, 3] = float("nan")
        scale[0, 1, 70, 9] = float("inf")
    lens = torch.tensor([groups * 32 - 100], device="cuda")
    _same(q, scale, zero, 40, levels=15, group_size=32, n_packed=groups * 32, n_tail=9, block_size=64, query_block=query_block, first=1, recent=1, causal=True,
          seq_lens=lens if what == "ordinary" else None)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("big", [2.0 ** 15, 2.0 ** -20])
def test_large_and_small_queries(dtype, big):
    require_gpu()
    q, scale, zero = _inputs(2, 8, 2, 4, 128, 90, dtype=dtype, seed=12)
    q = (q.float() * big).to(dtype)
    q[:, 1] *= 2.0 ** -3
    if dtype == BF16:
        q[0, 2] = (q[0, 2].float() * 2.0 ** 60).to(BF16)        # past the fp16 numbers
        q[0, 3] = (q[0, 3].float() * 2.0 ** -60).to(BF16)
    for query_block in (1, 4):
        _same(q, scale, zero, 9, levels=15, group_size=32, n_packed=2880, query_block=query_block)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_a_large_channel_that_no_key_has(dtype):
    """The other channels decide, 2^-32 (fp16: 2^-20) of the largest."""
    require_gpu()
    q, scale, zero = _inputs(2, 8, 2, 6, 128, 120, dtype=dtype, seed=15)
    q *= 2.0 ** (-12 if dtype == F16 else -22)
    q[..., 17] = 2.0 ** (8 if dtype == F16 else 10)
    zero[..., :120, 17], scale[..., :120, 17] = 0, 0
    for query_block in (1, 6):
        _same(q, scale, zero, 11, levels=15, group_size=32, n_packed=3840, query_block=query_block)


@pytest.mark.parametrize("bits,group", [(2, 32), (4, 64), (8, 32)])
def test_scores_bound_the_products(bits, group):
    """What a store's own scales say of its keys, as far as a slot's rounding to fp16 goes; and a block that holds a key along the query
    is chosen."""
    require_gpu()
    s, k, _ = store(2, 2, 1024, 0, 128, bits=bits, group=group, seed=13)
    q = torch.randn((2, 4, 1, 128), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").half()
    bound = group_bounds(q, s["k_scale"], s["k_zero"], 2 ** bits - 1)[..., None]
    product = (q.double() @ k.repeat_interleave(2, 1).transpose(2, 3)).view(2, 4, 1, -1, group)
    slack = 2.0 ** -11 * (q.double().abs().sum(-1) * k.abs().amax())[..., None, None]
    assert bool((product <= bound + slack).all())
    _same(q, s["k_scale"], s["k_zero"], 5, levels=2 ** bits - 1, group_size=group, n_packed=1024)


def test_output_stream_graph_and_repeats():
    require_gpu()
    q, scale, zero = _inputs(4, 8, 2, 5, 128, 200, seed=14)
    kw = dict(levels=15, group_size=32, n_packed=6400, n_tail=9, query_block=5, recent=1, causal=True)
    lens = torch.full((4,), 6409, device="cuda")
    want = {n: choose(q, scale, zero, 12, seq_lens=torch.full((4,), n, device="cuda"), **kw) for n in (6409, 700, 0)}
    out = torch.full((4, 2, 1, 12), 99, dtype=torch.int32, device="cuda")
    assert K.select_blocks(q, scale, zero, 12, out=out, **kw) is out and torch.equal(out, want[6409])
    # strided queries
    wide = torch.zeros((4, 5, 8, 256), dtype=F16, device="cuda")
    wide[..., :128] = q.transpose(1, 2)
    assert torch.equal(K.select_blocks(wide[..., :128].transpose(1, 2), scale, zero, 12, **kw), out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = K.select_blocks(q, scale, zero, 12, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, out)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = K.select_blocks(q, scale, zero, 12, seq_lens=lens, **kw)
    with torch.cuda.graph(second):
        again = K.select_blocks(q, scale, zero, 12, seq_lens=lens, **kw)
    for n in (6409, 700, 0, 6409):
        lens.fill_(n)
        graph.replay()
        second.replay()
        K.select_blocks(q, zero, scale, 12, **kw)      # eager work of other values between the replays
        torch.cuda.synchronize()
        assert torch.equal(got, want[n]) and torch.equal(again, want[n])


def test_empty_batch():
    require_gpu()
    q = torch.zeros((0, 4, 1, 64), dtype=F16, device="cuda")
    z = torch.zeros((0, 2, 3, 64), dtype=F16, device="cuda")
    assert K.select_blocks(q, z, z, 2, levels=3, group_size=32, n_packed=96).shape == (0, 2, 1, 2)


@pytest.mark.parametrize("D", [128, 80, 33])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Sq,query_block", [(1, 1), (6, 6)])
def test_equal_scores_beside_values_that_are_not_finite(Sq, query_block, dtype, D):
    """All blocks alike in float32 but a few that are not finite: those first, then the lowest, wherever the former lie."""
    require_gpu()
    q, scale, zero = _inputs(3, 8, 4, Sq, D, 100, seed=16, dtype=dtype, meta=F32, spare=0)
    scale[:], zero[:] = scale[:, :, :1].clone(), zero[:, :, :1].clone()
    zero[0, :, 50, 3] = float("nan")
    scale[1, :, 70, 9] = float("nan")
    zero[2, :, [20, 99], 0] = float("nan")
    got = _same(q, scale, zero, 6, levels=15, group_size=32, n_packed=3200, query_block=query_block)
    for b, odd in enumerate(([50], [70], [20, 99])):
        want = torch.tensor(list(range(6 - len(odd))) + odd, dtype=torch.int32, device="cuda")
        assert torch.equal(got[b], want.expand(4, 1, 6))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("groups", [60, 300])
def test_more_tiles_than_compute_units(groups, D, dtype):
    """280 tiles of up to 32 rows: one launch, of four waves a tile."""
    require_gpu()
    q, scale, zero = _inputs(2, 8, 2, 70, D, groups, dtype=dtype, seed=17 + D)
    for causal in (True, False):
        _same(q, scale, zero, 7, levels=15, group_size=32, n_packed=groups * 32, n_tail=30, first=1, recent=1, causal=causal)
    lens = torch.tensor([groups * 32 - 50, 40], device="cuda")
    _same(q, scale, zero, 7, levels=15, group_size=32, n_packed=groups * 32 - 3, n_tail=30, block_size=64, recent=2, causal=True, seq_lens=lens)


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 128), (BF16, 64), (F16, 256)])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,query_block,groups", [(4, 32, 8, 64, 16, 300), (2, 16, 2, 144, 16, 1000), (2, 24, 2, 9, 3, 33)])
def test_runs_of_many_units(B, Hq, Hkv, Sq, query_block, groups, dtype, D):
    """Two row tiles a tile or more, and (but in the last case) waves that walk two or three units of 32 groups each."""
    require_gpu()
    items, row_tiles, units = B * Hkv * -(-Sq // query_block), -(-Hq // Hkv * query_block // 32), -(-groups // 32)
    assert row_tiles >= 2 and (groups == 33 or items * row_tiles * units > 2048)
    q, scale, zero = _inputs(B, Hq, Hkv, Sq, D, groups, dtype=dtype, seed=18, signed=D == 64)
    _same(q, scale, zero, 6, levels=15, group_size=32, n_packed=groups * 32 - 7, n_tail=40, query_block=query_block, first=1, recent=1, causal=True)


@pytest.mark.parametrize("dtype,meta,D", [(F16, F16, 64), (F32, F32, 33), (BF16, F32, 128)])
@pytest.mark.parametrize("Sq,query_block", [(1, 1), (3, 2)])
def test_more_blocks_than_lds_holds(Sq, query_block, dtype, meta, D):
    """More than 16384 blocks: a choice by scores in memory."""
    require_gpu()
    groups = 16500
    q, scale, zero = _inputs(3, 4, 2, Sq, D, groups, dtype=dtype, meta=meta, seed=19)
    zero[0, 1, 16400, 3] = float("nan")
    zero[0, 0, 9000:9100], scale[0, 0, 9000:9100] = zero[0, 0, 77].clone(), scale[0, 0, 77].clone()       # a hundred alike
    scale[2, :, :groups], zero[2, :, :groups] = scale[2, :, :1].clone(), zero[2, :, :1].clone()     # all alike
    kw = dict(levels=15, group_size=8, n_packed=groups * 8, n_tail=5, query_block=query_block, causal=True)
    got = _same(q, scale, zero, 40, **kw)
    assert 16400 in got[0, 1, 0].tolist()
    assert torch.equal(got[2, 0, 0], torch.arange(40, dtype=torch.int32, device="cuda"))
    lens = torch.tensor([16390 * 8 + 3, 16 * 8, 200], device="cuda")
    _same(q, scale, zero, 40, first=2, recent=3, seq_lens=lens, **kw)
    # two groups a block: as many blocks need twice the groups, so fewer blocks than that, told apart in LDS again
    _same(q, scale, zero, 9, **dict(kw, block_size=16))
