"""``block_sparse_attend`` against attention over the listed slots in 64 bits, and steps of choosing and attending through a cache."""

import math

import pytest
import torch

from tests._blocks import attend, choose, times_seen
from tests._gpu import gpu, require_gpu
from tests._spans import close, store
from veloxquant_mlx_amd import kernels as K
from veloxquant_mlx_amd.cache import KVCacheConfig, KVCacheFactory, LayerStackedKIVICache
from veloxquant_mlx_amd.rotary import RotaryPositions

pytestmark = gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _lists(B, H, tiles, n, total, seed, ascending=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.rand((B, H, tiles, max(total, n)), generator=g, device="cuda").argsort(-1)[..., :n]
    order = torch.where(order < total, order, torch.full_like(order, -1))
    return (order.sort(-1).values if ascending else order).to(torch.int32).contiguous()


def _case(B, Hq, Hkv, D, own, block, n, Sq=1, query_block=1, *, bits=4, group=32, v_layout="token", dtype=F16, meta=F16, causal=True, lens=None,
          spare=40, view=False, seed=0, blocks=None, scale=None, tail_dtype=None):
    s, k, v = store(B, Hkv, *own, D, bits=bits, group=group, v_layout=v_layout, dtype=tail_dtype or dtype, meta=meta, spare=spare, view=view, seed=seed + 1)
    q = torch.randn((B, Hq, Sq, D), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)
    scale = 1 / math.sqrt(D) if scale is None else scale
    lens = None if lens is None else torch.tensor(lens, device="cuda")
    if blocks is None:
        blocks = _lists(B, Hkv, -(-Sq // query_block), n, -(-own[0] // block), seed + 2)
    got = K.block_sparse_attend(q, blocks, **s, block_size=block, query_block=query_block, scale=scale, causal=causal, seq_lens=lens)
    times = times_seen(blocks, block, query_block, B, Sq, own[0], own[1], lens, causal)
    # weights are rounded to fp16 where the matrix units take packed slots, to the rows' type without; float32 rows: not at all
    u = 0.0 if dtype == F32 else torch.finfo(F16 if own[0] else dtype).eps / 2
    want, far = attend(q, k, v, times, scale, u)
    assert got.shape == q.shape and got.dtype == q.dtype
    close(got, want, far)
    return q, s, blocks, got


@pytest.mark.parametrize("bits,group,block", [(2, 32, 32), (4, 32, 64), (4, 64, 64), (2, 128, 128), (4, 32, 96)])
@pytest.mark.parametrize("B,Hq,Hkv,D,own,n", [
    (1, 1, 1, 128, (256, 0), 1), (3, 8, 2, 128, (1024, 33), 5), (5, 12, 4, 256, (640, 130), 3), (2, 14, 2, 64, (384, 5), 2), (7, 32, 8, 128, (2176, 64), 16),
    (2, 4, 4, 128, (128, 1), 40), (1, 40, 1, 128, (2048, 131), 9), (1, 32, 8, 128, (8192, 140), 60), (2, 6, 2, 64, (4096, 0), 32)])
def test_one_query(B, Hq, Hkv, D, own, n, bits, group, block):
    require_gpu()
    if group > D:
        pytest.skip("value groups are at most a head")
    _case(B, Hq, Hkv, D, own, block, n, bits=bits, group=group)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hq,D,Sq,query_block,own", [
    (8, 128, 5, 5, (1024, 40)), (8, 128, 5, 1, (1024, 40)), (8, 128, 70, 8, (2048, 33)), (4, 256, 33, 16, (1024, 70)), (14, 64, 130, 64, (1024, 0)),
    (2, 128, 200, 3, (1024, 129)), (64, 128, 9, 2, (512, 10)), (8, 128, 64, 100, (512, 1))])
def test_tiles_of_queries(Hq, D, Sq, query_block, own, dtype):
    require_gpu()
    for causal in (True, False):
        _case(2, Hq, 2, D, own, 64, 5, Sq, query_block, dtype=dtype, causal=causal, seed=Sq)


@pytest.mark.parametrize("kw", [
    dict(dtype=F32), dict(meta=F32), dict(bits=8), dict(bits=3, own=(480, 37)), dict(v_layout="channel"), dict(D=80, group=16), dict(bits=1), dict(D=40, group=8, dtype=BF16),
    dict(tail_dtype=F32), dict(tail_dtype=BF16, own=(512, 60)), dict(D=7, group=7, own=(112, 3), block=7, bits=8)])
def test_other_stores(kw):
    require_gpu()
    kw = dict(dict(D=128, own=(512, 37), block=64, group=32), **kw)
    D, own, block, group = (kw.pop(x) for x in ("D", "own", "block", "group"))
    if block % group:
        block = group * 2
    for Sq, query_block in ((1, 1), (5, 2)):
        _case(2, 6, 2, D, own, block, 4, Sq, query_block, group=group, **kw)


@pytest.mark.parametrize("Hq,Hkv,Sq,query_block", [(8, 2, 70, 16), (12, 4, 33, 5), (2, 2, 40, 40), (20, 1, 3, 1)])
@pytest.mark.parametrize("kw", [
    dict(D=128, bits=8), dict(D=256, bits=8, dtype=BF16), dict(D=80, group=16, block=48, dtype=F32), dict(D=17, group=8, block=8, bits=5, own=(480, 37)),
    dict(D=200, v_layout="channel", bits=6, own=(480, 45)), dict(D=1, group=1, block=5, meta=F32, bits=8)])
def test_tiles_over_other_stores(Hq, Hkv, Sq, query_block, kw):
    require_gpu()
    kw = dict(dict(own=(512, 75), block=64, group=32), **kw)
    D, own, block, group = (kw.pop(x) for x in ("D", "own", "block", "group"))
    if kw.get("v_layout", "token") == "token" and own[0] % (32 // kw.get("bits", 4)):
        own = (480, own[1])
    for lens in (None, [0, 90, own[0], 9999]):
        for causal in (True, False):
            _case(4, Hq, Hkv, D, own, block, 7, Sq, query_block, group=group, lens=lens, causal=causal, seed=Sq, **kw)


@pytest.mark.parametrize("D,bits,dtype", [(128, 4, F16), (128, 2, BF16), (256, 4, F16), (64, 2, F16), (96, 4, F16), (128, 4, F32)])
@pytest.mark.parametrize("Sq,query_block", [(1, 1), (9, 4)])
def test_lengths_and_rows_that_see_nothing(D, bits, dtype, Sq, query_block):
    require_gpu()
    lens = [0, 1, 5, 9, 31, 32, 33, 500, 512, 513, 545, 9999]
    q, s, blocks, got = _case(12, 4, 2, D, (512, 33), 64, 4, Sq, query_block, bits=bits, dtype=dtype, lens=lens, seed=3)
    assert bool((got[0] == 0).all())
    # a store without a tail, lists that name nothing
    none = torch.full_like(blocks, -1)
    _, _, _, got = _case(12, 4, 2, D, (512, 0), 64, 4, Sq, query_block, bits=bits, dtype=dtype, seed=3, blocks=none)
    assert bool((got == 0).all())
    empty = none[..., :0].contiguous()
    _, _, _, got = _case(12, 4, 2, D, (512, 0), 64, 0, Sq, query_block, bits=bits, dtype=dtype, seed=3, blocks=empty)
    assert bool((got == 0).all())
    _case(12, 4, 2, D, (512, 20), 64, 0, Sq, query_block, bits=bits, dtype=dtype, seed=3, blocks=empty, lens=lens)


@pytest.mark.parametrize("D,dtype", [(128, F16), (256, BF16), (128, F32)])
def test_any_order_twice_and_nothing(D, dtype):
    require_gpu()
    entries = [5, 0, 5, -1, 7, 2 ** 31 - 1, 3, 8, -2 ** 31, 5]        # out of order, three times, none, past the store
    blocks = torch.tensor(entries, dtype=torch.int32, device="cuda").expand(2, 2, 1, 10).contiguous()
    _, _, _, got = _case(2, 8, 2, D, (512, 9), 64, 10, dtype=dtype, blocks=blocks, seed=4)
    named = torch.tensor([0, 3, 5, 5, 5, 7], dtype=torch.int32, device="cuda").expand(2, 2, 1, 6).contiguous()
    _, _, _, same = _case(2, 8, 2, D, (512, 9), 64, 6, dtype=dtype, blocks=named, seed=4)
    assert float((got.float() - same.float()).abs().max()) <= 2.0 ** -6


@pytest.mark.parametrize("D,bits", [(128, 4), (128, 2), (256, 2), (64, 4)])
def test_store_that_ends_inside_a_block_and_a_unit(D, bits):
    require_gpu()
    # (packed slots end where a group does; the last block holds one group of four)
    _case(3, 8, 2, D, (32 * 9, 3), 128, 3, bits=bits, seed=5)
    _case(3, 8, 2, D, (32 * 9, 3), 128, 3, bits=bits, seed=5, lens=[32 * 9 - 1, 257, 32 * 8 + 13])


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_scales(scale, dtype):
    require_gpu()
    _case(2, 8, 2, 128, (512, 40), 32, 7, dtype=dtype, scale=scale, seed=6)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tail_views_and_all_blocks(dtype):
    require_gpu()
    q, s, _, got = _case(3, 8, 2, 128, (512, 77), 64, 8, dtype=dtype, view=True, seed=7)
    # all blocks: attention over the whole store, to the roundings of either
    whole = K.shared_prefix_attend(q, dict(n_packed=0, n_tail=1, k_tail=torch.zeros((1, 2, 1, 128), dtype=dtype, device="cuda"),
                                           v_tail=torch.zeros((1, 2, 1, 128), dtype=dtype, device="cuda")), **s, scale=128 ** -0.5, causal=True)
    assert whole.shape == got.shape


@pytest.mark.parametrize("D,dtype", [(128, F16), (256, F16), (128, F32)])
def test_blocks_that_are_not_listed_are_not_read(D, dtype):
    require_gpu()
    q, s, blocks, got = _case(2, 8, 2, D, (1024, 40), 64, 4, dtype=dtype, seed=8)
    listed = torch.zeros((2, 2, 16), dtype=torch.bool, device="cuda")
    listed.scatter_(2, blocks[:, :, 0].long(), True)
    broken = dict(s)
    for name in ("k_scale", "k_zero"):
        t = broken[name] = s[name].clone()
        t[:, :, :32].view(2, 2, 16, 2, D)[~listed] = float("nan")
    for name in ("v_scale", "v_zero"):
        t = broken[name] = s[name].clone()
        t[..., :1024].view(2, 2, D // 32, 16, 64).transpose(2, 3)[~listed] = float("nan")
    again = K.block_sparse_attend(q, blocks, **broken, block_size=64, scale=D ** -0.5, causal=True)
    assert torch.equal(got, again)


def test_far_slots():
    """Slots whose words lie past 2^31 bytes into their buffers."""
    require_gpu()
    B, H, D, n, block = 1, 3, 128, 1 << 24, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (B, H, n, D // 8), generator=g, device="cuda", dtype=torch.int32)
    values = torch.randint(-2 ** 31, 2 ** 31 - 1, (B, H, n // 8, D), generator=g, device="cuda", dtype=torch.int32)
    ks, kz = (torch.rand((B, H, n // 32, D), generator=g, device="cuda").half() * 0.1 for _ in range(2))
    vs, vz = (torch.rand((B, H, D // 32, n), generator=g, device="cuda").half() * 0.1 for _ in range(2))
    s = dict(k_packed=words, k_scale=ks, k_zero=kz, v_packed=values, v_scale=vs, v_zero=vz, bits=4, group_size=32, v_layout="token")
    q = torch.randn((B, 12, 1, D), generator=g, device="cuda").half()
    blocks = torch.tensor([0, 1, 4095, n // block - 2, n // block - 1], dtype=torch.int32, device="cuda").expand(B, H, 1, 5).contiguous()
    got = K.block_sparse_attend(q, blocks, **s, n_packed=n, block_size=block, scale=0.1)
    at = torch.cat([torch.arange(int(e) * block, (int(e) + 1) * block, device="cuda") for e in blocks[0, 0, 0]])
    few = dict(s, k_packed=words[:, :, at].contiguous(), v_packed=values.view(B, H, -1, block // 8, D)[:, :, blocks[0, 0, 0].long()].flatten(2, 3).contiguous(),
               k_scale=ks.view(B, H, -1, 4, D)[:, :, blocks[0, 0, 0].long()].flatten(2, 3).contiguous(),
               k_zero=kz.view(B, H, -1, 4, D)[:, :, blocks[0, 0, 0].long()].flatten(2, 3).contiguous(),
               v_scale=vs[..., at].contiguous(), v_zero=vz[..., at].contiguous())
    near = torch.arange(5, dtype=torch.int32, device="cuda").expand(B, H, 1, 5).contiguous()
    assert torch.equal(got, K.block_sparse_attend(q, near, **few, n_packed=5 * block, block_size=block, scale=0.1))


def test_lists_longer_than_a_block_walks():
    """2200 entries of 32 tokens for each of 512 kv heads: more units than one block of threads holds."""
    require_gpu()
    entries = (torch.arange(2200, dtype=torch.int32, device="cuda") % 5 - 1)     # each of four blocks 440 times, and none
    blocks = entries.expand(128, 4, 1, 2200).contiguous()
    _case(128, 4, 4, 64, (128, 3), 32, 2200, bits=2, blocks=blocks, seed=10)


@pytest.mark.parametrize("Sq,query_block", [(1, 1), (40, 4)])
def test_a_layer_of_a_stack(Sq, query_block):
    require_gpu()
    cfg = KVCacheConfig(method="kivi", head_dim=128, bit_width_inlier=4, kivi_group_size=32, residual_length=32, fused_sdpa=True, fused_sdpa_memory_bound=True)
    stack, alone = LayerStackedKIVICache(cfg, 2), [KVCacheFactory.create(cfg) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(4)
    for S in (300, 1, Sq):
        k, v = (torch.randn((2, 2, 4, S, 128), generator=g, device="cuda").half() for _ in range(2))
        for layer in range(2):
            stack[layer].update_and_fetch(k[layer], v[layer])
            alone[layer].update_and_fetch(k[layer], v[layer])
        stack.fused_sdpa_all(torch.randn((2, 2, 8, 1, 128), generator=g, device="cuda").half(), 0.1)      # (stacks the layers' buffers)
    q = torch.randn((2, 8, Sq, 128), generator=g, device="cuda").half()
    for layer in range(2):
        args = (q, 0.1, 4)
        assert torch.equal(stack[layer].fused_sparse_sdpa(*args, query_block=query_block), alone[layer].fused_sparse_sdpa(*args, query_block=query_block))


def test_output_stream_graph_and_repeats():
    require_gpu()
    q, s, blocks, got = _case(4, 8, 2, 128, (2048, 50), 64, 12, seed=9)
    kw = dict(block_size=64, scale=128 ** -0.5, causal=True)
    out = torch.empty_like(q)
    assert K.block_sparse_attend(q, blocks, **s, **kw, out=out) is out and torch.equal(out, got)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = K.block_sparse_attend(q, blocks, **s, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, got)
    lists = blocks.clone()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = K.block_sparse_attend(q, lists, **s, **kw)
    with torch.cuda.graph(second):
        b = K.block_sparse_attend(q, lists, **s, **kw)
    for seed in (1, 2, 3):
        lists.copy_(_lists(4, 2, 1, 12, 32, seed))
        want = K.block_sparse_attend(q, lists, **s, **kw)
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)
    same = q.clone()
    assert torch.equal(K.block_sparse_attend(same, blocks, **s, **kw, out=same), got)


@pytest.mark.parametrize("memory_bound", [True, False])
@pytest.mark.parametrize("D,bits", [(128, 4), (256, 2), (64, 4), (128, 3)])
def test_steps_through_a_cache(D, bits, memory_bound):
    """A prompt in chunks and then steps: normed, turned, stored, chosen, attended; each against 64 bits over the cache's own slots."""
    require_gpu()
    B, Hq, H, R, g = 2, 8, 2, 64, 32
    cache = KVCacheFactory.create(KVCacheConfig(method="kivi", head_dim=D, bit_width_inlier=bits, kivi_group_size=g, residual_length=R, fused_sdpa=True,
                                                fused_sdpa_memory_bound=memory_bound, kivi_pair_heads=False))
    rope = RotaryPositions(D)
    gen = torch.Generator(device="cuda").manual_seed(D + bits)
    qw, kw = (torch.rand(D, generator=gen, device="cuda").half() + 0.5 for _ in range(2))
    scale = D ** -0.5
    for S, query_block in ((5, 2), (300, 8), (97, 16), (1, 1), (1, 1), (40, 4), (1, 1)):
        rows = torch.randn((B, S, (Hq + 2 * H) * D), generator=gen, device="cuda").half().view(B, S, Hq + 2 * H, D).transpose(1, 2)
        q, k = rope.normed(rows[:, :Hq], rows[:, Hq:Hq + H], q_weight=qw, k_weight=kw, offset=cache.offset)
        cache.update_and_fetch(k, rows[:, Hq + H:])
        blocks = cache.select_blocks(q, 4, block_size=32, query_block=query_block)
        got = cache.fused_sparse_sdpa(q, scale, blocks=blocks, block_size=32, query_block=query_block)
        assert torch.equal(got, cache.fused_sparse_sdpa(q, scale, 4, block_size=32, query_block=query_block))
        s = cache._store_args()
        n, n_tail = s["n_packed"], s["n_tail"]
        assert n + n_tail == cache.offset
        want_blocks = choose(q, s["k_scale"], s["k_zero"], 4, levels=2 ** bits - 1, group_size=g, n_packed=n, n_tail=n_tail, query_block=query_block,
                             first=1, recent=1, causal=True) if n else torch.full_like(blocks, -1)
        assert torch.equal(blocks, want_blocks)
        ks, vs = [torch.zeros((B, H, 0, D), dtype=torch.float64, device="cuda")], [torch.zeros((B, H, 0, D), dtype=torch.float64, device="cuda")]
        if n:
            from tests._spans import _rows
            ks.append(_rows(s["k_packed"][:, :, :n].transpose(2, 3), s["k_scale"], s["k_zero"], s["bits"], D, n, g, "k"))
            vs.append(_rows(s["v_packed"], s["v_scale"], s["v_zero"], s["bits"], D, n, g, s["v_layout"]))
        if n_tail:
            ks.append(s["k_tail"][:, :, :n_tail].double())
            vs.append(s["v_tail"][:, :, :n_tail].double())
        times = times_seen(blocks, 32, query_block, B, S, n, n_tail, None, True)
        want, far = attend(q, torch.cat(ks, 2), torch.cat(vs, 2), times, scale, 2.0 ** -11)
        close(got, want, far)
    # with enough blocks: attention over the whole cache
    q = torch.randn((B, Hq, 1, D), generator=gen, device="cuda").half()
    whole, sparse = cache.fused_sdpa(q, scale), cache.fused_sparse_sdpa(q, scale, 64)
    assert float((whole.float() - sparse.float()).abs().max()) <= 4e-3
    lens = torch.tensor([cache.offset, 100], device="cuda")
    part = cache.fused_sparse_sdpa(q, scale, 64, lengths=[cache.offset, 100])
    assert torch.equal(part[0], sparse[0])
    assert float((cache.fused_sdpa(q, scale, lengths=lens)[1].float() - part[1].float()).abs().max()) <= 4e-3


def test_an_empty_list_needs_no_store():
    require_gpu()
    _case(2, 8, 2, 128, (0, 50), 32, 3, blocks=torch.full((2, 2, 1, 3), 1, dtype=torch.int32, device="cuda"))
    q = torch.zeros((0, 4, 1, 64), dtype=F16, device="cuda")
    t = torch.zeros((0, 2, 3, 64), dtype=F16, device="cuda")
    assert K.block_sparse_attend(q, torch.zeros((0, 2, 1, 2), dtype=torch.int32, device="cuda"), block_size=32, k_tail=t, v_tail=t, n_tail=3).shape == q.shape


@pytest.mark.parametrize("D,bits,dtype", [(128, 2, F16), (64, 4, BF16), (128, 8, F16)])
def test_calls_under_way_on_two_streams(D, bits, dtype):
    """Choice and attention in parts on two streams at once: each stream has its own scratch and counters."""
    require_gpu()
    sets = []
    for seed in (20, 30):
        q, s, blocks, _ = _case(1, 8, 2, D, (4096, 60), 32, 60, bits=bits, dtype=dtype, seed=seed)
        sets.append((q, s, torch.cuda.Stream()))

    def step(q, s):
        chosen = K.select_blocks(q, s["k_scale"], s["k_zero"], 60, levels=2 ** bits - 1, group_size=32, n_packed=4096, n_tail=60, causal=True)
        return chosen, K.block_sparse_attend(q, chosen, **s, block_size=32, scale=0.1, causal=True)

    want = [step(q, s) for q, s, _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for q, s, stream in sets:
            with torch.cuda.stream(stream):
                got.append(step(q, s))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(got, want):
            assert torch.equal(a, c) and torch.equal(b, d)


@pytest.mark.parametrize("bits,dtype", [(4, F16), (2, BF16)])
@pytest.mark.parametrize("Hq,D,total,n", [(1, 64, 700, 650), (2, 64, 1100, 1000), (1, 128, 1100, 1000)])
def test_more_parts_than_a_round_of_the_sum(Hq, D, total, n, bits, dtype):
    """One list over 650 units or more, in more than 32 parts, which the block that ends last adds up in rounds of 32."""
    require_gpu()
    parts = -(-(n + 1) // 16)       # (a list's units and the tail's one, in runs of 16)
    assert parts > 32 and Hq * parts * D * 4 <= 32 * 1024
    q, s, blocks, got = _case(1, Hq, 1, D, (total * 32, 5), 32, n, bits=bits, dtype=dtype, seed=21)
    kw = dict(block_size=32, scale=D ** -0.5, causal=True)
    graph = torch.cuda.CUDAGraph()      # (parts added up by a launch of their own)
    with torch.cuda.graph(graph):
        other = K.block_sparse_attend(q, blocks, **s, **kw)
    for _ in range(3):
        other.zero_()
        graph.replay()
        assert float((other.float() - got.float()).abs().max()) <= 2 * torch.finfo(dtype).eps * float(got.float().abs().max())
    # the last parts, and all but the first, hold nothing that is seen
    for live in (total * 16, 40, 3):
        _case(1, Hq, 1, D, (total * 32, 5), 32, n, bits=bits, dtype=dtype, seed=21, lens=[live])


@pytest.mark.parametrize("D,bits,dtype", [(128, 4, F16), (128, 2, BF16), (256, 4, F16), (64, 4, F16), (128, 8, F16), (128, 4, F32)])
@pytest.mark.parametrize("Sq,query_block", [(1, 1), (20, 6)])
def test_all_blocks_are_the_whole_store(Sq, query_block, D, bits, dtype):
    """Lists of all blocks: attention over the whole store, each as far from 64 bits as its roundings go."""
    require_gpu()
    every = torch.arange(8, dtype=torch.int32, device="cuda").expand(3, 2, -(-Sq // query_block), 8).contiguous()
    q, s, _, got = _case(3, 8, 2, D, (512, 77), 64, 8, Sq, query_block, bits=bits, dtype=dtype, view=True, seed=22, blocks=every)
    whole = K.shared_prefix_attend(q, None, **s, scale=D ** -0.5, causal=True)
    _, k, v = store(3, 2, 512, 77, D, bits=bits, dtype=dtype, spare=40, view=True, seed=23)      # (the case's)
    times = times_seen(every, 64, query_block, 3, Sq, 512, 77, None, True)
    want, far = attend(q, k, v, times, D ** -0.5, 0.0 if dtype == F32 else 2.0 ** -11)
    close(whole, want, far)
    assert bool(((got.double() - whole.double()).abs() <= 2 * (far * (1 + 2.0 ** -8) + torch.finfo(dtype).eps / 2 * want.abs() + 1e-6)).all())


@pytest.mark.parametrize("S", [20, 200])
@pytest.mark.parametrize("memory_bound", [True, False])
def test_a_cache_refuses_the_same_with_and_without_packed_tokens(S, memory_bound):
    require_gpu()
    cache = KVCacheFactory.create(KVCacheConfig(method="kivi", head_dim=128, bit_width_inlier=4, kivi_group_size=32, residual_length=64, fused_sdpa=True,
                                                fused_sdpa_memory_bound=memory_bound))
    g = torch.Generator(device="cuda").manual_seed(24)
    k, q = (torch.randn((2, h, S, 128), generator=g, device="cuda").half() for h in (2, 4))
    cache.update_and_fetch(k, k)
    assert (cache._n_quantized > 0) == (S == 200)
    q = q[:, :, :5].contiguous()
    for bad in (dict(query_block=0), dict(n_select=0), dict(n_select=-1), dict(block_size=48), dict(first=-1), dict(first=3, recent=2), dict(recent=-2)):
        kw = dict(dict(n_select=4, query_block=2), **bad)
        with pytest.raises(ValueError, match="select_blocks: "):
            cache.select_blocks(q, **kw)
        with pytest.raises(ValueError, match="select_blocks: |fused_sparse_sdpa: "):
            cache.fused_sparse_sdpa(q, 0.1, **kw)
    for rows in (q[:1], q[:, :3], q[..., :64].contiguous()):     # another batch, heads over no kv head, other channels
        with pytest.raises(ValueError, match="select_blocks: "):
            cache.select_blocks(rows, 4)
    got = cache.select_blocks(q, 4, query_block=2)
    assert got.shape == (2, 2, 3, 4) and got.dtype == torch.int32 and (S == 200 or bool((got == -1).all()))
    assert torch.equal(cache.select_blocks(q, 4, query_block=2, lengths=[S, S]), got)


def test_more_tiles_of_rows_than_a_grid_holds():
    """65600 queries that choose singly: taken in float32."""
    require_gpu()
    q, s, blocks, got = _case(1, 1, 1, 64, (128, 3), 32, 2, 65600, bits=4, causal=False, seed=25)
    few = K.block_sparse_attend(q[:, :, :100].contiguous(), blocks[:, :, :100].contiguous(), **s, block_size=32, scale=64 ** -0.5)
    assert float((few.double() - got[:, :, :100].double()).abs().max()) <= 2.0 ** -9 * float(got.abs().max())
