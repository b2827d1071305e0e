"""Operators of a decode step that reads only a part of a long compressed context: queries and keys normed a head and turned to their
positions, the choice of the blocks of packed keys that a query attends to, and attention over those blocks and the plain tail.

``run`` computes each in its plain form, elementary torch operations in 32 bits (angles and the scores that blocks are chosen by in
64), or, where ``own`` is true, through this package's functions.

A packed store is laid out as the caches keep it: keys ``int32 [B, H, room, D / per]``, a word holding ``per = 32 / bits`` consecutive
channels of a token (lowest bits first), scale and zero ``[B, H, room / group, D]``; values ``int32 [B, H, room / per, D]``, a word
holding ``per`` consecutive tokens of a channel, scale and zero ``[B, H, D / group, room]``.  A packed slot stands for the fp16 number
``code * scale + zero``, so a group's keys lie in a channel between ``zero`` and ``zero + levels * scale``, ``levels`` the top code.  The
newest tokens follow as plain rows (the tail).  Query ``i`` of ``Sq`` stands at slot ``n - Sq + i`` of its sequence's ``n`` live ones.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
HEADS = {64: [(32, 8), (14, 2), (9, 3)], 128: [(32, 8), (28, 4), (40, 10)], 256: [(12, 4), (8, 4)]}
NORM_EPS = 1e-6
SPARE = 64   # slots of a store behind the packed ones


def listed():
    return [
        # one decode step of one sequence: queries and keys of one token, launch latency and nothing else
        dict(name="norm_rope_step", kind="norm_rope", hq=32, hkv=8, d=128, dims=128, batch=1, seq=1, traditional=False, scaling="none",
             far=9000, ragged=False, head_weights=False, dtype="bfloat16"),
        # a prompt of 8k tokens, half layout, frequencies scaled by parts for a long context
        dict(name="norm_rope_prompt", kind="norm_rope", hq=32, hkv=8, d=128, dims=128, batch=1, seq=8192, traditional=False,
             scaling="by_parts", far=0, ragged=False, head_weights=False, dtype="bfloat16"),
        # chunks of an odd length of a batch, each at its own far position, interleaved pairs over a quarter of the head, a weight row a head
        dict(name="norm_rope_part_ragged", kind="norm_rope", hq=12, hkv=4, d=256, dims=64, batch=7, seq=1003, traditional=True,
             scaling="linear", far=900000, ragged=True, head_weights=True, dtype="float16"),
        # float32 rows, small heads
        dict(name="norm_rope_float32", kind="norm_rope", hq=9, hkv=3, d=64, dims=64, batch=2, seq=2047, traditional=False, scaling="none",
             far=100000, ragged=False, head_weights=False, dtype="float32"),
        # one user's step over 8k tokens in groups of 32: latency
        dict(name="select_step", kind="select", hq=32, hkv=8, d=128, batch=1, packed=8192, tail=131, sq=1, query_block=1, levels=3, group=32,
             block=32, count=64, first=1, recent=2, ragged=False, dtype="float16", meta="float16"),
        # a serving batch at 32k, of different lengths: the bytes of the scales count
        dict(name="select_32k_batch", kind="select", hq=32, hkv=8, d=128, batch=16, packed=32768, tail=132, sq=1, query_block=1, levels=15,
             group=32, block=64, count=48, first=1, recent=2, ragged=True, dtype="float16", meta="float16"),
        # a prompt's chunk of 512 tokens behind 16k, eight queries choose together
        dict(name="select_chunk", kind="select", hq=32, hkv=8, d=128, batch=1, packed=16768, tail=140, sq=512, query_block=8, levels=15,
             group=32, block=64, count=32, first=1, recent=3, ragged=False, dtype="bfloat16", meta="float16"),
        # three proposed tokens a sequence, heads of 256 channels, float32 scales, an odd batch
        dict(name="select_verify_d256", kind="select", hq=12, hkv=4, d=256, batch=5, packed=19968, tail=77, sq=3, query_block=1, levels=15,
             group=64, block=128, count=21, first=0, recent=1, ragged=True, dtype="bfloat16", meta="float32"),
        # one user's step, 64 of 256 blocks, 2 bits: latency
        dict(name="attend_step", kind="attend", hq=32, hkv=8, d=128, batch=1, packed=8192, tail=131, sq=1, query_block=1, bits=2, group=32,
             block=32, count=64, first=1, recent=2, ragged=False, dtype="float16"),
        # a serving batch at 32k, 3k slots a step and kv head, of different lengths
        dict(name="attend_32k_batch", kind="attend", hq=32, hkv=8, d=128, batch=16, packed=32768, tail=132, sq=1, query_block=1, bits=4,
             group=32, block=64, count=48, first=1, recent=2, ragged=True, dtype="float16"),
        # a prompt's chunk of 512 tokens, every eight queries with blocks of their own: the largest
        dict(name="attend_chunk", kind="attend", hq=32, hkv=8, d=128, batch=1, packed=16768, tail=140, sq=512, query_block=8, bits=4, group=32,
             block=64, count=32, first=1, recent=3, ragged=False, dtype="bfloat16"),
        # three proposed tokens a sequence that choose together, heads of 256 channels, an odd batch
        dict(name="attend_verify_d256", kind="attend", hq=12, hkv=4, d=256, batch=5, packed=19968, tail=77, sq=3, query_block=3, bits=4,
             group=64, block=128, count=21, first=0, recent=1, ragged=True, dtype="float16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_rope", "select", "attend"])
    d = rng.choice([64, 128, 128, 256])
    hq, hkv = rng.choice(HEADS[d])
    if kind == "norm_rope":
        batch = _log_int(rng, 1, 16)
        return dict(kind=kind, hq=hq, hkv=hkv, d=d, dims=rng.choice([d, d, d // 2, d // 4]), batch=batch,
                    seq=max(1, min(_log_int(rng, 1, 8192), 8192 * 40 * 128 // (batch * (hq + hkv) * d))), traditional=rng.random() < 0.4,
                    scaling=rng.choice(["none", "linear", "by_parts"]), far=rng.choice([0, 5000, 131000, 1000000]), ragged=rng.random() < 0.4,
                    head_weights=rng.random() < 0.2, dtype=rng.choice(["float16", "bfloat16", "bfloat16", "float32"]))
    group = rng.choice([32, 32, 64])
    block = rng.choice([group, 64, 64, 128])
    count = _log_int(rng, 4, 96) if block < 128 else _log_int(rng, 4, 32)
    first, recent = rng.choice([0, 1, 1, 2]), rng.choice([0, 1, 2])
    batch, n = _log_int(rng, 1, 16), _log_int(rng, 300, 33000)
    what = rng.choice(["step", "step", "step", "verify", "chunk"])
    sq = query_block = 1
    if what == "verify":
        sq = rng.randint(2, 8)
        query_block = rng.choice([1, sq])
    elif what == "chunk":
        batch, sq, query_block = rng.choice([1, 1, 2]), _log_int(rng, 30, 512), rng.choice([4, 8, 16])
    tiles = -(-sq // query_block)
    n = max(300, min(n, 16 * 32768 * 8 * 128 // (batch * hkv * d)))
    most = 2 ** 27 // (batch * hkv * tiles * block * d)   # slots that the plain form lays out
    case = dict(kind=kind, hq=hq, hkv=hkv, d=d, batch=batch, packed=(n - 140) // group * group, tail=rng.randint(1, 160), sq=sq,
                query_block=query_block, levels=rng.choice([3, 15, 15]), group=group, block=block, count=max(4, min(count, most)), first=first,
                recent=recent, ragged=batch > 1 and rng.random() < 0.4, dtype=rng.choice(["float16", "float16", "bfloat16"]))
    if kind == "select":
        case["meta"] = rng.choice(["float16", "float16", "float16", "float32"])
        case["batch"] = max(1, min(batch, 2 ** 26 // (hq * sq * max(1, case["packed"] // group))))
    else:
        case["bits"] = 2 if case.pop("levels") == 3 else 4
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """Live slots of every sequence: from a third to the whole of the room."""
    n = case["packed"] + case["tail"]
    if not case["ragged"]:
        return [n] * case["batch"]
    return [n - (b * 7919) % (2 * n // 3 + 1) for b in range(case["batch"])]


def _frequencies(dims, scaling):
    """Angular frequencies, float64: 10000^(-2i/dims); 'linear' positions divided by 8, 'by_parts' long wavelengths divided
    by 8, short ones kept and those between blended."""
    f = 10000.0 ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if scaling == "linear":
        return f / 8
    if scaling == "by_parts":
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / (4 - 1)).clamp(0, 1)
        return f * (keep + (1 - keep) / 8)
    return f


def _keys(gen, hkv, n, d, factors):
    """One sequence's keys [H, n, D]: channels of unlike spread, around a centre that moves every 64 tokens as a text's topic does."""
    centre = torch.randn((hkv, -(-n // 64), d), generator=gen, device="cuda") * 0.7
    return (torch.randn((hkv, n, d), generator=gen, device="cuda") + centre.repeat_interleave(64, 1)[:, :n]) * factors


def _pack(codes, bits):
    """Codes along the last axis to int32 words, lowest bits first."""
    per = 32 // bits
    codes = codes.view(*codes.shape[:-1], -1, per)
    words = codes[..., 0].to(torch.int32)
    for j in range(1, per):
        words |= codes[..., j].to(torch.int32) << (bits * j)
    return words


def _quantise(x, group, levels, meta):
    """Groups along the last axis: codes, and scale and zero."""
    g = x.view(*x.shape[:-1], -1, group)
    lo, hi = g.amin(-1), g.amax(-1)
    scale, zero = ((hi - lo) / levels).clamp_min(1e-4).to(meta), lo.to(meta)
    codes = ((g - zero.float()[..., None]) / scale.float()[..., None]).round_().clamp_(0, levels).to(torch.uint8)
    return codes.view(x.shape), scale, zero


def _store(gen, case, factors):
    """Keys and values of `packed` quantised tokens, with room behind them, and `tail` plain ones."""
    B, hkv, d, packed, tail, bits, g = (case[x] for x in ("batch", "hkv", "d", "packed", "tail", "bits", "group"))
    levels, per, room = 2 ** bits - 1, 32 // bits, packed + SPARE
    s = dict(n_packed=packed, n_tail=tail, bits=bits, group_size=g, v_layout="token")
    s["k_packed"] = torch.zeros((B, hkv, room, d // per), dtype=torch.int32, device="cuda")
    s["v_packed"] = torch.zeros((B, hkv, room // per, d), dtype=torch.int32, device="cuda")
    s["k_scale"], s["k_zero"] = (torch.zeros((B, hkv, room // g, d), dtype=torch.float16, device="cuda") for _ in range(2))
    s["v_scale"], s["v_zero"] = (torch.zeros((B, hkv, d // g, room), dtype=torch.float16, device="cuda") for _ in range(2))
    for b in range(B):
        k = _keys(gen, hkv, packed, d, factors)
        codes, scale, zero = _quantise(k.transpose(1, 2).contiguous(), g, levels, torch.float16)       # [H, D, n]: groups of tokens
        s["k_packed"][b, :, :packed] = _pack(codes.transpose(1, 2).contiguous(), bits)
        s["k_scale"][b, :, : packed // g], s["k_zero"][b, :, : packed // g] = scale.transpose(1, 2), zero.transpose(1, 2)
        codes, scale, zero = _quantise(torch.randn((hkv, packed, d), generator=gen, device="cuda"), g, levels, torch.float16)
        s["v_packed"][b, :, : packed // per] = _pack(codes.transpose(1, 2).contiguous(), bits).transpose(1, 2)
        s["v_scale"][b, :, :, :packed], s["v_zero"][b, :, :, :packed] = scale.transpose(1, 2), zero.transpose(1, 2)
    dtype = DTYPES[case["dtype"]]
    s["k_tail"] = (torch.randn((B, hkv, tail, d), generator=gen, device="cuda") * factors).to(dtype)
    s["v_tail"] = torch.randn((B, hkv, tail, d), generator=gen, device="cuda").to(dtype)
    return s


def _ends(case, lens, device):
    """[B, T, query_block]: one past the last slot that each query of a tile sees (the last tile's missing queries see nothing)."""
    sq, qb, n = case["sq"], case["query_block"], case["packed"] + case["tail"]
    tiles = -(-sq // qb)
    i = torch.arange(tiles * qb, device=device)
    live = torch.full((case["batch"],), n, device=device) if lens is None else lens
    end = (live.view(-1, 1) - sq + i + 1).clamp_min(0)
    return torch.where(i < sq, end, torch.zeros_like(end)).view(-1, tiles, qb)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    B, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
    if case["kind"] == "norm_rope":
        S = case["seq"]
        # queries, keys and values as one projection leaves them: views [B, H, S, D] of its rows
        rows = (torch.randn((B, S, (hq + 2 * hkv) * d), generator=gen, device="cuda") * 2.5).to(dtype)
        q = rows[..., : hq * d].view(B, S, hq, d).transpose(1, 2)
        k = rows[..., hq * d: (hq + hkv) * d].view(B, S, hkv, d).transpose(1, 2)
        first = torch.full((B,), case["far"], device="cuda", dtype=torch.int64)
        if case["ragged"]:
            first -= torch.randint(0, case["far"] // 2 + 1, (B,), generator=gen, device="cuda")
        shape = lambda h: (h, d) if case["head_weights"] else (d,)
        qw, kw = ((torch.rand(shape(h), generator=gen, device="cuda") + 0.5).to(dtype) for h in (hq, hkv))
        return dict(case=case, q=q, k=k, qw=qw, kw=kw, inv_freq=_frequencies(case["dims"], case["scaling"]).cuda(), first=first)
    factors = torch.randn((d,), generator=gen, device="cuda").mul(0.5).exp()
    state = dict(case=case, scale=1 / math.sqrt(d))
    state["q"] = torch.randn((B, hq, case["sq"], d), generator=gen, device="cuda").to(dtype)
    state["lens"] = torch.tensor(_lengths(case), device="cuda") if case["ragged"] else None
    if case["kind"] == "select":
        g, n = case["group"], case["packed"]
        like = dict(dtype=DTYPES[case["meta"]], device="cuda")
        state["k_scale"], state["k_zero"] = (torch.zeros((B, hkv, (n + SPARE) // g, d), **like) for _ in range(2))
        for b in range(B):
            k = _keys(gen, hkv, n, d, factors).view(hkv, n // g, g, d)
            lo, hi = k.amin(2), k.amax(2)
            state["k_scale"][b, :, : n // g], state["k_zero"][b, :, : n // g] = ((hi - lo) / case["levels"]).clamp_min(1e-4), lo
        return state
    state["store"] = _store(gen, case, factors)
    # blocks as a choice leaves them: ascending, the first and the last visible ones among them, -1 where fewer are visible
    end = _ends(case, state["lens"], "cuda").amax(-1).clamp_max(case["packed"])
    total = -(-case["packed"] // case["block"])
    visible = ((end + case["block"] - 1) // case["block"]).view(B, 1, -1, 1)
    j = torch.arange(total, device="cuda")
    rank = torch.rand((B, hkv, end.shape[1], total), generator=gen, device="cuda")
    rank = rank + 2 * (j < case["first"]) + 2 * (j >= visible - case["recent"])
    state["blocks"] = _chosen(rank.masked_fill(j >= visible, float("-inf")), case["count"])
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _chosen(score, count):
    """The `count` highest of the last axis (ties: the lowest index) in ascending order, int32; -1 where less than that is above -inf."""
    total = score.shape[-1]
    top, at = score.sort(dim=-1, descending=True, stable=True)
    at = at.masked_fill(top == float("-inf"), total)[..., :count]
    if total < count:
        at = torch.cat((at, at.new_full((*at.shape[:-1], count - total), total)), -1)
    at = at.sort(-1).values
    return at.masked_fill(at == total, -1).to(torch.int32)


def _plain_norm_rope(x, weight, cos, sin, dims, traditional):
    x = x.float()
    x = x / (x.square().mean(-1, keepdim=True) + NORM_EPS).sqrt() * (weight[:, None, :] if weight.ndim == 2 else weight).float()
    if traditional:
        a, b = x[..., 0:dims:2], x[..., 1:dims:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., : dims // 2], x[..., dims // 2: dims]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., dims:]), dim=-1)


def _tiles_of(q, case):
    """Queries as the rows of their tile, [B, Hkv, T, query_block, G, D] (the last tile filled up with zeros)."""
    B, hq, sq, d = q.shape
    hkv, qb = case["hkv"], case["query_block"]
    tiles = -(-sq // qb)
    if tiles * qb > sq:
        q = torch.cat((q, q.new_zeros((B, hq, tiles * qb - sq, d))), 2)
    return q.view(B, hkv, hq // hkv, tiles, qb, d).permute(0, 1, 3, 4, 2, 5)


def _plain_select(state):
    case, q = state["case"], state["q"]
    B, hkv, d, g, n = case["batch"], case["hkv"], case["d"], case["group"], case["packed"]
    rows = _tiles_of(q, case).double()
    shape = rows.shape
    rows = rows.reshape(B, hkv, -1, d)
    zero = state["k_zero"][:, :, : n // g].double().transpose(2, 3)
    scale = state["k_scale"][:, :, : n // g].double().transpose(2, 3)
    # sum of max(q z, q (z + L s)), q and s split by their signs
    s = torch.matmul(rows.clamp_min(0), scale.clamp_min(0)) + torch.matmul((-rows).clamp_min(0), (-scale).clamp_min(0))
    s = torch.matmul(rows, zero) + case["levels"] * s
    s = s.view(*shape[:-1], n // g).amax(4)                                          # [B, Hkv, T, query_block, groups]: over the heads
    end = _ends(case, state["lens"], q.device).clamp_max(n)[:, None]
    s = s.masked_fill(torch.arange(0, n, g, device=q.device) >= end[..., None], float("-inf")).amax(3)
    per = case["block"] // g
    total = -(-n // case["block"])
    if total * per > n // g:
        s = torch.cat((s, s.new_full((*s.shape[:-1], total * per - n // g), float("-inf"))), -1)
    s = s.view(*s.shape[:-1], total, per).amax(-1)
    j = torch.arange(total, device=q.device)
    visible = ((end.amax(-1, keepdim=True) + case["block"] - 1) // case["block"])
    kept = ((j < case["first"]) | (j >= visible - case["recent"])) & (j < visible)
    return _chosen(s.masked_fill(kept, float("inf")), case["count"])


def _gathered(s, slot):
    """Keys and values of packed slots [B, H, T, S] in 32 bits, [B, H, T, S, D]."""
    B, H = slot.shape[:2]
    b, h = torch.arange(B, device=slot.device).view(B, 1, 1, 1), torch.arange(H, device=slot.device).view(1, H, 1, 1)
    bits, g = s["bits"], s["group_size"]
    per, top = 32 // bits, 2 ** bits - 1
    shifts = torch.arange(0, 32, bits, device=slot.device, dtype=torch.int32)
    code = ((s["k_packed"][b, h, slot][..., None] >> shifts) & top).flatten(-2).float()
    k = (code * s["k_scale"][b, h, slot // g].float() + s["k_zero"][b, h, slot // g].float()).half().float()
    code = ((s["v_packed"][b, h, slot // per] >> (slot % per * bits).to(torch.int32)[..., None]) & top).float()
    scale, zero = (s[x].transpose(2, 3)[b, h, slot].float().repeat_interleave(g, -1) for x in ("v_scale", "v_zero"))
    return k, (code * scale + zero).half().float()


def _plain_attend(state):
    case, q, s = state["case"], state["q"], state["store"]
    B, hq, sq, d = q.shape
    hkv, n, block, qb = case["hkv"], case["packed"], case["block"], case["query_block"]
    rows = _tiles_of(q, case).float()
    T, G = rows.shape[2], rows.shape[4]
    blocks = state["blocks"].long()
    slot = blocks[..., None] * block + torch.arange(block, device=q.device)
    slot = torch.where((blocks[..., None] < 0) | (slot >= n), torch.full_like(slot, n), slot).flatten(-2)      # n: none
    k, v = _gathered(s, slot.clamp_max(n - 1))
    end = _ends(case, state["lens"], q.device)[:, None]                                       # [B, 1, T, query_block]
    x = rows.reshape(B, hkv, T, qb * G, d)
    near = torch.matmul(x, k.transpose(3, 4)).view(B, hkv, T, qb, G, -1)
    near = near.masked_fill((slot[:, :, :, None] >= end[..., None].clamp_max(n))[:, :, :, :, None], float("-inf"))
    kt, vt = s["k_tail"].float(), s["v_tail"].float()
    flat = x.reshape(B, hkv, T * qb * G, d)
    late = torch.matmul(flat, kt.transpose(2, 3)).view(B, hkv, T, qb, G, -1)
    at = n + torch.arange(case["tail"], device=q.device)
    late = late.masked_fill((at >= end[..., None])[:, :, :, :, None], float("-inf"))
    p = torch.cat((near, late), -1) * state["scale"]
    m = p.amax(-1, keepdim=True)
    p = (p - m.masked_fill(m == float("-inf"), 0)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1)                                                   # a row that sees nothing is zero
    o = torch.matmul(p[..., : near.shape[-1]].reshape(B, hkv, T, qb * G, -1), v).view(B, hkv, T, qb, G, d)
    o = o + torch.matmul(p[..., near.shape[-1]:].reshape(B, hkv, T * qb * G, -1), vt).view(B, hkv, T, qb, G, d)
    return o.permute(0, 1, 4, 2, 3, 5).reshape(B, hq, T * qb, d)[:, :, :sq].to(q.dtype).contiguous()


def run(state):
    case = state["case"]
    if own:
        from veloxquant_mlx_amd import kernels as K
        if case["kind"] == "norm_rope":
            return K.norm_rotary_embed(state["q"], state["k"], q_weight=state["qw"], k_weight=state["kw"], norm_eps=NORM_EPS,
                                       inv_freq=state["inv_freq"], offset=state["first"], traditional=case["traditional"])
        if case["kind"] == "select":
            return K.select_blocks(state["q"], state["k_scale"], state["k_zero"], case["count"], levels=case["levels"], group_size=case["group"],
                                   n_packed=case["packed"], n_tail=case["tail"], block_size=case["block"], query_block=case["query_block"],
                                   first=case["first"], recent=case["recent"], causal=True, seq_lens=state["lens"])
        return K.block_sparse_attend(state["q"], state["blocks"], **state["store"], block_size=case["block"], query_block=case["query_block"],
                                     scale=state["scale"], causal=True, seq_lens=state["lens"])
    if case["kind"] == "norm_rope":
        q = state["q"]
        at = state["first"][:, None] + torch.arange(case["seq"], device=q.device)
        angle = at[:, None, :, None].double() * state["inv_freq"]
        cos, sin = angle.cos().float(), angle.sin().float()
        return tuple(_plain_norm_rope(x, w, cos, sin, case["dims"], case["traditional"]).to(x.dtype)
                     for x, w in ((q, state["qw"]), (state["k"], state["kw"])))
    return _plain_select(state) if case["kind"] == "select" else _plain_attend(state)


def work(case):
    B, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "norm_rope":
        rows, weights = B * case["seq"] * (hq + hkv), (hq + hkv if case["head_weights"] else 2)
        return {"bytes": 2 * rows * d * size + weights * d * size + case["dims"] * 4 + 8 * B, "flops": rows * (case["dims"] * 3 + 4 * d)}
    sq, n, block, qb, G = case["sq"], case["packed"], case["block"], case["query_block"], hq // hkv
    tiles = -(-sq // qb)
    bytes_of, flops = B * hq * sq * d * size + 4 * B * hkv * tiles * case["count"], 0
    if case["kind"] == "attend":
        bytes_of += B * hq * sq * d * size
    for live in _lengths(case):
        packed, tail = min(live, n), max(0, live - n)
        seen = [max(0, min(packed, live - sq + i + 1)) for i in range(sq)]
        if case["kind"] == "select":
            bytes_of += hkv * -(-packed // case["group"]) * d * 2 * (4 if case["meta"] == "float32" else 2)
            flops += 4 * hq * d * sum(-(-x // case["group"]) for x in seen)
            continue
        # bytes of a packed slot and kv head: codes of k and v, scale and zero of a key group spread over its tokens, of the value groups
        slot = 2 * d * case["bits"] / 8 + 2 * d * 4 / case["group"]
        chosen = case["count"] * block
        bytes_of += hkv * (min(packed, tiles * chosen) * slot + tail * 2 * d * size)
        flops += 4 * d * hq * sum(min(x, chosen) + max(0, min(tail, live - sq + i + 1 - n)) for i, x in enumerate(seen))
    return {"bytes": int(bytes_of), "flops": int(flops)}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _exact_slots(s, b, h, at, which):
    """Keys or values of packed slots `at` of one kv head of one sequence in 64 bits, [n, D]."""
    bits, g = s["bits"], s["group_size"]
    per, words = 32 // bits, s[which + "_packed"][b, h].long() & 0xFFFFFFFF
    scale, zero = s[which + "_scale"][b, h].double(), s[which + "_zero"][b, h].double()
    if which == "k":
        c = torch.arange(scale.shape[1], device=at.device)
        code = (words[at][:, c // per] >> (c % per * bits)) & (2 ** bits - 1)
        return (code.double() * scale[at // g] + zero[at // g]).half().double()
    code = (words[at // per] >> (at % per * bits)[:, None]) & (2 ** bits - 1)
    c = torch.arange(words.shape[1], device=at.device) // g
    return (code.double() * scale[c][:, at].T + zero[c][:, at].T).half().double()


def exact(case, seed):
    if case["kind"] == "select":
        return None                                   # whole numbers
    B, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
    if case["kind"] == "norm_rope":
        state = prepare(case, seed)
        r, out = case["dims"], []
        place = state["first"].double().view(-1, 1) + torch.arange(case["seq"], device="cuda", dtype=torch.float64)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), place.view(B, 1, -1, 1) * state["inv_freq"])
        for x, w in ((state["q"], state["qw"]), (state["k"], state["kw"])):
            x, w = x.double(), w.double()
            y = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / d + NORM_EPS) * w.view(1, -1, 1, d)
            even, odd = (slice(0, r, 2), slice(1, r, 2)) if case["traditional"] else (slice(0, r // 2), slice(r // 2, r))
            z = torch.complex(y[..., even], y[..., odd]) * turn
            y[..., even], y[..., odd] = z.real, z.imag
            out.append(y)
        return tuple(out)
    sq, qb, block, n, G = case["sq"], case["query_block"], case["block"], case["packed"], hq // hkv
    tiles = -(-sq // qb)
    if B * hkv * tiles > 4000:
        return None
    state = prepare(case, seed)
    s = state["store"]
    out = torch.zeros((B, hq, sq, d), dtype=torch.float64, device="cuda")
    lens, lists = _lengths(case), state["blocks"].tolist()
    inside = torch.arange(block, device="cuda")
    for b in range(B):
        newest = torch.arange(max(0, lens[b] - n), device="cuda")
        for h in range(hkv):
            for t in range(tiles):
                named = torch.tensor([j for j in lists[b][h][t] if j >= 0], dtype=torch.int64, device="cuda")
                at = (named[:, None] * block + inside).flatten()
                at = at[at < min(n, lens[b])]
                k = torch.cat((_exact_slots(s, b, h, at, "k"), s["k_tail"][b, h, newest].double()))
                v = torch.cat((_exact_slots(s, b, h, at, "v"), s["v_tail"][b, h, newest].double()))
                place = torch.cat((at, n + newest))
                i = torch.arange(t * qb, min(sq, (t + 1) * qb), device="cuda")
                hidden = place > lens[b] - sq + i[:, None]
                x = state["q"][b, h * G: (h + 1) * G, i].double()
                w = torch.softmax((x @ k.T * state["scale"]).masked_fill(hidden, float("-inf")), -1)
                out[b, h * G: (h + 1) * G, i] = torch.nan_to_num(w) @ v
    return out
