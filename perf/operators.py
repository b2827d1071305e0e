"""Operators that stand around a compressed KV cache: rotary positions in front of it, attention of a batch whose sequences
share one long prefix, and differential attention.

``run`` computes each in its plain form, elementary torch operations in 32 bits (angles in 64), or, where ``own`` is true,
through this package's functions.

A packed store is laid out as the caches keep it: keys ``int32 [B, H, tokens, D / per]``, a word holding ``per = 32 / bits``
consecutive channels of a token (lowest bits first), scale and zero ``float16 [B, H, tokens / group, D]``; values
``int32 [B, H, tokens / per, D]``, a word holding ``per`` consecutive tokens of a channel, scale and zero
``float16 [B, H, D / group, tokens]``.  A packed slot stands for the fp16 number ``code * scale + zero``.  The newest tokens
follow as plain rows (the tail).
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
HEADS = {64: [(32, 8), (14, 2), (9, 3)], 128: [(32, 8), (28, 4), (40, 10)], 256: [(12, 4), (8, 4)]}
NORM_EPS = 1e-5
GAIN = 0.2   # 1 - 0.8, the gain of a differential layer's head norm


def listed():
    return [
        # one decode step of one sequence: queries and keys of one token, launch latency and nothing else
        dict(name="rope_step", kind="rope", hq=32, hkv=8, d=128, dims=128, batch=1, seq=1, traditional=False, scaling="none",
             far=9000, ragged=False, dtype="bfloat16"),
        # a prompt of 8k tokens, half layout, frequencies scaled by parts for a long context
        dict(name="rope_prompt", kind="rope", hq=32, hkv=8, d=128, dims=128, batch=1, seq=8192, traditional=False, scaling="by_parts",
             far=0, ragged=False, dtype="bfloat16"),
        # chunks of an odd length of a batch, each at its own far position, interleaved pairs over a quarter of the head
        dict(name="rope_part_ragged", kind="rope", hq=12, hkv=4, d=256, dims=64, batch=7, seq=1003, traditional=True, scaling="linear",
             far=900000, ragged=True, dtype="float16"),
        # float32 rows, small heads
        dict(name="rope_float32", kind="rope", hq=9, hkv=3, d=64, dims=64, batch=2, seq=2047, traditional=False, scaling="none",
             far=100000, ragged=False, dtype="float32"),
        # a handful of answers to a short prompt, 2 bits: latency
        dict(name="shared_short", kind="shared", hq=32, hkv=8, d=128, batch=4, prefix=640, prefix_tail=60, packed=0, tail=33, sq=1,
             bits=2, group=32, ragged=False, dtype="float16"),
        # a batch of odd size over a 16k document, 4 bits, answers of different lengths
        dict(name="shared_16k_ragged", kind="shared", hq=40, hkv=10, d=128, batch=21, prefix=16384, prefix_tail=140, packed=512, tail=131,
             sq=1, bits=4, group=32, ragged=True, dtype="float16"),
        # 128 answers over a 32k prompt with a thousand tokens each: the largest
        dict(name="shared_32k_batch", kind="shared", hq=32, hkv=8, d=128, batch=128, prefix=32768, prefix_tail=128, packed=896, tail=130,
             sq=1, bits=4, group=64, ragged=False, dtype="float16"),
        # plain rows, five proposed tokens a sequence checked at once
        dict(name="shared_rows_verify", kind="shared", hq=32, hkv=8, d=128, batch=12, prefix=0, prefix_tail=4099, packed=0, tail=261, sq=5,
             bits=4, group=32, ragged=False, dtype="bfloat16"),
        # self-attention of a whole prompt with two maps a head
        dict(name="diff_prompt_4k", kind="diff", hq=32, hkv=8, d=128, batch=1, packed=0, tail=4096, sq=4096, bits=4, group=32,
             ragged=False, norm=True, dtype="bfloat16"),
        # prompts of an odd length, heads of 256 channels
        dict(name="diff_prompt_d256", kind="diff", hq=12, hkv=4, d=256, batch=3, packed=0, tail=1001, sq=1001, bits=4, group=32,
             ragged=False, norm=True, dtype="float16"),
        # one step of one sequence over a short compressed context: latency
        dict(name="diff_step_short", kind="diff", hq=32, hkv=8, d=128, batch=1, packed=576, tail=129, sq=1, bits=2, group=32,
             ragged=False, norm=True, dtype="float16"),
        # a serving batch at 32k, 4 bits, of different lengths: the bytes of the cache count
        dict(name="diff_step_32k", kind="diff", hq=32, hkv=8, d=128, batch=16, packed=32768, tail=132, sq=1, bits=4, group=64,
             ragged=True, norm=True, dtype="float16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "shared", "diff", "diff_step"])
    if kind == "rope":
        d = rng.choice([64, 128, 128, 256])
        hq, hkv = rng.choice(HEADS[d])
        batch = _log_int(rng, 1, 16)
        return dict(kind="rope", hq=hq, hkv=hkv, d=d, dims=rng.choice([d, d, d // 2, d // 4]), batch=batch,
                    seq=max(1, min(_log_int(rng, 1, 8192), 8192 * 40 * 128 // (batch * (hq + hkv) * d))), traditional=rng.random() < 0.4,
                    scaling=rng.choice(["none", "linear", "by_parts"]), far=rng.choice([0, 5000, 131000, 1000000]), ragged=rng.random() < 0.4,
                    dtype=rng.choice(["float16", "bfloat16", "bfloat16", "float32"]))
    d = rng.choice([128, 128, 256])
    hq, hkv = rng.choice(HEADS[d])
    bits, group = rng.choice([(2, 32), (4, 32), (4, 64)])
    rows = rng.random() < 0.25        # plain rows only
    dtype = rng.choice(["float16", "bfloat16"]) if rows else "float16"
    if kind == "shared":
        if rows and rng.random() < 0.5:
            d = 64
            hq, hkv = rng.choice(HEADS[d])
        batch, n = _log_int(rng, 1, 128), _log_int(rng, 300, 33000)
        sq = rng.choice([1, 1, 1, _log_int(rng, 2, 9)])
        batch = max(1, min(batch, 128 * 32 * 32768 * 128 // (hq * sq * n * d)))
        own_tokens = max(sq, min(_log_int(rng, 1, 1400), 128 * 8 * 1026 * 128 // (batch * hkv * d)))
        packed = 0 if rows else max(0, own_tokens - 128) // 64 * 64
        return dict(kind="shared", hq=hq, hkv=hkv, d=d, batch=batch, prefix=0 if rows else n // 64 * 64, prefix_tail=min(n, 9000) if rows else
                    rng.choice([0, 7, 130]) + (n < 64), packed=packed, tail=own_tokens - packed, sq=sq, bits=bits, group=group,
                    ragged=sq == 1 and rng.random() < 0.4, dtype=dtype)
    if kind == "diff":
        batch, n = _log_int(rng, 1, 4), _log_int(rng, 100, 4096)
        n = max(64, min(n, int(4096 * math.sqrt(32 * 128 / (batch * hq * d)))))
        return dict(kind="diff", hq=hq, hkv=hkv, d=d, batch=batch, packed=0, tail=n, sq=n, bits=bits, group=group, ragged=False,
                    norm=rng.random() < 0.7, dtype=rng.choice(["float16", "bfloat16"]))
    batch = _log_int(rng, 1, 16)
    n = max(200, min(_log_int(rng, 200, 33000), 16 * 32900 * 8 * 128 // (batch * hkv * d)))
    packed = 0 if rows else (n - 130) // 64 * 64 if n > 194 else 64
    return dict(kind="diff", hq=hq, hkv=hkv, d=d, batch=batch, packed=packed, tail=min(n - packed, 9000), sq=1, bits=bits, group=group,
                ragged=batch > 1 and rng.random() < 0.4, norm=rng.random() < 0.7, dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """Live slots of every sequence: from a third to the whole of the room."""
    n = case["packed"] + case["tail"]
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


def _pack(codes, bits):
    """Codes along the last axis to int32 words, lowest bits first."""
    per = 32 // bits
    codes = codes.view(*codes.shape[:-1], -1, per)
    words = codes[..., 0].to(torch.int32)
    for j in range(1, per):
        words |= codes[..., j].to(torch.int32) << (bits * j)
    return words


def _quantise(x, group, bits):
    """Groups along the last axis: codes, and scale and zero as float16."""
    g = x.view(*x.shape[:-1], -1, group)
    lo, hi = g.amin(-1), g.amax(-1)
    scale, zero = ((hi - lo) / (2 ** bits - 1)).clamp_min(1e-4).half(), lo.half()
    codes = ((g - zero.float()[..., None]) / scale.float()[..., None]).round_().clamp_(0, 2 ** bits - 1).to(torch.uint8)
    return codes.view(x.shape), scale, zero


def _store(gen, batch, hkv, d, packed, tail, bits, group, dtype, factors):
    """Keys and values of `packed` quantised tokens and `tail` plain ones."""
    s = dict(n_packed=packed, n_tail=tail, bits=bits, group_size=group, v_layout="token")
    if packed:
        per = 32 // bits
        like = dict(dtype=torch.int32, device="cuda")
        half = dict(dtype=torch.float16, device="cuda")
        s["k_packed"] = torch.empty((batch, hkv, packed, d // per), **like)
        s["v_packed"] = torch.empty((batch, hkv, packed // per, d), **like)
        s["k_scale"], s["k_zero"] = (torch.empty((batch, hkv, packed // group, d), **half) for _ in range(2))
        s["v_scale"], s["v_zero"] = (torch.empty((batch, hkv, d // group, packed), **half) for _ in range(2))
        for b in range(batch):
            k = torch.randn((hkv, packed, d), generator=gen, device="cuda") * factors
            codes, scale, zero = _quantise(k.transpose(1, 2).contiguous(), group, bits)       # [H, D, n]: groups of tokens
            s["k_packed"][b] = _pack(codes.transpose(1, 2).contiguous(), bits)
            s["k_scale"][b], s["k_zero"][b] = scale.transpose(1, 2), zero.transpose(1, 2)
            codes, scale, zero = _quantise(torch.randn((hkv, packed, d), generator=gen, device="cuda"), group, bits)
            s["v_packed"][b] = _pack(codes.transpose(1, 2).contiguous(), bits).transpose(1, 2)
            s["v_scale"][b], s["v_zero"][b] = scale.transpose(1, 2), zero.transpose(1, 2)
    if tail:
        s["k_tail"] = (torch.randn((batch, hkv, tail, d), generator=gen, device="cuda") * factors).to(dtype)
        s["v_tail"] = torch.randn((batch, hkv, tail, d), generator=gen, device="cuda").to(dtype)
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    B, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
    if case["kind"] == "rope":
        S = case["seq"]
        # queries, keys and values as one projection leaves them: views [B, H, S, D] of its rows
        rows = torch.randn((B, S, (hq + 2 * hkv) * d), generator=gen, device="cuda").to(dtype)
        q = rows[..., : hq * d].view(B, S, hq, d).transpose(1, 2)
        k = rows[..., hq * d: (hq + hkv) * d].view(B, S, hkv, d).transpose(1, 2)
        first = torch.full((B,), case["far"], device="cuda", dtype=torch.int64)
        if case["ragged"]:
            first -= torch.randint(0, case["far"] // 2 + 1, (B,), generator=gen, device="cuda")
        return dict(case=case, q=q, k=k, inv_freq=_frequencies(case["dims"], case["scaling"]).cuda(), first=first)
    factors = torch.randn((d,), generator=gen, device="cuda").mul(0.5).exp()
    state = dict(case=case, scale=1 / math.sqrt(d if case["kind"] == "shared" else d // 2))
    state["q"] = torch.randn((B, hq, case["sq"], d), generator=gen, device="cuda").to(dtype)
    how = (case["bits"], case["group"], dtype, factors)
    state["own_slots"] = _store(gen, B, hkv, d, case["packed"], case["tail"], *how)
    state["lens"] = torch.tensor(_lengths(case), device="cuda") if case["ragged"] else None
    if case["kind"] == "shared":
        state["prefix"] = _store(gen, 1, hkv, d, case["prefix"], case["prefix_tail"], *how)
    else:
        state["lam"] = torch.rand((hq,), generator=gen, device="cuda") * 0.6 + 0.2
        state["weight"] = torch.rand((d,), generator=gen, device="cuda") + 0.5 if case["norm"] else None
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _plain_rope(x, cos, sin, dims, traditional):
    x = x.float()
    if traditional:
        a, b = x[..., 0:dims:2], x[..., 1:dims:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., : dims // 2], x[..., dims // 2: dims]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., dims:]), dim=-1)


def _codes(words, bits):
    shifts = torch.arange(0, 32, bits, device=words.device, dtype=torch.int32)
    return ((words[..., None] >> shifts) & (2 ** bits - 1)).flatten(-2)


def _slots(s):
    """A store's keys and values in 32 bits, [B, H, n, D]."""
    k, v = [], []
    if s["n_packed"]:
        g, bits = s["group_size"], s["bits"]
        codes = _codes(s["k_packed"], bits).float()
        k.append((codes * s["k_scale"].float().repeat_interleave(g, 2) + s["k_zero"].float().repeat_interleave(g, 2)).half().float())
        codes = _codes(s["v_packed"].transpose(2, 3), bits).float()                             # [B, H, D, n]
        codes = codes * s["v_scale"].float().repeat_interleave(g, 2) + s["v_zero"].float().repeat_interleave(g, 2)
        v.append(codes.half().float().transpose(2, 3))
    if s["n_tail"]:
        k.append(s["k_tail"].float())
        v.append(s["v_tail"].float())
    return (k[0], v[0]) if len(k) == 1 else (torch.cat(k, 2), torch.cat(v, 2))


def _visible(sq, n, lens, device):
    """[B or 1, 1, Sq, n]: query i of a sequence of n slots sees the slots up to n - Sq + i."""
    slot = torch.arange(n, device=device)
    last = (n if lens is None else lens.view(-1, 1)) - sq + torch.arange(sq, device=device)
    return (slot <= last[..., None]).view(-1, 1, sq, n)


def _softmax(scores):
    e = (scores - scores.amax(-1, keepdim=True)).exp()
    return e / e.sum(-1, keepdim=True)


def run(state):
    case = state["case"]
    B, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
    if own:
        from veloxquant_mlx_amd import kernels as K
        if case["kind"] == "rope":
            return K.rotary_embed(state["q"], state["k"], inv_freq=state["inv_freq"], offset=state["first"], traditional=case["traditional"])
        if case["kind"] == "shared":
            return K.shared_prefix_attend(state["q"], state["prefix"], **state["own_slots"], scale=state["scale"], causal=True,
                                          seq_lens=state["lens"])
        return K.differential_attend(state["q"], state["lam"], **state["own_slots"], scale=state["scale"], causal=True,
                                     seq_lens=state["lens"], norm_weight=state["weight"], norm_eps=NORM_EPS,
                                     gain=GAIN if case["norm"] else 1.0)
    q = state["q"]
    if case["kind"] == "rope":
        at = state["first"][:, None] + torch.arange(case["seq"], device=q.device)
        angle = at[:, None, :, None].double() * state["inv_freq"]
        cos, sin = angle.cos().float(), angle.sin().float()
        return tuple(_plain_rope(x, cos, sin, case["dims"], case["traditional"]).to(x.dtype) for x in (q, state["k"]))
    sq, G = case["sq"], hq // hkv
    k, v = _slots(state["own_slots"])
    n = k.shape[2]
    hidden = ~_visible(sq, n, state["lens"], q.device)
    if case["kind"] == "shared":
        rows = q.float().view(B, hkv, G * sq, d)
        pk, pv = _slots(state["prefix"])
        n_prefix = pk.shape[2]
        together = rows.transpose(0, 1).reshape(hkv, B * G * sq, d)                # all sequences' rows of a kv head
        far = torch.matmul(together, pk[0].transpose(1, 2)).view(hkv, B, G * sq, n_prefix).transpose(0, 1)
        near = torch.matmul(rows, k.transpose(2, 3)).view(B, hq, sq, n).masked_fill(hidden, float("-inf")).view(B, hkv, G * sq, n)
        p = _softmax(torch.cat((far, near), -1) * state["scale"])
        o = torch.matmul(p[..., :n_prefix].transpose(0, 1).reshape(hkv, B * G * sq, n_prefix), pv[0])
        o = o.view(hkv, B, G * sq, d).transpose(0, 1) + torch.matmul(p[..., n_prefix:], v)
        return o.reshape(B, hq, sq, d).to(q.dtype)
    h = d // 2
    maps = []
    for half in (slice(0, h), slice(h, d)):
        s = torch.matmul(q[..., half].float().reshape(B, hkv, G * sq, h), k[..., half].transpose(2, 3)).view(B, hq, sq, n)
        maps.append(_softmax((s * state["scale"]).masked_fill_(hidden, float("-inf"))))
    a = maps[0] - state["lam"].view(1, hq, 1, 1) * maps[1]
    o = torch.matmul(a.view(B, hkv, G * sq, n), v).view(B, hq, sq, d)
    if state["weight"] is not None:
        o = o / (o.square().mean(-1, keepdim=True) + NORM_EPS).sqrt() * state["weight"] * GAIN
    return o.to(q.dtype)


def _seen(case):
    """Pairs of a query position and a slot of its own sequence that it sees, over the batch."""
    sq, n = case["sq"], case["packed"] + case["tail"]
    lens = _lengths(case) if case["ragged"] else [n] * case["batch"]
    return sum(sum(max(0, length - sq + i + 1) for i in range(sq)) for length in lens), sum(lens)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    B, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
    if case["kind"] == "rope":
        rows = B * case["seq"] * (hq + hkv)
        return {"bytes": 2 * rows * d * size + case["dims"] * 4 + 8 * B, "flops": rows * case["dims"] * 3}
    seen, live = _seen(case)
    n = case["packed"] + case["tail"]
    # bytes of a packed slot and kv head: codes of k and v, scale and zero of a key group spread over its tokens, of the value groups
    slot = 2 * d * case["bits"] / 8 + d * 4 / case["group"] + d / case["group"] * 4
    packed = live * case["packed"] / n if n else 0
    size_of = hkv * (packed * slot + (live - packed) * 2 * d * size)
    rows = B * hq * case["sq"]
    if case["kind"] == "shared":
        size_of += hkv * (case["prefix"] * slot + case["prefix_tail"] * 2 * d * size)
        flops = 4 * d * (rows * (case["prefix"] + case["prefix_tail"]) + hq * seen)
    else:
        flops = 4 * d * hq * seen      # two maps over half the channels each, one product of their difference with the values
    return {"bytes": int(size_of + 2 * rows * d * size), "flops": int(flops)}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _exact_rows(s, b, h, which):
    """Keys or values of one kv head of one sequence in 64 bits, [n, D]."""
    out = []
    if s["n_packed"]:
        bits, g = s["bits"], s["group_size"]
        w = s[which + "_packed"][b, h].long() & 0xFFFFFFFF
        code = torch.stack([(w >> (bits * j)) & (2 ** bits - 1) for j in range(32 // bits)], -1).double()
        scale, zero = s[which + "_scale"][b, h].double(), s[which + "_zero"][b, h].double()
        if which == "k":
            code = code.reshape(w.shape[0], -1)
            group = torch.arange(code.shape[0], device=w.device) // g
            x = code * scale[group] + zero[group]
        else:
            code = code.permute(0, 2, 1).reshape(-1, w.shape[1])
            group = torch.arange(code.shape[1], device=w.device) // g
            x = code * scale[group].T + zero[group].T
        out.append(x.half().double())
    if s["n_tail"]:
        out.append(s[which + "_tail"][b, h].double())
    return torch.cat(out)


def exact(case, seed):
    state = prepare(case, seed)
    B, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
    if case["kind"] == "rope":
        r, out = case["dims"], []
        place = state["first"].double().view(-1, 1) + torch.arange(case["seq"], device="cuda", dtype=torch.float64)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), place.view(B, 1, -1, 1) * state["inv_freq"])
        for x in (state["q"], state["k"]):
            y = x.double().clone()
            even, odd = (slice(0, r, 2), slice(1, r, 2)) if case["traditional"] else (slice(0, r // 2), slice(r // 2, r))
            z = torch.complex(x[..., even].double(), x[..., odd].double()) * turn
            y[..., even], y[..., odd] = z.real, z.imag
            out.append(y)
        return tuple(out)
    sq, G = case["sq"], hq // hkv
    if case["kind"] == "diff" and B * hq * sq * (case["packed"] + case["tail"]) > 2 ** 30:
        return None
    out = torch.empty((B, hq, sq, d), dtype=torch.float64, device="cuda")
    lens = state["lens"].tolist() if state["lens"] is not None else [case["packed"] + case["tail"]] * B
    for h in range(hkv):
        if case["kind"] == "shared":
            shared = [_exact_rows(state["prefix"], 0, h, w) for w in "kv"]
        for b in range(B):
            k, v = (_exact_rows(state["own_slots"], b, h, w)[: lens[b]] for w in "kv")
            before = 0
            if case["kind"] == "shared":
                before = shared[0].shape[0]
                k, v = torch.cat((shared[0], k)), torch.cat((shared[1], v))
            x = state["q"][b, h * G: (h + 1) * G].double()
            at = before + lens[b] - sq + torch.arange(sq, device="cuda")
            mask = torch.arange(k.shape[0], device="cuda") > at[:, None]
            if case["kind"] == "shared":
                s = (x @ k.T * state["scale"]).masked_fill(mask, float("-inf"))
                out[b, h * G: (h + 1) * G] = torch.softmax(s, -1) @ v
                continue
            m = d // 2
            one = torch.softmax((x[..., :m] @ k[:, :m].T * state["scale"]).masked_fill(mask, float("-inf")), -1)
            two = torch.softmax((x[..., m:] @ k[:, m:].T * state["scale"]).masked_fill(mask, float("-inf")), -1)
            lam = state["lam"][h * G: (h + 1) * G].double().view(-1, 1, 1)
            o = one @ v - lam * (two @ v)
            if state["weight"] is not None:
                o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + NORM_EPS) * state["weight"].double() * GAIN
            out[b, h * G: (h + 1) * G] = o
    return out
