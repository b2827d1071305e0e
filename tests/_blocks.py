"""Chosen blocks in 64 bits: what the tests of block choice and of attention over blocks compare with."""

import torch


def live_of(B, n_packed, n_tail, lens):
    room = n_packed + n_tail
    return torch.full((B,), room, device="cuda") if lens is None else lens.clamp(0, room)


def ends(B, Sq, n_packed, n_tail, lens, causal):
    """[B, Sq]: one past the last slot that a query sees."""
    live = live_of(B, n_packed, n_tail, lens)[:, None]
    return ((live - Sq + torch.arange(Sq, device="cuda") + 1).clamp_min(0).minimum(live) if causal else live.expand(B, Sq))


def group_bounds(q, k_scale, k_zero, levels):
    """[B, Hq, Sq, groups] in 64 bits: the largest product that a key of the group can have."""
    G = q.shape[1] // k_scale.shape[1]
    z = k_zero.double().repeat_interleave(G, 1)
    top = z + levels * k_scale.double().repeat_interleave(G, 1)
    out = []
    for i in range(q.shape[2]):
        x = q[:, :, i, None].double()
        out.append(torch.maximum(x * z, x * top).sum(-1))
    return torch.stack(out, 2)


def choose(q, k_scale, k_zero, n_select, *, levels, group_size, n_packed, n_tail=0, block_size=None, query_block=1, first=0, recent=0,
           causal=False, seq_lens=None):
    """What ``select_blocks`` returns, by sorting."""
    B, Hq, Sq, _ = q.shape
    H, block = k_scale.shape[1], block_size or group_size
    groups = -(-n_packed // group_size)
    out = torch.full((B, H, -(-Sq // query_block), n_select), -1, dtype=torch.int32)
    if groups == 0:
        return out.cuda()
    bound = group_bounds(q, k_scale[:, :, :groups], k_zero[:, :, :groups], levels).view(B, H, Hq // H, Sq, groups).amax(2).cpu()
    end = ends(B, Sq, n_packed, n_tail, seq_lens, causal).clamp_max(n_packed).tolist()
    for b in range(B):
        for t in range(out.shape[2]):
            queries = range(t * query_block, min(Sq, (t + 1) * query_block))
            visible = -(-end[b][queries[-1]] // block)
            for h in range(H):
                if visible <= n_select:
                    out[b, h, t, :visible] = torch.arange(visible, dtype=torch.int32)
                    continue
                score = []
                for j in range(visible):
                    near = [float(bound[b, h, i, u]) for i in queries for u in range(j * block // group_size, min((j + 1) * block // group_size, groups))
                            if u * group_size < end[b][i]]
                    top = float("nan") if any(x != x for x in near) else max(near)
                    kept = j < first or j >= visible - recent
                    score.append((0 if kept else 1 if top != top else 2, 0.0 if kept or top != top else -top, j))
                out[b, h, t] = torch.tensor(sorted(j for _, _, j in sorted(score)[:n_select]), dtype=torch.int32)
    return out.cuda()


def times_seen(blocks, block, query_block, B, Sq, n_packed, n_tail, lens, causal):
    """[B, Hkv, Sq, n_packed + n_tail]: how often a query sees a slot."""
    H, n = blocks.shape[1], n_packed + n_tail
    times = torch.zeros((B, H, blocks.shape[2], n), dtype=torch.float64, device="cuda")
    slot = torch.arange(n_packed, device="cuda")
    for x in range(blocks.shape[3]):
        e = blocks[..., x, None].long()
        times[..., :n_packed] += ((slot >= e * block) & (slot < (e + 1) * block) & (e >= 0)).double()
    times[..., n_packed:] = 1
    times = times.repeat_interleave(query_block, 2)[:, :, :Sq]
    end = ends(B, Sq, n_packed, n_tail, lens, causal)
    return times * (torch.arange(n, device="cuda") < end[:, None, :, None])


def attend(q, k, v, times, scale, u):
    """sum p v / sum p with p = times * exp(scale q k) in 64 bits, and how far a kernel may be from it (as ``tests._spans.attend``): float32
    scores and sums, weights rounded by ``u`` of their size."""
    B, Hq, Sq, D = q.shape
    G = Hq // k.shape[1]
    q, k, v, times = q.double(), k.repeat_interleave(G, 1), v.repeat_interleave(G, 1), times.repeat_interleave(G, 1)
    seen = times > 0
    s = (q @ k.transpose(2, 3)) * scale
    m = s.masked_fill(~seen, float("-inf")).amax(-1, keepdim=True)
    p = times * torch.exp((s - m.nan_to_num(neginf=0.0)).masked_fill(~seen, float("-inf")))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    size = ((q.abs() @ k.abs().transpose(2, 3)) * abs(scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    big = q.abs().amax(-1, keepdim=True) * (k.abs().amax((2, 3), keepdim=True) if k.shape[2] else 0) * abs(scale)
    ds = (D + 2) * 2.0 ** -24 * size + 2.0 ** -11 * big
    far = (p @ v.abs()) * (2 * u + 2 * ds + 2.0 ** -18 + times.sum(-1, keepdim=True) * 2.0 ** -24)
    return p @ v, far
