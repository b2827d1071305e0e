"""Stores of slots and the 64-bit attention that the tests of shared prefixes and differential attention compare with."""

import math

import torch

from veloxquant_mlx_amd import kernels as K


def store(B, H, n_packed, n_tail, D, bits=4, group=32, v_layout="token", dtype=torch.float16, meta=torch.float16, seed=0, spare=0, view=False):
    """Keys and values of ``n_packed`` quantised slots and ``n_tail`` plain ones: the arguments of the attention calls and, in
    64 bits, the rows they stand for.  ``spare``: room behind the live slots, packed and plain, filled with NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    factors = torch.randn(D, generator=g, device="cuda").mul(0.5).exp()
    s = dict(n_packed=n_packed, n_tail=n_tail, bits=bits, group_size=group, v_layout=v_layout)
    ks, vs = [], []
    if n_packed:
        per = 32 // bits
        cap = n_packed + spare
        unit = math.lcm(group, per)
        cap = -(-cap // unit) * unit
        k = (torch.randn((B, H, n_packed, D), generator=g, device="cuda") * factors).half()
        v = torch.randn((B, H, n_packed, D), generator=g, device="cuda").half()
        kp, ksc, kz = K.kivi_quant_pack(k, -2, group, bits, meta_dtype=meta)
        vp, vsc, vz = K.kivi_quant_pack(v, -1, group, bits, meta_dtype=meta, v_layout=v_layout)
        ks.append(_rows(kp.transpose(2, 3), ksc, kz, bits, D, n_packed, group, "k"))
        vs.append(_rows(vp, vsc, vz, bits, D, n_packed, group, v_layout))
        nan = float("nan")

        def room(t, axis, n):   # the same array with room for n along an axis
            shape = list(t.shape)
            shape[axis] = n
            big = torch.full(shape, nan, dtype=t.dtype, device="cuda") if t.is_floating_point() else torch.full(shape, -1, dtype=t.dtype, device="cuda")
            big.narrow(axis, 0, t.shape[axis]).copy_(t)
            return big

        s.update(k_packed=room(kp, 2, cap), k_scale=room(ksc, 2, -(-cap // group)), k_zero=room(kz, 2, -(-cap // group)))
        if v_layout == "token":
            s.update(v_packed=room(vp, 2, cap // per), v_scale=room(vsc, 3, cap), v_zero=room(vz, 3, cap))
        else:
            s.update(v_packed=room(vp, 2, cap), v_scale=room(vsc, 2, cap), v_zero=room(vz, 2, cap))
    if n_tail:
        k = (torch.randn((B, H, n_tail, D), generator=g, device="cuda") * factors).to(dtype)
        v = torch.randn((B, H, n_tail, D), generator=g, device="cuda").to(dtype)
        ks.append(k.double())
        vs.append(v.double())
        for name, t in (("k_tail", k), ("v_tail", v)):
            if view:     # rows of a [B, n, H + 1, D] projection
                big = torch.full((B, n_tail + spare, H + 1, D), float("nan"), dtype=dtype, device="cuda").transpose(1, 2)[:, 1:]
            else:
                big = torch.full((B, H, n_tail + spare, D), float("nan"), dtype=dtype, device="cuda")
            big[:, :, :n_tail] = t
            s[name] = big
    none = torch.zeros((B, H, 0, D), dtype=torch.float64, device="cuda")
    return s, torch.cat([none, *ks], 2), torch.cat([none, *vs], 2)


def _rows(words, scale, zero, bits, D, n, group, layout):
    """The fp16 numbers packed slots stand for, in 64 bits, [B, H, n, D]."""
    per = 32 // bits
    at = torch.arange(n, device="cuda")
    ch = torch.arange(D, device="cuda")
    w = (words.long() if words.dtype == torch.int32 else words.long()) & 0xFFFFFFFF
    if layout == "k":          # words [B, H, W, n]
        code = (w[:, :, ch // per] >> (bits * (ch % per))[:, None]) & (2 ** bits - 1)
        code = code.transpose(2, 3)
        sc, z = scale[:, :, at // group], zero[:, :, at // group]
    elif layout == "token":    # words [B, H, n / per, D]
        code = (w[:, :, at // per] >> (bits * (at % per))[:, None]) & (2 ** bits - 1)
        sc, z = (t[:, :, ch // group][..., :n].transpose(2, 3) for t in (scale, zero))
    else:                      # words [B, H, n, W]
        code = (w[..., ch // per] >> (bits * (ch % per))) & (2 ** bits - 1)
        sc, z = scale[..., ch // group], zero[..., ch // group]
    return (code.double() * sc.double() + z.double()).half().double()


def seen(B, Sq, before, n_own, lens, causal, window):
    """[B, Sq, before + n_own] bool: what the queries see."""
    lens = torch.full((B,), n_own, device="cuda") if lens is None else lens.clamp(0, n_own)
    total = (before + lens)[:, None, None]
    slot = torch.arange(before + n_own, device="cuda")
    end = total - Sq + torch.arange(Sq, device="cuda")[:, None] + 1
    m = slot < (end if causal else total.expand(B, Sq, 1))
    if window:
        m = m & (slot >= end - window)
    return m


def attend(q, k, v, mask, scale, u):
    """softmax(q k^T scale) v over the slots that ``mask`` [B, Sq, n] shows, in 64 bits, and how far a kernel may be from it that forms
    scores and sums in float32 and rounds the weights by ``u`` of their size (before the output's own rounding):

    * a score is off by ds: D + 2 float32 roundings of the absolute products' sum and of the multiple of the scale, and one step of fp16 of the
      largest product where a packed slot was rounded twice; a weight by a factor exp(ds), its exponential and reference by 2^-18
    * weights are rounded by u, their sum is formed of the rounded ones; n additions of float32."""
    B, Hq, Sq, D = q.shape
    G = Hq // k.shape[1]
    q, k, v = q.double(), k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = (q @ k.transpose(2, 3)) * scale
    s = s.masked_fill(~mask[:, None], float("-inf"))
    p = torch.softmax(s, -1).nan_to_num(0.0)
    p = p * mask[:, None]
    o = p @ v
    size = (q.abs() @ k.abs().transpose(2, 3)) * abs(scale)
    size = size.masked_fill(~mask[:, None], 0.0).amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros((B, Hq, Sq, 1))
    big = q.abs().amax(-1, keepdim=True) * (k.abs().amax((2, 3), keepdim=True) if k.shape[2] else 0) * abs(scale)
    ds = (D + 2) * 2.0 ** -24 * size + 2.0 ** -11 * big
    far = (p @ v.abs()) * (2 * u + 2 * ds + 2.0 ** -18 + s.shape[-1] * 2.0 ** -24)
    return o, far


def close(got, want, far):
    """One rounding to the output's type on top of ``far``."""
    half_step = torch.finfo(got.dtype).eps / 2
    bound = far * (1 + half_step) + half_step * want.abs() + torch.finfo(got.dtype).smallest_normal
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float(off.max())}, {float((off / bound).max())} of the bound"
