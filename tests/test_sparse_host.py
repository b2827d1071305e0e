"""Refusals of normed rotary positions, block choice and attention over blocks (no GPU)."""

import os
import re

import pytest
import torch

from veloxquant_mlx_amd import _lib, kernels as K
from veloxquant_mlx_amd.cache import KVCacheConfig, KVCacheFactory

REFUSED = (_lib.VQ_ERR_INVALID, _lib.VQ_ERR_UNSUPPORTED)


@pytest.mark.parametrize("struct,mirror", [("vq_norm_rotary_args", _lib.NormRotaryArgs), ("vq_block_select_args", _lib.BlockSelectArgs),
                                           ("vq_block_attend_args", _lib.BlockAttendArgs)])
def test_structures_match_the_header(struct, mirror):
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "veloxquant_hip.h")).read()
    body = text[text.index(f"typedef struct {struct} {{"):text.index(f"}} {struct};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in body.split(";"):
        for part in decl.split("{")[-1].strip().split(","):
            part = re.sub(r"\[.*?\]", "", part).strip()
            if part:
                names.append(re.findall(r"[A-Za-z_][A-Za-z0-9_]*", part)[-1])
    assert names == [f[0] for f in mirror._fields_]


def test_packed_blocks_are_the_structures():
    for pack, mirror in ((_lib.BLOCK_SELECT_PACK, _lib.BlockSelectArgs),):
        values = list(range(1, len(mirror._fields_) + 1))
        a = mirror.from_buffer_copy(pack.pack(*values))
        assert [getattr(a, n) for n, _ in mirror._fields_] == values
    head = bytes(_lib.ROTARY_PACK.size)
    a = _lib.NormRotaryArgs.from_buffer_copy(head + _lib.NORM_PACK.pack(1, 2, 3, 4, 5, 0.5))
    assert list(a.weight) == [1, 2] and list(a.weight_stride) == [3, 4] and a.weight_dtype == 5 and a.eps == 0.5
    b = _lib.BlockAttendArgs.from_buffer_copy(bytes(_lib.STORE_ATTEND_PACK.size) + _lib.BLOCK_LISTS_PACK.pack(1, 2, 3, 4, 5, 6))
    assert (b.blocks, b.count, b.block_tokens, b.query_block, b.counters, b.counters_len) == (1, 2, 3, 4, 5, 6)


def _norm(**kw):
    a = _lib.NormRotaryArgs()
    r = a.rotary
    r.B, r.S, r.D, r.dims, r.inv_freq, r.freq_dtype, r.attention_factor = 1, 4, 8, 8, 4096, _lib.VQ_F64, 1.0
    r.x[0], r.out[0], r.heads[0] = 4096, 8192, 2
    a.eps = 1e-6
    for name, v in kw.items():
        setattr(a if name in ("eps", "weight_dtype") else r, name, v)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(dtype=_lib.VQ_U8), "dtype"), (dict(dims=7), "dims"), (dict(dims=10), "dims"), (dict(layout=2), "layout"), (dict(freq_dtype=_lib.VQ_F16), "frequencies"),
    (dict(positions=4096, pos_dtype=_lib.VQ_F32), "positions"), (dict(inv_freq=None), "frequencies"), (dict(B=-1), "sizes"), (dict(inverse=1), "turned back"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(B=1 << 20, S=1 << 20), "rows")])
def test_norm_rotary_refuses(kw, what):
    lib = _lib.load()
    assert lib.vq_norm_rotary(_norm(**kw), None) in REFUSED
    assert what in _lib.last_error()


def test_norm_rotary_checks_weights_and_rows():
    lib = _lib.load()
    a = _norm(weight_dtype=_lib.VQ_I32)
    a.weight[0] = 4096
    assert lib.vq_norm_rotary(a, None) == _lib.VQ_ERR_INVALID and "weight dtype" in _lib.last_error()
    a = _norm()
    a.weight[0], a.weight_stride[0] = 4096, 3
    assert lib.vq_norm_rotary(a, None) == _lib.VQ_ERR_INVALID and "weight rows" in _lib.last_error()
    a = _norm()
    a.rotary.out[0] = None
    assert lib.vq_norm_rotary(a, None) == _lib.VQ_ERR_INVALID and "outputs must be given" in _lib.last_error()
    assert lib.vq_norm_rotary(None, None) == _lib.VQ_ERR_INVALID
    for empty in (dict(B=0), dict(S=0)):
        assert lib.vq_norm_rotary(_norm(**empty), None) == 0


def test_norm_rotary_embed_refuses():
    q, f = torch.zeros(1, 2, 3, 8), torch.ones(4)
    with pytest.raises(RuntimeError, match="norm_rotary_embed: .*no CPU path"):
        K.norm_rotary_embed(q, inv_freq=f)
    with pytest.raises(ValueError, match=r"norm_rotary_embed: q and k must be \[B, H, S, D\]"):
        K.norm_rotary_embed(q[0], inv_freq=f)
    with pytest.raises(ValueError, match="k_weight without k"):
        K.norm_rotary_embed(q, k_weight=torch.ones(8), inv_freq=f)
    for w in (torch.ones(7), torch.ones(3, 8), torch.ones(1, 2, 8)):
        with pytest.raises(ValueError, match="weight for q"):
            K.norm_rotary_embed(q, q_weight=w, inv_freq=f)
    with pytest.raises(ValueError, match="one dtype"):
        K.norm_rotary_embed(q, q, q_weight=torch.ones(8), k_weight=torch.ones(8).half(), inv_freq=f)
    with pytest.raises(ValueError, match="unsupported dtype"):
        K.norm_rotary_embed(q, q_weight=torch.ones(8).double(), inv_freq=f)
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="norm_eps"):
            K.norm_rotary_embed(q, norm_eps=eps, inv_freq=f)


def _select(**kw):
    a = _lib.BlockSelectArgs()
    a.q = a.k_scale = a.k_zero = a.out = 4096
    a.B, a.Hq, a.Hkv, a.Sq, a.D, a.n_packed, a.cap_tokens, a.n_tail = 2, 8, 2, 1, 128, 640, 1024, 9
    a.block_tokens, a.query_block, a.count, a.first, a.recent, a.group, a.levels = 64, 1, 4, 1, 1, 32, 15
    for name, v in kw.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(B=0), "bad sizes"), (dict(D=257), "bad sizes"), (dict(Hq=7), "multiple of H_kv"), (dict(dtype=_lib.VQ_U8), "q dtype"), (dict(meta_dtype=_lib.VQ_BF16), "scale and zero"),
    (dict(n_packed=-1), "token counts"), (dict(cap_tokens=639), "token counts"), (dict(group=0), "group size"), (dict(levels=0), "levels"), (dict(levels=256), "levels"),
    (dict(block_tokens=48), "no multiple"), (dict(block_tokens=0), "no multiple"), (dict(query_block=0), "query_block"), (dict(first=3, recent=2), "first"), (dict(count=0), "first"),
    (dict(recent=-1), "first"), (dict(n_tail=1 << 30), "2.30"), (dict(B=1 << 23), "query rows"), (dict(q=None), "null"), (dict(k_zero=None), "null"), (dict(out=None), "null"),
    (dict(causal=1, Sq=650), "exceeds")])
def test_select_refuses(kw, what):
    lib = _lib.load()
    assert lib.vq_block_select(_select(**kw)) in REFUSED
    assert re.search(what, _lib.last_error()), _lib.last_error()
    assert lib.vq_block_select_workspace(_select(**kw)) == 0
    assert lib.vq_block_select(None) == _lib.VQ_ERR_INVALID


def test_select_asks_for_a_workspace():
    lib = _lib.load()
    need = lib.vq_block_select_workspace(_select())
    assert need > 0
    assert lib.vq_block_select(_select()) == _lib.VQ_ERR_WORKSPACE
    assert lib.vq_block_select(_select(workspace=4096, workspace_bytes=need - 1)) == _lib.VQ_ERR_WORKSPACE
    assert lib.vq_block_select(_select(workspace=4097, workspace_bytes=need)) == _lib.VQ_ERR_WORKSPACE
    assert lib.vq_block_select_workspace(_select(count=10)) == 0      # every block is chosen
    assert lib.vq_block_select_workspace(_select(n_packed=0)) == 0


def test_select_blocks_refuses():
    q, z = torch.zeros(1, 4, 1, 64), torch.zeros(1, 2, 8, 64)
    kw = dict(levels=15, group_size=32, n_packed=256)
    with pytest.raises(RuntimeError, match="select_blocks: .*no CPU path"):
        K.select_blocks(q, z, z, 2, **kw)
    with pytest.raises(ValueError, match="select_blocks: q must be"):
        K.select_blocks(q[0], z, z, 2, **kw)
    with pytest.raises(ValueError, match="select_blocks: q must be"):
        K.select_blocks(q, z[0], z, 2, **kw)


def _attend(**kw):
    a = _lib.BlockAttendArgs()
    s = a.store
    s.q = s.out = 4096
    s.B, s.Hq, s.Hkv, s.Sq, s.D, s.scale = 2, 8, 2, 1, 128, 0.1
    for n in ("k_packed", "k_scale", "k_zero", "v_packed", "v_scale", "v_zero", "k_tail", "v_tail"):
        setattr(s.own, n, 4096)
    s.own.n_packed, s.own.cap_tokens, s.own.n_tail, s.pack_bits, s.group, s.v_layout = 640, 1024, 9, 4, 32, _lib.VQ_V_TOKEN_PACKED
    a.blocks, a.count, a.block_tokens, a.query_block = 4096, 4, 64, 1
    for name, v in kw.items():
        obj, _, field = name.rpartition("__")
        if field in ("blocks", "count", "block_tokens", "query_block"):
            setattr(a, field, v)
        else:
            setattr(getattr(s, obj) if obj else s, field, v)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(B=0), "bad sizes"), (dict(Hq=7), "multiple of H_kv"), (dict(D=300), "must be <= 256"), (dict(dtype=_lib.VQ_U8), "q/out dtype"), (dict(own__k_tail=None), "null tail pointer"),
    (dict(own__k_zero=None), "null packed pointer"), (dict(own__cap_tokens=639), "exceeds cap"), (dict(sliding_window=5), "no sliding window"), (dict(causal=1, Sq=650), "exceeds"),
    (dict(prefix__n_tail=3, prefix__k_tail=4096, prefix__v_tail=4096), "no shared prefix"), (dict(block_tokens=0), "block size"), (dict(query_block=0), "query_block"),
    (dict(count=-1), "list length"), (dict(blocks=None), "null blocks"), (dict(pack_bits=9), "pack_bits"), (dict(B=1 << 25), "query rows")])
def test_attend_refuses(kw, what):
    lib = _lib.load()
    assert lib.vq_block_attend(_attend(**kw)) in REFUSED
    assert what in _lib.last_error(), _lib.last_error()
    assert lib.vq_block_attend_workspace(_attend(**kw)) == 0
    assert lib.vq_block_attend(None) == _lib.VQ_ERR_INVALID


def test_block_sparse_attend_refuses():
    q, t = torch.zeros(1, 4, 1, 64), torch.zeros(1, 2, 8, 64)
    blocks = torch.zeros(1, 2, 1, 3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="block_sparse_attend: .*no CPU path"):
        K.block_sparse_attend(q, blocks, block_size=32, k_tail=t, v_tail=t, n_tail=8)
    with pytest.raises(ValueError, match="block_sparse_attend: q must be 4D"):
        K.block_sparse_attend(q[0], blocks, block_size=32, k_tail=t, v_tail=t, n_tail=8)


def test_caches_that_cannot_choose():
    base = dict(method="kivi", bit_width_inlier=4, kivi_group_size=32, residual_length=32)
    q = torch.zeros(1, 4, 1, 128)
    plain = KVCacheFactory.create(KVCacheConfig(head_dim=128, **base))
    for call in (lambda c: c.fused_sparse_sdpa(q, 0.1, 4), lambda c: c.select_blocks(q, 4)):
        with pytest.raises(RuntimeError, match="was not enabled"):
            call(plain)
        empty = KVCacheFactory.create(KVCacheConfig(head_dim=128, fused_sdpa=True, **base))
        with pytest.raises(RuntimeError, match="before any tokens"):
            call(empty)


def test_sizes_past_one_call_are_refused():
    """The limits that the documentation names; each refusal comes ahead of any launch."""
    lib = _lib.load()
    many = dict(B=1, Hq=8, Hkv=8, n_packed=32768, cap_tokens=32768, block_tokens=32)
    assert lib.vq_block_select(_select(**many, Sq=8192)) == _lib.VQ_ERR_UNSUPPORTED and "scores" in _lib.last_error()
    assert lib.vq_block_select_workspace(_select(**many, Sq=8191)) > 0 and lib.vq_block_select_workspace(_select(**many, Sq=8192, query_block=2)) > 0
    assert lib.vq_block_select(_select(B=1, Hq=1, Hkv=1, Sq=1 << 23, n_packed=32)) == _lib.VQ_ERR_UNSUPPORTED and "scores" in _lib.last_error()
    assert lib.vq_block_select(_select(B=1, Hq=2, Hkv=1, Sq=1 << 23, n_packed=32)) == _lib.VQ_ERR_UNSUPPORTED and "query rows" in _lib.last_error()
    assert lib.vq_norm_rotary(_norm(D=7, dims=6, S=1 << 25), None) == _lib.VQ_ERR_UNSUPPORTED and "rows" in _lib.last_error()      # two heads
