"""Refusals of the shared-prefix and differential attention entry points (no GPU)."""

import pytest
import torch

from veloxquant_mlx_amd import _lib, kernels as K


def _args(**kw):
    a = _lib.StoreAttendArgs()
    a.q = a.out = 4096
    a.B, a.Hq, a.Hkv, a.Sq, a.D, a.scale = 2, 8, 2, 1, 128, 0.1
    a.own.k_tail = a.own.v_tail = 4096
    a.own.n_tail = 300
    a.lam = 4096
    for name, v in kw.items():
        obj, _, field = name.rpartition("__")
        setattr(getattr(a, obj) if obj else a, field, v)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(B=0), "bad sizes"), (dict(Hq=7), "multiple of H_kv"), (dict(D=300), "must be <= 256"), (dict(dtype=_lib.VQ_U8), "q/out dtype"),
    (dict(own__n_tail=0), "no key/value slots"), (dict(own__n_tail=-1), "negative token count"), (dict(own__k_tail=None), "null tail pointer"),
    (dict(tail_dtype=_lib.VQ_I32), "tail dtype"), (dict(own__n_packed=64), "null packed pointer"), (dict(sliding_window=-1), "sliding window"),
    (dict(causal=1, Sq=301), "exceeds"), (dict(q=None), "null q"), (dict(own__n_tail=1 << 30), "2.30 slots"), (dict(B=1 << 25), "query rows")])
@pytest.mark.parametrize("call", ["vq_shared_prefix_attend", "vq_differential_attend"])
def test_refused(call, kw, what):
    lib = _lib.load()
    assert getattr(lib, call)(_args(**kw)) in (_lib.VQ_ERR_INVALID, _lib.VQ_ERR_UNSUPPORTED)
    msg = _lib.last_error()
    import re
    assert re.search(what, msg), msg
    assert getattr(lib, call + "_workspace")(_args(**kw)) == 0
    assert getattr(lib, call)(None) == _lib.VQ_ERR_INVALID


@pytest.mark.parametrize("kw,what", [
    (dict(pack_bits=9), "pack_bits"), (dict(pack_bits=4, group=0), "group_size"), (dict(pack_bits=4, group=32, meta_dtype=_lib.VQ_BF16), "meta"),
    (dict(pack_bits=4, group=32, meta_dtype=_lib.VQ_F16, v_layout=5), "v_layout"),
    (dict(pack_bits=4, group=32, meta_dtype=_lib.VQ_F16, own__cap_tokens=32), "exceeds cap"),
    (dict(pack_bits=4, group=32, meta_dtype=_lib.VQ_F16, v_layout=1, own__cap_tokens=70), "word aligned")])
def test_packed_stores_refused(kw, what):
    lib = _lib.load()
    packed = {f"own__{n}": 4096 for n in ("k_packed", "k_scale", "k_zero", "v_packed", "v_scale", "v_zero")}
    a = _args(**{**packed, "own__n_packed": 64, "own__cap_tokens": 64, **kw})
    assert lib.vq_shared_prefix_attend(a) == _lib.VQ_ERR_INVALID and what in _lib.last_error()


def test_differential_refusals():
    lib = _lib.load()
    for kw, what in [(dict(lam=None), "lam"), (dict(lam_stride=2), "lam"), (dict(norm_weight=4096, norm_dtype=_lib.VQ_I32), "norm weight"),
                     (dict(D=65), "even"), (dict(prefix__n_tail=3, prefix__k_tail=4096, prefix__v_tail=4096), "no shared prefix")]:
        assert lib.vq_differential_attend(_args(**kw)) == _lib.VQ_ERR_INVALID and what in _lib.last_error()


@pytest.mark.parametrize("call,maps", [("vq_shared_prefix_attend", 1), ("vq_differential_attend", 2)])
@pytest.mark.parametrize("dtype,D", [(_lib.VQ_F32, 128), (_lib.VQ_F16, 128), (_lib.VQ_BF16, 256), (_lib.VQ_F16, 80)])
def test_workspace_is_asked_for(call, maps, dtype, D):
    lib = _lib.load()
    a = _args(dtype=dtype, tail_dtype=dtype, D=D, own__n_tail=5000)
    for f in ("k_strides", "v_strides"):
        for i, st in enumerate((2 * 5000 * D, 5000 * D, D)):
            getattr(a.own, f)[i] = st
    need = getattr(lib, call + "_workspace")(a)
    assert need > 0 and need % (2 * 8 * maps * (D + 2) * 4) == 0
    for ws, size in ((None, 0), (4096, need - 1), (4100, need)):
        a.workspace, a.workspace_bytes = ws, size
        assert getattr(lib, call)(a) == _lib.VQ_ERR_WORKSPACE and str(need) in _lib.last_error()


def test_host_tensors_are_refused():
    q = torch.zeros((1, 2, 1, 64))
    for call in (lambda: K.shared_prefix_attend(q, {}, k_tail=q, v_tail=q, n_tail=1), lambda: K.differential_attend(q, 0.5, k_tail=q, v_tail=q, n_tail=1)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def _cache(**kw):
    from veloxquant_mlx_amd.cache import KVCacheConfig, KVCacheFactory
    return KVCacheFactory.create(KVCacheConfig(**{**dict(method="kivi", head_dim=128, bit_width_inlier=4, fused_sdpa=True), **kw}))


def test_caches_that_cannot_be_shared():
    for kw, what in ((dict(fused_sdpa_memory_bound=True), "batch of one"), (dict(), "memory_bound"), (dict(fused_sdpa=False), "memory_bound"),
                     (dict(method="kivi_sink", fused_sdpa_memory_bound=True), "must be a KIVIKVCache")):
        with pytest.raises(ValueError, match=what):
            _cache(**kw).share()


def test_differential_attention_needs_a_packed_cache_with_tokens():
    q = torch.zeros((1, 4, 1, 128), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="not enabled"):
        _cache(fused_sdpa=False).fused_differential_sdpa(q, 0.1, 0.1)
    with pytest.raises(RuntimeError, match="before any tokens"):
        _cache().fused_differential_sdpa(q, 0.1, 0.1)
