"""Frequencies of rotary positions and the refusals of ``rotary_embed`` (no GPU)."""

import math

import pytest
import torch

from veloxquant_mlx_amd import _lib, kernels as K
from veloxquant_mlx_amd.rotary import RotaryPositions, rotary_frequencies


def test_unscaled_frequencies():
    f, factor = rotary_frequencies(8, 10000.0)
    assert factor == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15, atol=0)
    assert torch.equal(rotary_frequencies(8, 10000.0, {"rope_type": "default"})[0], f)


def test_linear_and_ntk():
    f, _ = rotary_frequencies(64, 10000.0)
    assert torch.equal(rotary_frequencies(64, 10000.0, {"type": "linear", "factor": 4})[0], f / 4)
    g, factor = rotary_frequencies(64, 10000.0, {"rope_type": "ntk", "factor": 4})
    # the slowest pair is slowed by the factor, the fastest not at all
    assert factor == 1.0 and math.isclose(float(g[-1]), float(f[-1]) / 4, rel_tol=1e-12) and float(g[0]) == 1.0


@pytest.mark.parametrize("name", ["by_parts", "llama3"])
def test_by_parts(name):
    L, factor, lo, hi = 8192, 8.0, 1.0, 4.0
    f, _ = rotary_frequencies(128, 500000.0)
    g, att = rotary_frequencies(128, 500000.0, {"rope_type": name, "factor": factor, "low_freq_factor": lo, "high_freq_factor": hi,
                                                "original_max_position_embeddings": L})
    assert att == 1.0
    kinds = set()
    for w, x in zip(f.tolist(), g.tolist()):
        wavelength = 2 * math.pi / w
        if wavelength < L / hi:
            want, kind = w, "kept"
        elif wavelength > L / lo:
            want, kind = w / factor, "slowed"
        else:
            s = (L / wavelength - lo) / (hi - lo)
            want, kind = (1 - s) * w / factor + s * w, "blended"
        kinds.add(kind)
        assert math.isclose(x, want, rel_tol=1e-12)
    assert kinds == {"kept", "slowed", "blended"}


def test_yarn():
    L, factor, base, dims = 4096, 16.0, 10000.0, 128
    f, _ = rotary_frequencies(dims, base)
    g, att = rotary_frequencies(dims, base, {"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": L})
    assert math.isclose(att, 0.1 * math.log(factor) + 1)
    lo = math.floor(dims * math.log(L / (32 * 2 * math.pi)) / (2 * math.log(base)))
    hi = math.ceil(dims * math.log(L / (1 * 2 * math.pi)) / (2 * math.log(base)))
    for i, (w, x) in enumerate(zip(f.tolist(), g.tolist())):
        r = min(max((i - lo) / (hi - lo), 0), 1)
        assert math.isclose(x, w * (1 - r) + w / factor * r, rel_tol=1e-12)
    assert rotary_frequencies(dims, base, {"type": "yarn", "factor": 2, "original_max_position_embeddings": L, "attention_factor": 1.5})[1] == 1.5


@pytest.mark.parametrize("dims,base,scaling", [
    (7, 10000.0, None), (0, 10000.0, None), (8, 1.0, None), (8, float("nan"), None), (8, 10000.0, {"rope_type": "other", "factor": 2}),
    (8, 10000.0, {"factor": 2}), (8, 10000.0, {"rope_type": "linear"}), (8, 10000.0, {"rope_type": "linear", "factor": 0.5}),
    (8, 10000.0, {"rope_type": "linear", "factor": 2, "low_freq_factor": 1}), (2, 10000.0, {"rope_type": "ntk", "factor": 2}),
    (8, 10000.0, {"rope_type": "linear", "type": "ntk", "factor": 2}),
    (8, 10000.0, {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": 4096, "beta_fast": 1, "beta_slow": 2}),
    (8, 10000.0, {"rope_type": "by_parts", "factor": 2, "low_freq_factor": 4, "high_freq_factor": 1, "original_max_position_embeddings": 8192})])
def test_frequencies_refuse(dims, base, scaling):
    with pytest.raises(ValueError, match="rotary_frequencies"):
        rotary_frequencies(dims, base, scaling)


def test_own_frequencies():
    r = RotaryPositions(8, inv_freq=torch.tensor([1.0, 0.5, 0.25, 0.1]), traditional=True, device="cpu")
    assert r.inv_freq.dtype == torch.float64 and r.attention_factor == 1.0 and r.traditional
    with pytest.raises(ValueError, match="inv_freq"):
        RotaryPositions(8, inv_freq=torch.ones(3), device="cpu")
    with pytest.raises(ValueError, match="inv_freq"):
        RotaryPositions(8, inv_freq=torch.ones(4), scaling={"type": "linear", "factor": 2}, device="cpu")


def test_host_tensors_are_refused():
    q = torch.zeros(1, 2, 3, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        K.rotary_embed(q, inv_freq=torch.ones(4))
    with pytest.raises(ValueError, match=r"must be \[B, H, S, D\]"):
        K.rotary_embed(q[0], inv_freq=torch.ones(4))
    with pytest.raises(ValueError, match="k_out without k"):
        K.rotary_embed(q, inv_freq=torch.ones(4), k_out=q)


def _args(**kw):
    a = _lib.RotaryArgs()
    a.B, a.S, a.D, a.dims, a.inv_freq, a.freq_dtype, a.attention_factor = 1, 4, 8, 8, 4096, _lib.VQ_F64, 1.0
    a.x[0], a.out[0], a.heads[0] = 4096, 8192, 2
    for name, v in kw.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(dtype=_lib.VQ_U8), "dtype"), (dict(dims=7), "dims"), (dict(dims=0), "dims"), (dict(dims=10), "dims"), (dict(layout=2), "layout"),
    (dict(freq_dtype=_lib.VQ_F16), "frequencies"), (dict(positions=4096, pos_dtype=_lib.VQ_F32), "positions"), (dict(inv_freq=None), "frequencies"),
    (dict(B=-1), "sizes"), (dict(S=1 << 31), "positions a sequence"), (dict(B=1 << 30, S=1 << 10), "too many rows")])
def test_entry_point_refuses(kw, what):
    lib = _lib.load()
    assert lib.vq_rotary(_args(**kw), None) in (_lib.VQ_ERR_INVALID, _lib.VQ_ERR_UNSUPPORTED)
    assert what in _lib.last_error()


def test_entry_point_checks_rows():
    lib = _lib.load()
    a = _args()
    a.out[0] = None
    assert lib.vq_rotary(a, None) == _lib.VQ_ERR_INVALID and "outputs must be given" in _lib.last_error()
    a = _args()
    a.out[0] = a.x[0]
    a.x_strides[0][2], a.out_strides[0][2] = 8, 16
    assert lib.vq_rotary(a, None) == _lib.VQ_ERR_INVALID and "in place" in _lib.last_error()
    assert lib.vq_rotary(None, None) == _lib.VQ_ERR_INVALID
    for empty in (dict(B=0), dict(S=0)):
        assert lib.vq_rotary(_args(**empty), None) == 0


@pytest.mark.parametrize("struct,mirror", [("vq_rotary_args", _lib.RotaryArgs), ("vq_kv_store", _lib.KVStore), ("vq_store_attend_args", _lib.StoreAttendArgs)])
def test_structures_match_the_header(struct, mirror):
    import os
    import re
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
