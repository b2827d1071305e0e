"""Scales of any sign and size, for every kernel of attention over spans."""

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests._spans import attend, close, seen, store
from tests.test_gpu_differential import reference
from veloxquant_mlx_amd import kernels as K

pytestmark = gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("scale", [-0.1, 0.0, 2.0, 1e-30])
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("kw", [
    dict(B=3, D=128, n=(256, 9), own=(0, 33)), dict(B=48, D=128, n=(1024, 9), own=(128, 33)), dict(B=2, D=256, n=(512, 9), own=(64, 33), bits=2),
    dict(B=2, D=64, n=(0, 100), own=(0, 233), Sq=150, dtype=BF16), dict(B=2, D=128, n=(256, 9), own=(256, 33), Sq=90), dict(B=2, D=80, n=(0, 30), own=(0, 33), Sq=3, dtype=F32)])
def test_scales(kw, maps, scale):
    """A row of equal scores (scale zero) is the mean; a negative scale turns the order round."""
    require_gpu()
    kw = dict(dict(Sq=1, bits=4, dtype=F16), **kw)
    B, D, Sq, dtype, Hq, H = kw["B"], kw["D"], kw["Sq"], kw["dtype"], 8, 2
    opts = dict(bits=kw["bits"], dtype=dtype, spare=8)
    o, ok, ov = store(B, H, *kw["own"], D, seed=2, **opts)
    q = torch.randn((B, Hq, Sq, D), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(dtype)
    u = 0.0 if dtype == F32 else torch.finfo(F16 if kw["own"][0] + kw["n"][0] * (maps == 1) else dtype).eps / 2
    if maps == 1:
        p, pk, pv = store(1, H, *kw["n"], D, seed=1, **opts)
        k, v = torch.cat([pk.expand(B, -1, -1, -1), ok], 2), torch.cat([pv.expand(B, -1, -1, -1), ov], 2)
        got = K.shared_prefix_attend(q, p, **o, scale=scale, causal=False)
        want, far = attend(q, k, v, seen(B, Sq, 0, k.shape[2], None, False, 0), scale, u)
    else:
        got = K.differential_attend(q, -0.3, **o, scale=scale, causal=False)
        want, far = reference(q, ok, ov, -0.3, seen(B, Sq, 0, ok.shape[2], None, False, 0), scale, u)
    close(got, want, far)
