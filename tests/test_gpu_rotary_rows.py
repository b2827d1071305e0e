"""``rotary_embed`` into rows that lie between others: the same bits as into new tensors, and nothing else written."""

import pytest
import torch

from tests._gpu import gpu, require_gpu
from veloxquant_mlx_amd.rotary import RotaryPositions

pytestmark = gpu


@pytest.mark.parametrize("traditional,D,dims", [(False, 128, 128), (True, 64, 32), (False, 20, 12)])
@pytest.mark.parametrize("B,S", [(1, 1), (2, 1), (2, 19)])
@pytest.mark.parametrize("place", ["q and cache", "q", "k", "q and v", "dense and k"])
def test_one_side_in_place(traditional, D, dims, B, S, place):
    require_gpu()
    Hq, Hk = 8, 2
    rows = torch.randn((B, S, (Hq + 2 * Hk) * D), generator=torch.Generator(device="cuda").manual_seed(D), device="cuda").half()
    part = lambda r, lo, H: r[..., lo * D:(lo + H) * D].view(B, S, H, D).transpose(1, 2)
    rope = RotaryPositions(dims, traditional=traditional)
    before = rows.clone()
    q, k, v = (part(rows, *x) for x in ((0, Hq), (Hq, Hk), (Hq + Hk, Hk)))
    want = rope(q, k, offset=5)
    buf = torch.full((B, Hk, 64, D), 7.0, device="cuda", dtype=torch.float16)
    out, k_out = {"q and cache": (q, buf[:, :, 11:11 + S]), "q": (q, None), "k": (None, k), "q and v": (q, v),
                  "dense and k": (torch.empty_like(want[0]), k)}[place]
    got = rope(q, k, offset=5, out=out, k_out=k_out)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for lo, H, o, w in ((0, Hq, out is q, want[0]), (Hq, Hk, k_out is k, want[1]), (Hq + Hk, Hk, k_out is v, want[1])):
        assert torch.equal(part(rows, lo, H), w if o else part(before, lo, H))
    if place == "q and cache":
        buf[:, :, 11:11 + S] = 7
    assert bool((buf == 7).all())
