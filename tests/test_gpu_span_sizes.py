"""Sizes of attention over spans that other tests leave out."""

import pytest
import torch

from tests._gpu import gpu, require_gpu
from tests.test_gpu_shared_prefix import _case

pytestmark = gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [1, 3, 81, 129, 255])
@pytest.mark.parametrize("B,Hq,Hkv,n,own,Sq", [(1, 1, 1, 5, 12, 1), (3, 3, 1, 0, 40, 1), (1, 5, 5, 300, 7, 3), (1, 1, 1, 3000, 1, 1)])
def test_odd_heads(dtype, D, B, Hq, Hkv, n, own, Sq):
    """Odd numbers of records of odd size, in one part and in many."""
    require_gpu()
    _case(B, Hq, Hkv, D, (0, n), (0, own), Sq, dtype=dtype, seed=D)


@pytest.mark.parametrize("bits,v_layout", [(4, "channel"), (3, "channel"), (2, "token")])
def test_odd_heads_over_packed_slots(bits, v_layout):
    require_gpu()
    _case(3, 3, 1, 81, (96, 5), (32, 6), 1, bits=bits, v_layout=v_layout)
