"""Scratch of attention over spans (no GPU)."""

import pytest

from tests.test_span_host import _args
from veloxquant_mlx_amd import _lib


@pytest.mark.parametrize("call,maps", [("vq_shared_prefix_attend", 1), ("vq_differential_attend", 2)])
@pytest.mark.parametrize("D,B,Hq", [(81, 1, 1), (81, 3, 1), (255, 1, 7), (1, 1, 1), (2, 1, 1), (66, 1, 3), (80, 1, 1)])
def test_the_pairs_behind_the_sums_are_aligned(call, maps, D, B, Hq):
    """A record is D floats of sums and a pair behind all sums, which is read as eight bytes: the sums take whole 16 bytes."""
    if maps == 2 and D % 2:
        pytest.skip("two halves")
    a = _args(B=B, Hq=Hq, Hkv=1, D=D, own__n_tail=40)      # one part a row
    records = B * Hq * maps
    need = getattr(_lib.load(), call + "_workspace")(a)
    assert (need - 8 * records) % 16 == 0 and need >= records * (D + 2) * 4
