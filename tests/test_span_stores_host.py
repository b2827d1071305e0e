"""Stores that the attention calls over spans refuse before anything reaches the library (no GPU)."""

import pytest
import torch

from veloxquant_mlx_amd import kernels as K


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(K, "_need_gpu", lambda *a: None)


@pytest.mark.parametrize("q_heads", [0, 2])
def test_a_store_without_heads(host, q_heads):
    q, none, some = (torch.zeros((2, h, n, 64), dtype=torch.float16) for h, n in ((q_heads, 1), (0, 5), (2, 5)))
    own = dict(k_tail=none, v_tail=none, n_tail=5)
    for call in (lambda: K.shared_prefix_attend(q, None, **own), lambda: K.differential_attend(q, 0.3, **own),
                 lambda: K.shared_prefix_attend(q, dict(k_tail=none[:1], v_tail=none[:1], n_tail=5)),
                 lambda: K.shared_prefix_attend(q, dict(k_tail=none[:1], v_tail=none[:1], n_tail=5), **own)):
        with pytest.raises(ValueError, match="over 0 kv heads of 64 channels"):
            call()
    for prefix, mine in ((some[:1], none), (none[:1], some)):
        with pytest.raises(ValueError, match="differ in kv heads"):
            K.shared_prefix_attend(q, dict(k_tail=prefix, v_tail=prefix, n_tail=5), k_tail=mine, v_tail=mine, n_tail=5)


def test_heads_without_channels(host):
    q, k = torch.zeros((2, 2, 1, 64), dtype=torch.float16), torch.zeros((2, 2, 5, 0), dtype=torch.float16)
    with pytest.raises(ValueError, match="over 2 kv heads of 0 channels"):
        K.differential_attend(q, 0.3, k_tail=k, v_tail=k, n_tail=5)
