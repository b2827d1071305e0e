"""KIVI cache of a batch of sequences behind a prefix that they share.

Many sequences that start with the same tokens (a system prompt, a document asked about more than once, samples of one prompt) hold
those tokens once: the prefix, packed, for a batch of one, and behind it every sequence's own tokens in a memory-bound
:class:`KIVIKVCache`.  Attention of few tokens a sequence reads the prefix for all of them together
(:func:`veloxquant_mlx_amd.kernels.shared_prefix_attend`, which names the stores it does so for; longer chunks read it a sequence)::

    cache.update_and_fetch(k, v)           # the prompt, a batch of one
    shared = cache.share()
    shared.update_and_fetch(k, v)          # [B, H, S, D]: the next tokens of B sequences
    out = shared.fused_sdpa(q, scale)

Positions go on behind the prefix: ``offset`` counts its tokens.
"""

from __future__ import annotations

import torch

from .. import kernels as K
from .kivi_cache import KIVIKVCache, batch_lengths, own_half_of_paired_output, pad_queries_for_paired_heads


class SharedPrefixKIVICache:
    """``[prefix | own tokens]`` of every sequence of a batch; :meth:`KIVIKVCache.share` makes one.

    The prefix is a copy of the cache's tokens at that time and does not change any more; several objects may stand on one
    (:meth:`branch`).  A cache of its own in every other respect: ``update_and_fetch``, ``fused_sdpa``, ``trim`` (of the own tokens),
    ``offset``, ``nbytes``; but no ``state``: a prompt-cache file holds the cache that was shared.  ``fused_sdpa_max_ctx`` bounds
    prefix and own tokens together (the own packed store is sized by what the prefix leaves)."""

    _memory_bound = True   # attention goes through fused_sdpa; update_and_fetch returns placeholders

    def __init__(self, cache: KIVIKVCache) -> None:
        if type(cache) is not KIVIKVCache or not cache._memory_bound:
            raise ValueError("SharedPrefixKIVICache: the prefix must be a KIVIKVCache with fused_sdpa_memory_bound=True")
        if cache.offset == 0 or cache._shape_bhd[0] != 1:
            raise ValueError(f"SharedPrefixKIVICache: the prefix must hold tokens of a batch of one, got {cache.offset} tokens of a batch "
                             f"of {cache._shape_bhd[0]}")
        prefix = KIVIKVCache(cache._config)
        prefix._max_ctx = None   # (no room for more tokens)
        prefix.state = cache.state
        prefix._kv_heads = cache._kv_heads
        self._join(prefix)

    def _join(self, prefix: KIVIKVCache) -> None:
        self._prefix = prefix
        self._prefix_args = prefix._store_args()
        self._kv_heads = abs(prefix._kv_heads) if prefix._pair else prefix._shape_bhd[1]
        self._head_dim = prefix._shape_bhd[2] // (2 if prefix._pair else 1)
        self._own = KIVIKVCache(prefix._config)
        self._own._launch_stores = False   # (no launch of this cache stores a token that was held back)
        if self._own._max_ctx is not None:   # of the whole context
            self._own._max_ctx = max(0, self._own._max_ctx - prefix.offset)

    def branch(self) -> "SharedPrefixKIVICache":
        """Another batch on the same prefix, without tokens of its own yet."""
        other = object.__new__(SharedPrefixKIVICache)
        other._join(self._prefix)
        return other

    @property
    def prefix_length(self) -> int:
        return self._prefix.offset

    @property
    def offset(self) -> int:
        """Tokens of a sequence, the prefix included: the position of the next one."""
        return self._prefix.offset + self._own.offset

    def size(self) -> int:
        return self.offset

    def empty(self) -> bool:
        return False

    def _heads_under(self, heads: int) -> int:
        """The kv head count under ``heads`` of keys or queries.  A prefix restored without its ``meta_state`` shows pairs of heads, not whether
        the last one is whole: one head less where the heads do not divide over an even count, as in :class:`KIVIKVCache`."""
        H = self._kv_heads
        return H - 1 if self._prefix._kv_heads < 0 and H % 2 == 0 and H > 2 and heads % H and heads % (H - 1) == 0 else H

    def update_and_fetch(self, keys: torch.Tensor, values: torch.Tensor):
        """Append ``[B,H,S,D]`` keys and values to the sequences' own tokens, quantised as they age as in any
        :class:`KIVIKVCache`; returns zero-stride placeholders of the whole length."""
        dtype = self._prefix._tail_k.dtype if self._prefix_args["n_tail"] else keys.dtype
        if keys.ndim == 4 and self._own.offset == 0 and keys.shape[1] == self._heads_under(keys.shape[1]):
            self._kv_heads = keys.shape[1]
        if (keys.ndim != 4 or keys.shape[1] != self._kv_heads or keys.shape[3] != self._head_dim or values.shape != keys.shape
                or keys.dtype != dtype or values.dtype != dtype):
            raise ValueError(f"SharedPrefixKIVICache.update_and_fetch: keys and values must be [B, {self._kv_heads}, S, {self._head_dim}] {dtype} "
                             f"as the prefix is, got {tuple(keys.shape)} {keys.dtype} and {tuple(values.shape)} {values.dtype}")
        if self._own.offset and keys.shape[0] != self._own._shape_bhd[0]:
            raise ValueError(f"SharedPrefixKIVICache.update_and_fetch: {keys.shape[0]} sequences, this cache holds {self._own._shape_bhd[0]}")
        self._own.update_and_fetch(keys, values)
        z = self._own._zero_scalar.expand(keys.shape[0], self._kv_heads, self.offset, self._head_dim)
        return z, z

    def fused_sdpa(self, q: torch.Tensor, scale: float, *, causal: bool = True, sliding_window: int = 0,
                   lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of ``q [B,H_q,S_q,D]`` over prefix and own tokens, queries aligned to the end, under the masks of
        :meth:`KIVIKVCache.fused_sdpa`.  ``lengths`` (int ``[B]``, on the device or the host) gives every sequence of a right-padded
        batch its number of live tokens, the prefix included (and so no fewer than those).  The same bits from run to run."""
        name = "SharedPrefixKIVICache.fused_sdpa"
        if lengths is not None:
            if not (isinstance(lengths, torch.Tensor) and lengths.is_cuda) and min(torch.as_tensor(lengths).reshape(-1).tolist(), default=0) < self.prefix_length:
                raise ValueError(f"{name}: lengths count the prefix of {self.prefix_length} tokens")
            lengths = batch_lengths(name, lengths, q) - self.prefix_length
        pair, H = self._prefix._pair, self._kv_heads
        if pair:
            if q.ndim == 4 and self._own.offset == 0:
                H = self._heads_under(q.shape[1])
            if q.ndim != 4 or q.shape[3] != self._head_dim or q.shape[1] % H:
                raise ValueError(f"{name}: q {tuple(q.shape)} over {H} kv heads of {self._head_dim} channels")
            q = pad_queries_for_paired_heads(q, H)
        own = self._own._store_args() if self._own.offset else {}
        out = K.shared_prefix_attend(q, self._prefix_args, **own, scale=float(scale), causal=bool(causal), seq_lens=lengths,
                                     sliding_window=int(sliding_window or 0))
        return own_half_of_paired_output(out, H) if pair else out

    def is_trimmable(self) -> bool:
        return True

    def trim(self, n: int) -> int:
        """Drop the last ``n`` own tokens of every sequence; the prefix stays."""
        return self._own.trim(n)

    @property
    def nbytes(self) -> int:
        """Bytes of the own tokens and, once, of the prefix."""
        return self._prefix.nbytes + self._own.nbytes


__all__ = ["SharedPrefixKIVICache"]
