"""Rotary positions of a model's queries and keys, in front of a cache's ``update_and_fetch``.

:class:`RotaryPositions` keeps what a model keeps (the frequencies on the GPU, the layout of the pairs, the factor of a
scaled context) and turns queries and keys in one launch (:func:`veloxquant_mlx_amd.kernels.rotary_embed`)::

    rope = RotaryPositions(128, base=500000.0)
    q, k = rope(q, k, offset=cache.offset)
    cache.update_and_fetch(k, v)
    out = cache.fused_sdpa(q, scale)

Models that norm queries and keys a head do both in one launch: ``rope.normed(q, k, q_weight=.., k_weight=.., offset=..)``.
"""

from __future__ import annotations

import math

import torch

from . import kernels as K

_SCALINGS = {
    "linear": {"factor"},
    "ntk": {"factor"},
    "by_parts": {"factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"},
    "yarn": {"factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "attention_factor"},
}
_SCALINGS["llama3"] = _SCALINGS["by_parts"]   # the name model configurations give it
_DEFAULTS = {"beta_fast": 32.0, "beta_slow": 1.0, "attention_factor": None}


def rotary_frequencies(dims: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """Angular frequencies ``[dims / 2]`` (float64, on the host) and the factor on the turned rows.

    Unscaled: ``w_i = base^(-2i / dims)``, factor 1.  ``scaling``: a dict whose ``"rope_type"`` (or ``"type"``) is

    * ``"linear"``    positions divided by ``factor``
    * ``"ntk"``       ``base`` times ``factor^(dims / (dims - 2))``: the slowest pair is slowed by ``factor``, the fastest not at all
    * ``"by_parts"`` (``"llama3"``)  with ``L = original_max_position_embeddings``: pairs that turn fewer than ``low_freq_factor`` times over ``L``
      positions are slowed by ``factor``, those that turn more than ``high_freq_factor`` times are kept, in between blended
    * ``"yarn"``      the same with a ramp over the pair index, between the pairs that turn ``beta_fast`` (32) and ``beta_slow`` (1)
      times over ``L`` positions; rows are scaled by ``attention_factor`` (``0.1 ln(factor) + 1``)

    and ``"default"`` (or None) for none.  Other keys are refused."""
    if dims < 2 or dims % 2:
        raise ValueError(f"rotary_frequencies: dims={dims} must be even and at least 2")
    if not base > 1:
        raise ValueError(f"rotary_frequencies: base={base} must be above 1")
    i = torch.arange(0, dims, 2, dtype=torch.float64)
    freq = float(base) ** (-i / dims)
    given = dict(scaling or {})
    kinds = {given.pop(key) for key in ("rope_type", "type") if key in given}
    kind = kinds.pop() if kinds else "default"
    if kinds:
        raise ValueError("rotary_frequencies: rope_type and type differ")
    if kind == "default" and not given:
        return freq, 1.0
    if kind not in _SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling {kind!r} is not one of default, {', '.join(sorted(_SCALINGS))}")
    wanted = _SCALINGS[kind]
    if set(given) - wanted or wanted - set(given) - set(_DEFAULTS):
        raise ValueError(f"rotary_frequencies: {kind!r} takes {sorted(wanted)}, got {sorted(given)}")
    given = {key: _DEFAULTS[key] for key in wanted if key in _DEFAULTS} | given
    factor = float(given["factor"])
    if not factor >= 1:
        raise ValueError(f"rotary_frequencies: factor={factor} must be at least 1")
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "ntk":
        if dims == 2:
            raise ValueError("rotary_frequencies: 'ntk' needs at least two pairs")
        return (float(base) * factor ** (dims / (dims - 2))) ** (-i / dims), 1.0
    length = float(given["original_max_position_embeddings"])
    if not length > 0:
        raise ValueError("rotary_frequencies: original_max_position_embeddings must be positive")
    if kind == "yarn":
        fast, slow = float(given["beta_fast"]), float(given["beta_slow"])
        if not fast > slow > 0:
            raise ValueError("rotary_frequencies: beta_fast must be above beta_slow, both positive")
        # the (fractional) pair index that turns `n` times over `length` positions
        pair = lambda n: dims * math.log(length / (n * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dims - 1)
        slowed = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        att = given["attention_factor"]
        return freq * (1 - slowed) + freq / factor * slowed, 0.1 * math.log(factor) + 1.0 if att is None else float(att)
    lo, hi = float(given["low_freq_factor"]), float(given["high_freq_factor"])
    if not hi > lo:
        raise ValueError("rotary_frequencies: high_freq_factor must be above low_freq_factor")
    kept = ((length * freq / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
    return freq * kept + freq / factor * (1 - kept), 1.0


class RotaryPositions:
    """Rotary positions over the first ``dims`` channels of a head: pairs ``(i, i + dims/2)``, with ``traditional``
    ``(2i, 2i + 1)``.  ``base`` and ``scaling`` as for :func:`rotary_frequencies`; ``inv_freq`` (``[dims / 2]``) in place of
    both for frequencies of a model's own."""

    def __init__(self, dims: int, *, base: float = 10000.0, traditional: bool = False, scaling: dict | None = None,
                 inv_freq: torch.Tensor | None = None, device="cuda:0") -> None:
        if inv_freq is None:
            inv_freq, self.attention_factor = rotary_frequencies(dims, base, scaling)
        else:
            if scaling is not None or tuple(inv_freq.shape) != (dims // 2,) or dims % 2:
                raise ValueError(f"RotaryPositions: inv_freq must be [{dims // 2}], without scaling, got {tuple(inv_freq.shape)}")
            self.attention_factor = 1.0
        self.dims, self.traditional = int(dims), bool(traditional)
        self.inv_freq = inv_freq.to(device=device, dtype=torch.float64)

    def __call__(self, q: torch.Tensor, k: torch.Tensor | None = None, *, offset: int | torch.Tensor = 0,
                 positions: torch.Tensor | None = None, inverse: bool = False, out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None):
        """``q'`` or ``(q', k')`` at positions ``offset + s`` or ``positions`` (:func:`~veloxquant_mlx_amd.kernels.rotary_embed`).
        ``inverse``: rows that this object turned come back (the factor is taken out again)."""
        factor = 1 / self.attention_factor if inverse else self.attention_factor
        return K.rotary_embed(q, k, inv_freq=self.inv_freq, offset=offset, positions=positions, traditional=self.traditional,
                              attention_factor=factor, inverse=inverse, out=out, k_out=k_out)

    def normed(self, q: torch.Tensor, k: torch.Tensor | None = None, *, q_weight: torch.Tensor | None = None,
               k_weight: torch.Tensor | None = None, norm_eps: float = 1e-6, offset: int | torch.Tensor = 0,
               positions: torch.Tensor | None = None, out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
        """The same behind the norm of every head's row, for models that norm queries and keys a head: one launch for both
        (:func:`~veloxquant_mlx_amd.kernels.norm_rotary_embed`)."""
        return K.norm_rotary_embed(q, k, q_weight=q_weight, k_weight=k_weight, norm_eps=norm_eps, inv_freq=self.inv_freq, offset=offset,
                                   positions=positions, traditional=self.traditional, attention_factor=self.attention_factor, out=out,
                                   k_out=k_out)


__all__ = ["RotaryPositions", "rotary_frequencies"]
