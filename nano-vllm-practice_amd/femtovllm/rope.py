"""Rotary-embedding tables.

``rope_tables`` for ``ops.qk_norm_rope_cache_write``, ``scaled_rope_tables``
for ``ops.rope_cache_write``.

``rope_tables`` are built as ``QwenRotaryEmbedding.__init__`` builds its ``cos`` / ``sin``
buffers (femtovllm/models/qwen/qwen3.py:22-52): ``inv_freq_i = (1/base) **
(2 i / d_head)`` for ``i < d_head/2`` in float32, ``theta = p * inv_freq``
for ``p < max_seqlen``, duplicated to ``d_head`` columns.  A model that
already holds the buffers passes them directly (as float32).
"""

import math

import torch


def rope_tables(max_seqlen: int, d_head: int, base: float = 1000000.0, device=None):
    """(cos, sin), each (max_seqlen, d_head) float32."""
    if d_head % 2 != 0:
        raise ValueError(f"d_head must be even, now {d_head=}")
    inv_freq = torch.arange(d_head // 2, device=device).float()
    inv_freq = (1.0 / base) ** (2 * inv_freq / d_head)
    theta = torch.arange(max_seqlen, device=device).float()[:, None] * inv_freq[None, :]
    theta = torch.cat((theta, theta), dim=-1)
    return torch.cos(theta), torch.sin(theta)


def scaled_rope_tables(
    max_seqlen: int,
    rotary_dim: int,
    base: float = 10000.0,
    scaling: str = "none",
    factor: float = 1.0,
    original_max_seqlen: int = 0,
    low_freq_factor: float = 1.0,
    high_freq_factor: float = 4.0,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    attention_factor: float = None,
    device=None,
):
    """(cos, sin), each (max_seqlen, rotary_dim / 2) float32: pair i turns by ``p * w_i`` at position p.

    ``w_i = base ** (-2 i / rotary_dim)``, changed for contexts ``factor`` times
    those of ``original_max_seqlen`` by ``scaling``:

    * ``"none"``;
    * ``"linear"``: ``w_i / factor`` (interpolated positions);
    * ``"ntk"``: the base times ``factor ** (rotary_dim / (rotary_dim - 2))``, so
      that the slowest pair turns ``factor`` times slower and the fastest as before;
    * ``"wavelength"``: pairs of a wavelength ``2 pi / w_i`` up to
      ``original_max_seqlen / high_freq_factor`` keep it, from
      ``original_max_seqlen / low_freq_factor`` on it is ``factor`` times longer,
      between them the two are mixed linearly in ``original_max_seqlen / wavelength``;
    * ``"yarn"``: pairs that turn more than ``beta_fast`` times in
      ``original_max_seqlen`` tokens keep ``w_i``, those that turn less than
      ``beta_slow`` times get ``w_i / factor``, with a linear ramp over the pairs
      between; cos and sin are multiplied by ``attention_factor`` (by default
      ``0.1 ln(factor) + 1``).

    Angles are formed in 64 bits: at position 10^5 a float32 angle of the
    fastest pair is off by up to 2^-8.
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even and at least 2, now {rotary_dim=}")
    if scaling not in ("none", "linear", "ntk", "wavelength", "yarn"):
        raise ValueError(f"unknown {scaling=}")
    if scaling != "none" and not factor >= 1.0:
        raise ValueError(f"factor must be at least 1, now {factor=}")
    if scaling in ("wavelength", "yarn") and original_max_seqlen < 1:
        raise ValueError(f"{scaling=} needs original_max_seqlen")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64, device=device)
    if scaling == "ntk" and half > 1:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    w = base ** (-2.0 * i / rotary_dim)
    amplitude = 1.0
    if scaling == "linear":
        w = w / factor
    elif scaling == "wavelength":
        if not high_freq_factor > low_freq_factor > 0:
            raise ValueError("high_freq_factor must be above low_freq_factor, and both above 0")
        turns = original_max_seqlen * w / (2.0 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0.0, 1.0)
        w = w * (keep + (1.0 - keep) / factor)
    elif scaling == "yarn":
        if not beta_fast > beta_slow > 0:
            raise ValueError("beta_fast must be above beta_slow, and both above 0")
        # the pair (not whole) that turns `turns` times in the original context
        pair_of = lambda turns: half * math.log(original_max_seqlen / (2.0 * math.pi * turns)) / math.log(base)
        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        slow = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        w = w * ((1.0 - slow) + slow / factor)
        amplitude = 0.1 * math.log(factor) + 1.0 if attention_factor is None else attention_factor
    angle = torch.arange(max_seqlen, dtype=torch.float64, device=device)[:, None] * w[None, :]
    return (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()
