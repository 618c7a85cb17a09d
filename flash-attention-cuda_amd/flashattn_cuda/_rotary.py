"""Frequencies of rotary positions, also for contexts longer than the trained one.

Pair i of ``rotary_dim / 2`` turns by ``w_i = base ** (-2 i / rotary_dim)`` per
position. A context ``stretch`` times the trained length is reached by slowing
the turns:

* ``"linear"``: every w_i / stretch (positions pressed together; position
  interpolation, Chen et al. 2023).
* ``"base"``: a larger base, ``base * stretch ** (R / (R - 2))``, which leaves the
  fastest pair as it is and slows the slowest by ``stretch`` ("NTK-aware" scaling).
* ``"parts"``: pairs that complete more than ``fast_turns`` turns over
  ``trained_length`` keep w_i, those under ``slow_turns`` take w_i / stretch, a ramp
  in i between; with it goes a temperature, ``0.1 ln(stretch) + 1`` on q and k (YaRN,
  Peng et al. 2023).

Models are trained with these rules as published, so their constants are kept as they
are: also the ends of the ramp in "parts", whole pairs cut off at 0 and at R - 1 (past
the last pair, R / 2 - 1: the ramp may end beyond it), and a ramp of no length, which
becomes one of 1e-3 pairs.
"""

import math

import torch


def rope_frequencies(rotary_dim, base=10000.0, scaling=None, stretch=1.0, trained_length=None,
                     fast_turns=32.0, slow_turns=1.0, device=None):
    """(inv_freq, factor): the float64 frequencies ``rope`` and ``append_paged``
    take, and the factor that goes with them (1.0 except for ``"parts"``)."""
    if rotary_dim < 16 or rotary_dim % 16 != 0:
        raise ValueError(f"rotary_dim must be a positive multiple of 16, got {rotary_dim}")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError(f"base must be finite and > 1, got {base}")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'parts', got {scaling!r}")
    if not (math.isfinite(stretch) and stretch >= 1.0):
        raise ValueError(f"stretch must be finite and >= 1, got {stretch}")
    if scaling == "base":
        base = base * stretch ** (rotary_dim / (rotary_dim - 2))
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    inv_freq = base ** -exponent
    factor = 1.0
    if scaling == "linear":
        inv_freq = inv_freq / stretch
    elif scaling == "parts":
        if trained_length is None or trained_length <= 0:
            raise ValueError("scaling 'parts' needs trained_length > 0")
        if not fast_turns > slow_turns > 0:
            raise ValueError(
                f"fast_turns must exceed slow_turns > 0, got {fast_turns} and {slow_turns}")

        def pair_of(turns):  # the (fractional) pair that completes `turns` over the length
            return (rotary_dim * math.log(trained_length / (turns * 2 * math.pi))
                    / (2 * math.log(base)))

        low = max(math.floor(pair_of(fast_turns)), 0)
        high = min(math.ceil(pair_of(slow_turns)), rotary_dim - 1)
        ramp = (torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)
        slowed = ramp.clamp(0.0, 1.0)
        inv_freq = inv_freq * (1.0 - slowed) + inv_freq / stretch * slowed
        factor = 0.1 * math.log(stretch) + 1.0
    return inv_freq.to(device if device is not None else "cpu"), factor
