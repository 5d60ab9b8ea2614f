"""Tables of the rotary position embedding, as ``kernels.qk_norm_rope`` reads them.

Pair i of a head's first ``rotary_dim`` elements turns by the angle position *
f_i, with f_i = base^(-2 i / rotary_dim) (J. Su et al., "RoFormer", 2021) and,
for contexts longer than the trained ones, f_i changed by a ``scaling`` rule.
Angles are computed in 64 bits: far positions have angles of many turns, of
which 32 bits would keep too little.
"""

from __future__ import annotations

import math

import torch


def _number(rule: dict, name: str, default=None) -> float:
    value = rule.get(name, default)
    if value is None:
        raise ValueError(f"rotary scaling {rule['type']!r} needs {name!r}")
    value = float(value)
    if not math.isfinite(value) or value <= 0:
        raise ValueError(f"rotary scaling: {name} must be positive")
    return value


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None):
    """(frequencies [rotary_dim / 2] in float64, factor of the cosines and sines).

    ``scaling`` is None or a dict whose "type" is one of

    * "linear": positions divided by "factor" (S. Chen et al., "Extending context
      window ... via positional interpolation", 2023);
    * "ntk": base * factor^(d / (d - 2)) in place of the base, which leaves the
      fastest pair as it is and slows the slowest by "factor";
    * "yarn": pairs of more than "beta_fast" (32) turns within
      "original_max_position" tokens keep their frequency, those of fewer than
      "beta_slow" (1) are slowed by "factor", a ramp over the pair's index lies
      between; cosines and sines are multiplied by "attention_factor" (0.1
      ln(factor) + 1) (B. Peng et al., "YaRN", 2023);
    * "llama3": wavelengths below original_max_position / "high_freq_factor" keep
      their frequency, those above original_max_position / "low_freq_factor"
      are slowed by "factor", between them the frequencies are mixed linearly
      in turns.
    """
    rotary_dim = int(rotary_dim)
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("base must be positive")
    rule = dict(scaling) if scaling is not None else {}
    kind = rule.get("type")
    if scaling is not None and kind not in ("linear", "ntk", "yarn", "llama3"):
        raise ValueError(f"Unknown rotary scaling {kind!r}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("rotary scaling 'ntk' needs a rotary_dim above 2")
        base = base * _number(rule, "factor") ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-i / rotary_dim)
    if kind in (None, "ntk"):
        return freq, 1.0
    factor = _number(rule, "factor")
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "yarn":
        if base <= 1:
            raise ValueError("rotary scaling 'yarn' needs a base above 1")
        length = _number(rule, "original_max_position")

        def pair_of(turns):  # the (real) pair index that makes so many turns within `length` tokens
            return rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_of(_number(rule, "beta_fast", 32.0))), 0)
        high = min(math.ceil(pair_of(_number(rule, "beta_slow", 1.0))), rotary_dim - 1)
        ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return freq / factor * ramp + freq * (1.0 - ramp), _number(rule, "attention_factor",
                                                                   0.1 * math.log(factor) + 1.0)
    length = _number(rule, "original_max_position")
    low, high = _number(rule, "low_freq_factor"), _number(rule, "high_freq_factor")
    if high <= low:
        raise ValueError("rotary scaling: high_freq_factor must exceed low_freq_factor")
    turns = length * freq / (2 * math.pi)
    keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
    return freq / factor * (1.0 - keep) + freq * keep, 1.0


def rotary_table(max_positions: int, rotary_dim: int, base: float = 10000.0, scaling: dict | None = None,
                 device=None) -> torch.Tensor:
    """float32 [max_positions, rotary_dim]: row p holds the cosines, then the
    sines, of position p's rotary_dim / 2 angles (``rotary_frequencies``)."""
    if int(max_positions) <= 0:
        raise ValueError("max_positions must be positive")
    freq, factor = rotary_frequencies(rotary_dim, base, scaling)
    freq = freq.to(device)
    angle = torch.arange(int(max_positions), dtype=torch.float64, device=freq.device)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], dim=1) * factor).float()
