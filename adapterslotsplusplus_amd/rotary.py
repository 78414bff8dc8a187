"""Rotary positions: how far each pair of a head's elements turns per position.

The engine's kernels (`rotate_heads`, `rotate_into_cache`) take frequencies as
64-bit fractions of a turn.  A position times such a fraction, modulo 2^64, is
the angle modulo one turn without any rounding, so there is no table of
cosines and no longest position.  What is left is the frequency's own error, a
few 2^-53 of it and 2^-65 turns: under 2^-22 turns at position 2^31.
"""
from __future__ import annotations

import math
from typing import List, Mapping, Optional, Tuple

import torch


def _number(scaling: Mapping, name: str, kind: str, default: Optional[float] = None, positive: bool = True) -> float:
    v = scaling.get(name)
    if v is None:
        v = default
    if v is None:
        raise RuntimeError(f"Rotary: {kind} scaling needs {name!r}")
    v = float(v)
    if not (math.isfinite(v) and (v > 0 or not positive)):
        raise RuntimeError(f"Rotary: {name} must be a {'positive' if positive else 'finite'} number, got {v}")
    return v


def frequencies(dim: int, base: float = 10000.0, scaling: Optional[Mapping] = None) -> Tuple[List[float], float]:
    """(radians a position for each of the dim / 2 pairs, what cosine and sine
    are multiplied by).  Pair i turns by base ** (-2 i / dim) a position.
    scaling, for contexts `factor` times as long as the trained ones:

      type "linear"  every frequency divided by factor
      type "ntk"     base raised by factor ** (dim / (dim - 2)), so that the
                     slowest pair is stretched by factor and the fastest not at all
      type "yarn"    pairs that turn at least beta_fast (32) times over
                     original_length stay, those that turn at most beta_slow (1)
                     times are divided by factor, linearly by the pair's index
                     between; cosine and sine times attention_factor
                     (0.1 ln(factor) + 1 for factors above 1)
      type "bands"   the same between high_freq_factor (4) and low_freq_factor
                     (1) turns over original_length, linearly by the turns
    """
    if dim < 2 or dim % 2:
        raise RuntimeError(f"Rotary: {dim} elements do not form pairs")
    base = float(base)
    if not (math.isfinite(base) and base > 1.0):
        raise RuntimeError(f"Rotary: base must be above 1, got {base}")
    half = dim // 2
    scaling = dict(scaling) if scaling else {"type": "none"}
    kind = scaling.get("type")
    if kind not in ("none", "linear", "ntk", "yarn", "bands"):
        raise RuntimeError(f"Rotary: unknown scaling {kind!r}")
    factor = 1.0 if kind == "none" else _number(scaling, "factor", kind)
    if kind == "ntk" and dim > 2:
        base *= factor ** (dim / (dim - 2.0))
        if not 1.0 < base < math.inf:
            raise RuntimeError(f"Rotary: factor {factor} takes the base out of range")
    plain = [base ** (-2.0 * i / dim) for i in range(half)]
    if kind == "linear":
        return [f / factor for f in plain], 1.0
    if kind == "yarn":
        length = _number(scaling, "original_length", kind)

        def pair(turns: float) -> float:  # the (fractional) index that turns so often over the trained length
            return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair(_number(scaling, "beta_fast", kind, 32.0))), 0)
        high = min(math.ceil(pair(_number(scaling, "beta_slow", kind, 1.0))), dim - 1)
        stretch = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(half)]
        more = _number(scaling, "attention_factor", kind, 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0, positive=False)
        return [f / factor * s + f * (1.0 - s) for f, s in zip(plain, stretch)], more
    if kind == "bands":
        length = _number(scaling, "original_length", kind)
        low, high = (_number(scaling, n, kind, d, positive=False) for n, d in (("low_freq_factor", 1.0), ("high_freq_factor", 4.0)))
        if not high > low:
            raise RuntimeError("Rotary: high_freq_factor must be above low_freq_factor")
        keep = [min(max((length * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for f in plain]
        return [f / factor * (1.0 - s) + f * s for f, s in zip(plain, keep)], 1.0
    return plain, 1.0


class Rotary:
    """A model's rotation: `dim` elements of each head turn, pairs (i, i + dim / 2)
    or, interleaved, (2i, 2i + 1); see frequencies() for base and scaling.
    turns: int64 [dim / 2] on the device, 2^64ths of a turn a position."""

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, scaling: Optional[Mapping] = None,
                 device=None):
        freq, self.factor = frequencies(dim, base, scaling)
        self.dim, self.interleaved = int(dim), bool(interleaved)
        # 2^64 / (2 pi) is a double's 53 bits; so is each frequency.
        fixed = [round(f / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for f in freq]
        fixed = [v - (1 << 64) if v >= 1 << 63 else v for v in fixed]
        if device is None:
            device = "cuda"
        self.turns = torch.tensor(fixed, dtype=torch.int64).to(device)
