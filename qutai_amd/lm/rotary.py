"""Rotary positions beyond the Decoder's default: pairs (2i, 2i+1) or halves
(i, i + R/2), over the first R channels of a head, with frequencies scaled for
contexts longer than those a model was trained on."""
from __future__ import annotations

import ctypes
from functools import lru_cache
from math import isfinite, log, pi

LAYOUTS = ("interleaved", "half")
SCALINGS = {"linear": {"factor"}, "base": {"factor"},
            "parts": {"factor", "original_length", "low", "high", "magnitude"}}


def _number(value, low):
    """Whether this is a finite number above ``low`` that a float holds."""
    if not isinstance(value, (int, float)) or isinstance(value, bool):
        return False
    try:
        return isfinite(value) and value > low
    except OverflowError:  # an integer beyond every float
        return False


def checked_scaling(scaling, rotary_dim):
    """The scaling as a dict with every default filled in (None without one);
    ValueError where it is not one."""
    if scaling is None:
        return None
    if not isinstance(scaling, dict) or scaling.get("kind") not in tuple(SCALINGS):
        raise ValueError(f"a rotary scaling is a dict whose kind is one of {', '.join(SCALINGS)}")
    kind = scaling["kind"]
    if set(scaling) - {"kind"} - SCALINGS[kind] or not _number(scaling.get("factor"), 0):
        raise ValueError(f"{kind} scaling takes {', '.join(sorted(SCALINGS[kind]))}, of which factor is needed, above 0")
    if kind == "base" and rotary_dim <= 2:
        raise ValueError("base scaling needs more than one pair")
    result = dict(scaling)
    if kind == "parts":
        result = {"low": 1.0, "high": 32.0, **result}
        result.setdefault("magnitude", 0.1 * log(result["factor"]) + 1.0 if result["factor"] > 1 else 1.0)
        if not _number(result.get("original_length"), 0):
            raise ValueError("parts scaling needs the original_length, above 0")
        if not _number(result["magnitude"], 0) or not 2.0 ** -126 <= result["magnitude"] < 1e30:
            raise ValueError("parts scaling needs a magnitude that fp32 holds, from 2^-126 to 1e30")
        if not _number(result["low"], -1) or result["low"] < 0 or not _number(result["high"], result["low"]):
            raise ValueError("parts scaling needs 0 <= low < high turns")
    return result


class Rotary:
    """The turns of a head's pairs: pair i of the first ``rotary_dim`` (all)
    channels by theta^(-2i/rotary_dim) radians a position.  ``layout``: a pair is
    channels (2i, 2i+1), "interleaved", or (i, i + rotary_dim/2), "half".
    ``scaling`` stretches the context by a ``factor``:

    * ``{"kind": "linear", "factor": f}``: every frequency divided by f;
    * ``{"kind": "base", "factor": f}``: theta times f^(R/(R-2)), which divides the
      lowest frequency by f and leaves the highest;
    * ``{"kind": "parts", "factor": f, "original_length": n, "low": 1, "high": 32,
      "magnitude": 0.1 ln f + 1}``: frequencies that make ``high`` turns or more in
      n positions stay, those of ``low`` or fewer are divided by f, those between
      are blended linearly in their turns; turned channels are multiplied by the
      magnitude.
    """

    def __init__(self, dim, theta=10000.0, *, rotary_dim=None, layout="interleaved", scaling=None):
        rotary_dim = dim if rotary_dim is None else rotary_dim
        if type(dim) is not int or not 0 < dim <= 256 or type(rotary_dim) is not int or rotary_dim % 2 \
                or not 0 < rotary_dim <= dim:
            raise ValueError("rotary positions take heads of up to 256 channels, of which an even number is turned")
        if layout not in LAYOUTS or not _number(theta, 0):
            raise ValueError("the layout is interleaved or half, theta a positive number")
        self.scaling = scaling = checked_scaling(scaling, rotary_dim)
        self.dim, self.theta, self.rotary_dim, self.layout = dim, float(theta), rotary_dim, layout
        self.magnitude, base = 1.0, self.theta
        kind = None if scaling is None else scaling["kind"]
        try:
            if kind == "base":
                base *= scaling["factor"] ** (rotary_dim / (rotary_dim - 2))
            frequencies = [base ** (-2 * i / rotary_dim) for i in range(rotary_dim // 2)]
        except OverflowError:
            raise ValueError("theta and the scaling's factor give frequencies beyond every float") from None
        if kind == "linear":
            frequencies = [f / scaling["factor"] for f in frequencies]
        elif kind == "parts":
            self.magnitude = float(scaling["magnitude"])
            low, high = scaling["low"], scaling["high"]
            for i, f in enumerate(frequencies):
                kept = min(1.0, max(0.0, (scaling["original_length"] * f / (2 * pi) - low) / (high - low)))
                frequencies[i] = f * (kept + (1 - kept) / scaling["factor"])
        self.frequencies = tuple(frequencies)  # radians a position
        if not isfinite(base) or not all(isfinite(f) for f in frequencies):
            raise ValueError("the scaled frequencies are not finite")
        self._turns = (ctypes.c_double * len(frequencies))(*(f / (2 * pi) for f in frequencies))

    @property
    def turns(self):
        """Address of the whole turns a position of every pair (fp64, host)."""
        return ctypes.addressof(self._turns)


@lru_cache(maxsize=16)
def default_rotary(dim, theta):
    """The Decoder's own rotation as a Rotary, made once for a width and theta: a block
    asks for it every time it runs over packed sequences."""
    return Rotary(dim, theta)
