"""Rotary position embedding: which pairs of a head turn, and how fast.

Position p turns pair i of a head by the angle p * f_i: (y0, y1) = c * (x0 cos - x1 sin, x1 cos + x0 sin).
The pairs are (i, i + r/2) in the ``half`` layout and (2i, 2i + 1) in the ``interleaved`` one, over the first
r = ``rotary_dim`` columns of the head; the others pass through. Without scaling f_i = base^(-2i/r) and c = 1.
``scaling`` stretches the frequencies for contexts longer than the trained one:

* ``{"type": "linear", "factor": s}``: f_i / s for every pair;
* ``{"type": "banded", "factor": s, "low": a, "high": b, "original_context": n}``: pairs that turn more than b times
  in n positions keep f_i, those that turn less than a times take f_i / s, linear in the turns between;
* ``{"type": "yarn", "factor": s, "original_context": n, "beta_fast": b, "beta_slow": a}``: the same idea, linear in
  the pair's index between the (whole) indices at which a pair turns b and a times in n positions, and
  c = 0.1 ln s + 1.

The frequencies are 64-bit numbers. The kernel takes each as turns per position in two 64-bit words and reduces p * f_i
to a part of one turn exactly, so that the angle of position 2^52 is as good as that of position 1.
"""

from dataclasses import dataclass, field
from fractions import Fraction
import math

import torch

LAYOUTS = ("half", "interleaved")
_TURN = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
_SCALINGS = {
    "linear": ("factor",),
    "banded": ("factor", "low", "high", "original_context"),
    "yarn": ("factor", "original_context", "beta_fast", "beta_slow"),
}


def _positive(value):
    return type(value) in (int, float) and math.isfinite(value) and value > 0


@dataclass(frozen=True)
class RotaryEmbedding:
    """Rotation of one head size; shared by every plan that writes rotated keys."""

    head_dim: int
    rotary_dim: int | None = None
    layout: str = "half"
    base: float = 10000.0
    scaling: dict | None = None
    frequencies: tuple = field(init=False, repr=False, compare=False)  # radians per position of each pair
    rates: torch.Tensor = field(init=False, repr=False, compare=False)  # turns per position, fp64 [2, r / 2]: words, rests
    factor: float = field(init=False, repr=False, compare=False)  # on cos and sin
    _uploads: dict = field(init=False, repr=False, compare=False, default_factory=dict)  # rates by device

    def __post_init__(self):
        if type(self.head_dim) is not int or self.head_dim <= 0:
            raise ValueError("head_dim must be a positive integer")
        dim = self.head_dim if self.rotary_dim is None else self.rotary_dim
        if type(dim) is not int or not 0 < dim <= self.head_dim or dim % 2:
            raise ValueError("rotary_dim must be an even integer in [2, head_dim]")
        if self.layout not in LAYOUTS:
            raise ValueError(f"rotary layout must be one of {LAYOUTS}")
        if not _positive(self.base) or self.base <= 1:
            raise ValueError("rotary base must be a finite number above 1")
        scaling = None if self.scaling is None else dict(self.scaling)
        if scaling is not None:
            names = _SCALINGS.get(scaling.get("type"))
            if names is None or set(scaling) != {"type", *names}:
                raise ValueError(f"rotary scaling takes 'type' and the numbers of one of {_SCALINGS}")
            if not all(_positive(scaling[name]) for name in names):
                raise ValueError("rotary scaling takes finite positive numbers")
            if scaling["type"] == "banded" and scaling["high"] <= scaling["low"]:
                raise ValueError("banded rotary scaling requires high > low")
            if scaling["type"] == "yarn" and scaling["beta_fast"] < scaling["beta_slow"]:
                raise ValueError("yarn rotary scaling requires beta_fast >= beta_slow")
        object.__setattr__(self, "rotary_dim", dim)
        object.__setattr__(self, "scaling", scaling)
        frequencies, factor = _frequencies(dim, float(self.base), scaling)
        turns = [Fraction(f) / _TURN for f in frequencies]
        rates = [[float(t) for t in turns], [float(t - Fraction(float(t))) for t in turns]]
        object.__setattr__(self, "frequencies", tuple(frequencies))
        object.__setattr__(self, "rates", torch.tensor(rates, dtype=torch.float64))
        object.__setattr__(self, "factor", factor)

    def rates_on(self, device):
        """The rates on a device: uploaded once, and whole before any stream reads them."""
        rates = self._uploads.get(device)
        if rates is None:
            with torch.cuda.device(device):
                rates = self.rates.to(device)
                torch.cuda.current_stream(device).synchronize()
            rates = self._uploads.setdefault(device, rates)
        return rates


def _frequencies(dim, base, scaling):
    """Radians per position of every pair, and the factor on cos and sin."""
    plain = [base ** (-2 * i / dim) for i in range(dim // 2)]
    if scaling is None:
        return plain, 1.0
    s = scaling["factor"]
    if scaling["type"] == "linear":
        return [f / s for f in plain], 1.0
    context = scaling["original_context"]
    if scaling["type"] == "banded":
        low, high = scaling["low"], scaling["high"]
        keep = [min(max((context * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for f in plain]
        return [f * (k + (1 - k) / s) for f, k in zip(plain, keep)], 1.0

    def pair(turns):  # the (real) index of the pair that makes this many turns in the context
        return dim * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(pair(scaling["beta_fast"])), 0), min(math.ceil(pair(scaling["beta_slow"])), dim - 1)
    keep = [1 - min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(dim // 2)]
    return [f * (k + (1 - k) / s) for f, k in zip(plain, keep)], 0.1 * math.log(s) + 1
