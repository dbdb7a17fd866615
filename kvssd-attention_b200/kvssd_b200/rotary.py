"""Rotary position embeddings: the frequencies of a head's pairs and their long-context scalings.

``RotaryEmbedding`` describes what a model was trained with; ``frequencies`` are the FP64 radians a
position that ``ops.rotary`` and ``ops.append`` take. The reference has no counterpart: it caches
keys as it is given them (src/kvssd/store.py:27-67).
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch

from . import ops

SCALINGS = ("none", "linear", "ntk", "smooth", "yarn")


@dataclass(frozen=True)
class RotaryEmbedding:
    """Pair i of ``rotary_dim // 2`` pairs turns by position * base^(-2 i / rotary_dim), rescaled for
    contexts ``factor`` times ``original_length``:

    * ``linear``: every frequency divided by the factor (positions interpolated);
    * ``ntk``: the base raised to base * factor^(rotary_dim / (rotary_dim - 2)), which divides the
      slowest pair's frequency by the factor and leaves the fastest;
    * ``smooth``: pairs that make more than ``high`` turns over the original length keep their
      frequency, those below ``low`` turns are divided, in between the two are blended by the turns;
    * ``yarn``: as ``smooth`` with a ramp over the pair's index between the pairs of ``high`` and of
      ``low`` turns, and cos and sin multiplied by 0.1 ln(factor) + 1.

    ``low`` and ``high`` default to 1 and 4 turns (``smooth``) or 1 and 32 (``yarn``).
    """

    head_dim: int
    rotary_dim: int | None = None  # None: the whole head
    base: float = 10000.0
    interleaved: bool = False
    scaling: str = "none"
    factor: float = 1.0
    original_length: int | None = None
    low: float = 1.0
    high: float | None = None
    _on_device: dict = field(default_factory=dict, init=False, repr=False, compare=False)

    def __post_init__(self) -> None:
        if self.rotary_dim is None:
            object.__setattr__(self, "rotary_dim", self.head_dim)
        if not 2 <= self.rotary_dim <= self.head_dim or self.rotary_dim % 2:
            raise ValueError("rotary_dim must be even and between 2 and head_dim")
        if self.scaling not in SCALINGS:
            raise ValueError(f"unknown scaling '{self.scaling}'; choose one of: {', '.join(SCALINGS)}")
        if not 1.0 < self.base < math.inf or not 1.0 <= self.factor < math.inf:  # NaN: neither
            raise ValueError("base must be above 1 and factor at least 1, both finite")
        if self.scaling == "ntk" and self.rotary_dim == 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        if self.scaling in ("smooth", "yarn"):
            if not self.original_length or self.original_length < 1:
                raise ValueError(f"{self.scaling} scaling needs the original_length")
            if self.high is None:
                object.__setattr__(self, "high", 4.0 if self.scaling == "smooth" else 32.0)
            if not 0 < self.low < self.high < math.inf:
                raise ValueError("low and high turns must be positive, ascending and finite")

    @property
    def magnitude(self) -> float:
        """Factor of cos and sin (above 1 for ``yarn`` only)."""
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "yarn" else 1.0

    def frequencies(self) -> torch.Tensor:
        """Radians a position, float64 [rotary_dim // 2], on the CPU."""
        dim, pair = self.rotary_dim, torch.arange(self.rotary_dim // 2, dtype=torch.float64)
        base = self.base
        if self.scaling == "ntk":
            base = base * self.factor ** (dim / (dim - 2))
        freq = base ** (-2.0 * pair / dim)
        if self.scaling == "linear":
            return freq / self.factor
        if self.scaling == "smooth":
            turns = self.original_length * freq / (2 * math.pi)
            kept = ((turns - self.low) / (self.high - self.low)).clamp(0, 1)
            return freq * kept + freq / self.factor * (1 - kept)
        if self.scaling == "yarn":
            ends = [dim * math.log(self.original_length / (turns * 2 * math.pi))
                    / (2 * math.log(self.base)) for turns in (self.high, self.low)]
            first, last = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), dim - 1)
            divided = ((pair - first) / max(last - first, 1e-3)).clamp(0, 1)
            return freq / self.factor * divided + freq * (1 - divided)
        return freq

    def on(self, device: torch.device | str) -> torch.Tensor:
        """``frequencies()`` on ``device``, kept there for later calls. The first call on a device copies
        them, which cannot be captured in a graph."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        held = self._on_device.get(device)
        if held is None:
            held = self._on_device[device] = self.frequencies().to(device)
        return held

    def apply(self, x: torch.Tensor, positions: torch.Tensor,
              out: torch.Tensor | None = None) -> torch.Tensor:
        """ops.rotary of ``x`` [tokens, heads, head_dim] at ``positions`` [tokens]."""
        if x.ndim != 3 or x.shape[-1] != self.head_dim:
            raise ValueError(f"x must be [tokens, heads, {self.head_dim}]")
        return ops.rotary(x, positions, self.on(x.device), interleaved=self.interleaved,
                          magnitude=self.magnitude, out=out)
