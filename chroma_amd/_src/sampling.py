"""How a token is drawn from a row of logits: temperature, top-k, top-p and min-p.

``Sampling`` describes one row; ``pack`` lays the settings of several rows out for the device
(``chroma_hip_run_sample``), and ``draw`` draws from a downloaded row by the same rule, for programs that do not run on the
device. (The reference's chat script samples on the host, from the downloaded row, scripts/chat.py:82-98.)
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Any, Dict, Sequence, Tuple

import numpy as np

from chroma_amd._src.dtypes import BFLOAT16, bf16_to_float32


@dataclass(frozen=True)
class Sampling:
    """In descending order of the logits, ties to the lower id, token i has the weight ``exp((x_i - x_max) / temperature)``, and
    of the row's tokens are kept

    * the first ``top_k`` (0: all);
    * of those, the fewest first ones whose weights reach ``top_p`` of their sum;
    * of those, the ones of at least ``min_p`` (the largest weighs 1), one at least.

    A random number u from [0, 1) draws the first token whose running sum of weights exceeds u times the kept sum. A
    temperature of 0 takes the largest logit."""

    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    def __post_init__(self) -> None:
        if not isinstance(self.top_k, (int, np.integer)) or self.top_k < 0:
            raise ValueError(f"top_k must be an integer of at least 0, got {self.top_k!r}")
        for name, low, high in (("temperature", 0.0, float(np.finfo(np.float32).max)), ("top_p", 0.0, 1.0), ("min_p", 0.0, 1.0)):
            if not low <= getattr(self, name) <= high:
                raise ValueError(f"{name} must lie in [{low}, {high}], got {getattr(self, name)}")


def check_uniform(value: Any) -> np.float32:
    """A random number as float32 (one that rounds up to 1 becomes the largest below)."""
    if not 0.0 <= value < 1.0:
        raise ValueError(f"uniform must lie in [0, 1), got {value}")
    return min(np.float32(value), np.nextafter(np.float32(1), np.float32(0)))


def pack(sampling: Sequence[Sampling], uniform: Sequence[float]) -> Dict[str, np.ndarray]:
    """The rows' settings as the arrays of ``chroma_hip_sample_call``."""
    arrays = {name: np.array([getattr(one, name) for one in sampling], dtype=np.float32) for name in ("temperature", "top_p", "min_p")}
    arrays["top_k"] = np.array([min(one.top_k, 2**31) for one in sampling], dtype=np.int64)
    arrays["uniform"] = np.array([check_uniform(value) for value in uniform], dtype=np.float32)
    return arrays


def draw(row: np.ndarray, sampling: Sampling, uniform: float) -> Tuple[int, float]:
    """(token id, logarithm of its share of the kept weights) of a row (float32 or bfloat16) on the host; -1 where every logit
    is -inf, the first NaN's id where one is NaN."""
    arrays = pack([sampling], [uniform])
    temperature, top_p, min_p, u = (float(arrays[name][0]) for name in ("temperature", "top_p", "min_p", "uniform"))
    x = (bf16_to_float32(row) if row.dtype == BFLOAT16 else row).astype(np.float64)
    if np.isnan(x).any():
        return int(np.isnan(x).argmax()), math.nan
    top = x.max()
    if top == -math.inf:
        return -1, -math.inf
    if temperature == 0:
        return int(x.argmax()), 0.0
    order = np.argsort(-x, kind="stable")
    x = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        depth = np.where(x == top, 0.0, (top - x) / temperature)
    # units of 2^-44 of the largest, as the device sums them
    units = np.rint(np.exp(-depth) * 2.0**44).astype(np.uint64)
    sums = units.cumsum()
    kept = sampling.top_k if 0 < sampling.top_k < len(x) else len(x)
    if top_p < 1:
        # the goal in exact integers: a share is a multiple of 2^-149
        goal = max(1, (int(top_p * 2.0**149) * int(sums[kept - 1]) + 2**149 - 1) >> 149)
        kept = min(kept, int(np.searchsorted(sums, np.uint64(goal))) + 1)
    if min_p > 0:
        kept = max(1, min(kept, int((units >= math.ceil(min_p * 2.0**44)).sum())))
    place = int(u * 2.0**149) * int(sums[kept - 1]) >> 149
    chosen = int(np.searchsorted(sums, np.uint64(place), side="right"))
    return int(order[chosen]), -float(depth[chosen]) - math.log(int(sums[kept - 1]) / 2.0**44)
