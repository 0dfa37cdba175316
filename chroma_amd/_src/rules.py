"""Rules that adjust logits before a token is chosen: penalties for repeated tokens, biases, allowed tokens.

``TokenRules`` describes one row; ``pack`` lays the rules of several rows out for the device
(``chroma_hip_run_top_adjusted``), and ``apply`` evaluates them on a downloaded row in the same float
arithmetic, for programs that do not run on the device. (No counterpart in the reference, whose chat script
samples from the raw row, scripts/chat.py:82-98.)
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Dict, Mapping, Optional, Sequence, Union

import numpy as np

from chroma_amd._src.dtypes import BFLOAT16, bf16_to_float32, float32_to_bf16


def _ids(value: Any, name: str) -> np.ndarray:
    ids = np.asarray(value)
    if ids.ndim != 1 or (len(ids) and not np.issubdtype(ids.dtype, np.integer)):
        raise TypeError(f"{name} must be a 1-D sequence of integer token ids")
    return ids.astype(np.int64)


@dataclass(frozen=True, eq=False)
class TokenRules:
    """What happens to a row of logits before tokens are chosen from it, in this order:

    * a token that occurs c > 0 times in ``history``: ``x > 0 ? x / repetition : x * repetition``, then minus
      ``presence + frequency * c``;
    * plus ``bias``: a mapping of token ids to numbers, or an array over the vocabulary;
    * -inf for tokens outside ``allowed``: token ids, or a boolean array over the vocabulary.

    The arithmetic is float32's, the result rounded once to the logits' type."""

    history: Sequence[int] = ()
    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: Optional[Union[Mapping[int, float], np.ndarray]] = None
    allowed: Optional[Any] = None

    def __post_init__(self) -> None:
        with np.errstate(over="ignore"):
            factors = {name: np.float32(getattr(self, name)) for name in ("repetition", "presence", "frequency")}
        for name, factor in factors.items():
            if not np.isfinite(factor):
                raise ValueError(f"{name} must be finite in float32, got {getattr(self, name)}")
        if factors["repetition"] <= 0:
            raise ValueError(f"repetition must be positive in float32, got {self.repetition}")
        object.__setattr__(self, "history", _ids(self.history, "history"))
        if self.bias is not None and not isinstance(self.bias, Mapping):
            bias = np.asarray(self.bias, dtype=np.float32)
            if bias.ndim != 1:
                raise ValueError("bias must be a mapping of token ids or an array over the vocabulary")
            object.__setattr__(self, "bias", bias)
        if self.allowed is not None:
            allowed = np.asarray(self.allowed)
            if allowed.ndim != 1:
                raise TypeError("allowed must be token ids or a boolean array over the vocabulary")
            object.__setattr__(self, "allowed", allowed if allowed.dtype == np.bool_ else _ids(allowed, "allowed"))

    def check(self, vocab_size: int) -> None:
        """Raise unless every id and array fits a vocabulary of ``vocab_size`` tokens."""
        bias_ids = _ids(list(self.bias), "bias") if isinstance(self.bias, Mapping) else np.empty(0, np.int64)
        allowed_ids = self.allowed if self.allowed is not None and self.allowed.dtype != np.bool_ else np.empty(0, np.int64)
        for name, ids in (("history", self.history), ("bias", bias_ids), ("allowed", allowed_ids)):
            if len(ids) and (ids.min() < 0 or ids.max() >= vocab_size):
                raise IndexError(f"{name} token ids must lie in [0, {vocab_size})")
        for name, array in (("bias", self.bias), ("allowed", self.allowed)):
            if isinstance(array, np.ndarray) and (name == "bias" or array.dtype == np.bool_) and len(array) != vocab_size:
                raise ValueError(f"{name} holds {len(array)} values, the vocabulary {vocab_size}")
        if self.allowed is not None and not (self.allowed.any() if self.allowed.dtype == np.bool_ else len(self.allowed)):
            raise ValueError("no token is allowed")

    def write_bias(self, row: np.ndarray) -> None:
        """Write the bias into a row of zeros."""
        if isinstance(self.bias, np.ndarray):
            row[:] = self.bias
        else:
            for token, value in (self.bias or {}).items():
                row[token] = value

    def allowed_row(self, vocab_size: int) -> np.ndarray:
        if self.allowed is None:
            return np.ones(vocab_size, dtype=np.bool_)
        if self.allowed.dtype == np.bool_:
            return self.allowed
        row = np.zeros(vocab_size, dtype=np.bool_)
        row[self.allowed] = True
        return row

    def apply(self, row: np.ndarray) -> np.ndarray:
        """The adjusted row (float32 or bfloat16) on the host."""
        vocab_size = len(row)
        self.check(vocab_size)
        x = bf16_to_float32(row) if row.dtype == BFLOAT16 else row.copy()
        with np.errstate(over="ignore", invalid="ignore"):
            ids, counts = np.unique(self.history, return_counts=True)
            old = x[ids]
            repetition, presence, frequency = (np.float32(v) for v in (self.repetition, self.presence, self.frequency))
            x[ids] = np.where(old > 0, old / repetition, old * repetition) - (presence + frequency * counts.astype(np.float32))
            if self.bias is not None:
                bias = np.zeros(vocab_size, dtype=np.float32)
                self.write_bias(bias)
                x += bias
        x[~self.allowed_row(vocab_size)] = -np.inf
        return float32_to_bf16(x) if row.dtype == BFLOAT16 else x


def unread(rules: Sequence[TokenRules]) -> TokenRules:
    """What a row that nobody reads is given beside ``rules``: the bias and the allowed tokens that all of them share, so
    that it does not end the sharing, and nothing else."""
    row = TokenRules()
    for name in ("bias", "allowed"):
        value = getattr(rules[0], name)
        if all(getattr(rule, name) is value for rule in rules):
            object.__setattr__(row, name, value)
    return row


def pack(rules: Sequence[TokenRules], vocab_size: int) -> Dict[str, Optional[np.ndarray]]:
    """The rows' rules as the arrays of ``chroma_hip_adjust_call``: history [rows, longest] padded with -1, its
    lengths, the three factors, bias [rows, vocab] and mask words [rows, ceil(vocab / 32)] (bias and mask as one
    row when every row's is the same object, None when no row has one)."""
    for rule in rules:
        rule.check(vocab_size)
    lengths = np.array([len(rule.history) for rule in rules], dtype=np.int64)
    history = None
    if lengths.any():
        history = np.full((len(rules), int(lengths.max())), -1, dtype=np.int64)
        for row, rule in zip(history, rules):
            row[: len(rule.history)] = rule.history
    arrays: Dict[str, Optional[np.ndarray]] = {"history": history, "history_lengths": None if history is None else lengths}
    for name in ("repetition", "presence", "frequency"):
        arrays[name] = None if history is None else np.array([getattr(rule, name) for rule in rules], dtype=np.float32)

    def rows_of(values: Sequence[Any]) -> Sequence[int]:
        """The rows to lay out: one when all share it."""
        return [0] if all(value is values[0] for value in values) else range(len(values))

    arrays["bias"] = arrays["mask"] = None
    if any(rule.bias is not None for rule in rules):
        chosen = rows_of([rule.bias for rule in rules])
        arrays["bias"] = np.zeros((len(chosen), vocab_size), dtype=np.float32)
        for row, i in zip(arrays["bias"], chosen):
            rules[i].write_bias(row)
    if any(rule.allowed is not None for rule in rules):
        chosen = rows_of([rule.allowed for rule in rules])
        words = arrays["mask"] = np.full((len(chosen), -(-vocab_size // 32)), 0xFFFFFFFF, dtype=np.uint32)
        bits = np.zeros(words.shape[1] * 32, dtype=np.bool_)
        for row, i in zip(words, chosen):
            if rules[i].allowed is not None:
                bits[:vocab_size] = rules[i].allowed_row(vocab_size)
                row[:] = np.packbits(bits, bitorder="little").view(np.uint32)
    return arrays
