"""The layers of a transformer over packed batches."""
import math

import numpy as np

from ... import _C
from ...random import dropout
from ..Module import Module
from .linear import Linear


class LayerNorm(Module):
    """(x - mean) / sqrt(var + eps) * weights + bias over the last axis."""

    def __init__(self, features: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        kw = {}
        if device is not None:
            kw["device"] = device
        if dtype is not None:
            kw["dtype"] = dtype
        self.eps = eps
        self.requires_bias = bias
        self.weights = _C.ones([features], requires_grad=True, **kw)
        if bias:
            self.bias = _C.zeros([features], requires_grad=True, **kw)

    def forward(self, x):
        return _C.layer_norm(x, self.weights, self.bias if self.requires_bias else None, self.eps)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling=None):
    """(radians per position of each pair, the factor on the rotated values) as float64 and a float.

    Pair j turns base^(-2 j / rotary_dim) a position.  `scaling` stretches a model to longer contexts:
      {"kind": "linear", "factor": f}   positions divided by f
      {"kind": "base", "factor": f}     a base of base * f^(rotary_dim / (rotary_dim - 2)): the slowest pair turns f times
                                        slower, the fastest as before
      {"kind": "by_parts", "factor": f, "original": n, "slow": 1, "fast": 32}
                                        pairs that turn less than `slow` times over the original context of n positions
                                        are f times slower, those that turn more than `fast` times are as before, linear
                                        in their turns in between; the rotated values times 0.1 ln f + 1 (Peng, Quesnelle,
                                        Fan and Shippole, 2023)"""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_frequencies: rotary_dim {rotary_dim} is not even")
    if not base > 0:
        raise ValueError("rotary_frequencies: base must be positive")
    j = np.arange(rotary_dim // 2, dtype=np.float64)
    kind = None if scaling is None else scaling["kind"]
    factor = 1.0 if scaling is None else float(scaling["factor"])
    if not (factor > 0 and math.isfinite(factor)):
        raise ValueError("rotary_frequencies: factor must be positive")
    if kind == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = float(base) ** (-2 * j / max(1, rotary_dim))
    if kind in (None, "base"):
        return f, 1.0
    if kind == "linear":
        return f / factor, 1.0
    if kind == "by_parts":
        slow, fast = float(scaling.get("slow", 1)), float(scaling.get("fast", 32))
        if not fast > slow:
            raise ValueError("rotary_frequencies: fast must be above slow")
        turns = float(scaling["original"]) * f / (2 * math.pi)
        keep = np.clip((turns - slow) / (fast - slow), 0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    raise ValueError(f"rotary_frequencies: unknown scaling {kind!r}")


def packed_positions(q_lengths, k_lengths=None):
    """Each query's place in its sequence, for Rotary: a sequence with more keys than queries ends at its last key."""
    k_lengths = q_lengths if k_lengths is None else k_lengths
    runs = [np.arange(k - q, k, dtype=np.int64) for q, k in zip(q_lengths, k_lengths, strict=True)]
    return _C.Variable(np.concatenate([np.zeros(0, np.int64), *runs]), dtype=_C.dtype.int64)


class Rotary(Module):
    """Turns pairs of the first `heads` vectors of each row by their position (rsl.rotary); no parameters.

    `rotary_dim`: how much of each vector turns (all of it unless given); `interleaved`: pairs of neighbours rather than of
    halves; `base` and `scaling` as rotary_frequencies takes them."""

    def __init__(self, head_dim: int, rotary_dim=None, base: float = 10000.0, interleaved: bool = False, scaling=None) -> None:
        super().__init__()
        self.head_dim, self.rotary_dim = head_dim, head_dim if rotary_dim is None else rotary_dim
        if self.rotary_dim > head_dim:
            raise ValueError("rotary_dim is above head_dim")
        self.interleaved = interleaved
        self.frequencies, self.scale = rotary_frequencies(self.rotary_dim, base, scaling)
        # Sent before any recording, in which a copy from the host has no place.
        self._held = self._on_device() if _C.hip.is_available() else None

    def _on_device(self):
        return _C._Tensor(self.frequencies, [len(self.frequencies)], _C.device.hip, _C.dtype.float64)

    def forward(self, x, positions, heads: int):
        if self._held is None:
            self._held = self._on_device()
        return _C.rotary(x, positions, self._held, heads=heads, head_dim=self.head_dim, interleaved=self.interleaved,
                         scale=self.scale)


class RandomDropout(Module):
    """residual + what is kept of x / (1 - rate), from an rsl.Generator; with `active` off, residual + x.

    (Dropout draws on the host and does not scale what it keeps.)"""

    def __init__(self, rate: float, generator) -> None:
        super().__init__()
        if not 0 <= rate <= 1:
            raise ValueError("rate lies in [0, 1]")
        self.rate, self.generator, self.active = rate, generator, True

    def forward(self, x, residual=None):
        if self.active:
            return dropout(x, self.rate, self.generator, residual)
        return x if residual is None else residual + x


class GatedLinear(Module):
    """act(x @ Wg + bg) * (x @ Wu + bu), both projections from one matrix [Wg | Wu]."""

    def __init__(self, in_features: int, hidden: int, gate: str = "silu", bias: bool = True) -> None:
        super().__init__()
        self.gate, self.requires_bias = gate, bias
        self.weights = _C.randn(0, 1, [in_features, 2 * hidden], requires_grad=True)
        if bias:
            self.bias = _C.randn(0, 1, [2 * hidden], requires_grad=True)

    def forward(self, x):
        return _C.gated_linear(x, self.weights, self.bias if self.requires_bias else None, self.gate)


class GatedFeedForward(Module):
    """A GatedLinear and the projection back."""

    def __init__(self, features: int, hidden: int, gate: str = "silu", bias: bool = True) -> None:
        super().__init__()
        self.up, self.down = GatedLinear(features, hidden, gate, bias), Linear(hidden, features, bias)

    def forward(self, x):
        return self.down(self.up(x))


class VocabularyLoss(Module):
    """A Linear to a vocabulary and the mean softmax cross entropy of its outputs, without holding them.

    targets: int64, negative where a row is not counted; weights: each row's in place of the mean."""

    def __init__(self, features: int, vocabulary: int, bias: bool = True) -> None:
        super().__init__()
        self.head = Linear(features, vocabulary, bias)

    def _bias(self):
        return self.head.bias if self.head.requires_bias else None

    def forward(self, x, targets, weights=None):
        return _C.linear_cross_entropy(x, self.head.weights, self._bias(), targets, weights)

    def rows(self, x, targets):
        """Each row's loss, without a gradient."""
        return _C.linear_cross_entropy_rows(x, self.head.weights, self._bias(), targets)

    def logits(self, x):
        return self.head(x)


class SelfAttention(Module):
    """One projection to queries, keys and values, attention over the plan's packed sequences, one projection back.

    x is [tokens, features], the sequences one after another; `plan` an AttentionPlan of the layer's heads.  With `rotary`
    (a Rotary of the head's size) queries and keys are turned by `positions`."""

    def __init__(self, features: int, heads: int, kv_heads=None, head_dim=None, bias: bool = True, rotary=None) -> None:
        super().__init__()
        self.heads, self.kv_heads = heads, heads if kv_heads is None else kv_heads
        if head_dim is None and features % heads:
            raise ValueError("features must be a multiple of heads unless head_dim is given")
        self.head_dim = features // heads if head_dim is None else head_dim
        if rotary is not None and rotary.head_dim != self.head_dim:
            raise ValueError("the rotary layer is of another head_dim")
        self.qkv = Linear(features, (heads + 2 * self.kv_heads) * self.head_dim, bias)
        self.out = Linear(heads * self.head_dim, features, bias)
        self.rotary = rotary

    def plan(self, q_lengths, k_lengths=None, causal: bool = True):
        return _C.AttentionPlan(q_lengths, k_lengths, heads=self.heads, kv_heads=self.kv_heads,
                                head_dim=self.head_dim, causal=causal)

    def rows(self, x, positions=None):
        """Queries, keys and values of x side by side, turned where the layer has a rotary one."""
        rows = self.qkv(x)
        if self.rotary is None:
            return rows
        if positions is None:
            raise ValueError("rotary attention needs the rows' positions")
        return self.rotary(rows, positions, self.heads + self.kv_heads)

    def forward(self, x, plan, positions=None):
        return self.out(_C.attention_qkv(self.rows(x, positions), plan))
