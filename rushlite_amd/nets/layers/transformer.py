"""LayerNorm and SelfAttention over packed batches."""
from ... import _C
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


class SelfAttention(Module):
    """One projection to queries, keys and values, attention over the plan's packed sequences, one projection back.

    x is [tokens, features], the sequences one after another; `plan` an AttentionPlan of the layer's heads."""

    def __init__(self, features: int, heads: int, kv_heads=None, head_dim=None, bias: bool = True) -> None:
        super().__init__()
        self.heads, self.kv_heads = heads, heads if kv_heads is None else kv_heads
        if head_dim is None and features % heads:
            raise ValueError("features must be a multiple of heads unless head_dim is given")
        self.head_dim = features // heads if head_dim is None else head_dim
        self.qkv = Linear(features, (heads + 2 * self.kv_heads) * self.head_dim, bias)
        self.out = Linear(heads * self.head_dim, features, bias)

    def plan(self, q_lengths, k_lengths=None, causal: bool = True):
        return _C.AttentionPlan(q_lengths, k_lengths, heads=self.heads, kv_heads=self.kv_heads,
                                head_dim=self.head_dim, causal=causal)

    def forward(self, x, plan):
        return self.out(_C.attention_qkv(self.qkv(x), plan))
