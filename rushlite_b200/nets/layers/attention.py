from ... import _C
from ..Module import Module
from .linear import Linear


class CausalSelfAttention(Module):
    """Causal self-attention over packed sequences: x [tokens, features] and
    the ``Sequences`` it packs.  Fewer key/value heads than query heads share
    each key/value head among heads // kv_heads query heads.  float32, with
    features // heads at most 128."""

    def __init__(self, features: int, heads: int, kv_heads=None, bias: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or features < 1 or features % heads:
            raise ValueError("features must be a multiple of heads")
        if kv_heads < 1 or heads % kv_heads:
            raise ValueError("heads must be a multiple of kv_heads")
        if features // heads > 128:
            raise ValueError(f"the head dimension is at most 128, got {features // heads}")
        if dtype is not None and dtype != _C.dtype.float32:
            raise ValueError("CausalSelfAttention computes in float32 only")
        object.__setattr__(self, "heads", heads)
        object.__setattr__(self, "kv_heads", kv_heads)
        object.__setattr__(self, "head_dim", features // heads)
        kv = kv_heads * self.head_dim
        self.query = Linear(features, features, bias, device, dtype)
        self.key = Linear(features, kv, bias, device, dtype)
        self.value = Linear(features, kv, bias, device, dtype)
        self.out = Linear(features, features, bias, device, dtype)

    def forward(self, x, sequences):
        t, d = x.shape[0], self.head_dim
        q = _C.reshape(self.query(x), [t, self.heads, d])
        k = _C.reshape(self.key(x), [t, self.kv_heads, d])
        v = _C.reshape(self.value(x), [t, self.kv_heads, d])
        y = _C.causal_attention(q, k, v, sequences)
        return self.out(_C.reshape(y, [t, self.heads * d]))
