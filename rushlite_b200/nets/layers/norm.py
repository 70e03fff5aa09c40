from ... import _C
from ..Module import Module


class LayerNorm(Module):
    """y = (x - mean) / sqrt(var + eps) * weights + bias over the last
    dimension; weights start at 1, bias at 0."""

    def __init__(self, features: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        if features < 1:
            raise ValueError("features must be at least 1")
        if not 0 <= eps < float("inf"):
            raise ValueError("eps must be finite and not negative")
        if dtype is not None and dtype not in (_C.dtype.float32, _C.dtype.float64):
            raise ValueError("LayerNorm computes in float32 or float64 only")
        kw = {}
        if device is not None:
            kw["device"] = device
        if dtype is not None:
            kw["dtype"] = dtype
        object.__setattr__(self, "eps", eps)
        object.__setattr__(self, "requires_bias", bias)
        self.weights = _C.ones([features], requires_grad=True, **kw)
        if bias:
            self.bias = _C.zeros([features], requires_grad=True, **kw)

    def forward(self, x):
        return _C.layer_norm(x, self.weights, self.bias if self.requires_bias else None, self.eps)
