from .activation import ReLU, Sigmoid, Softmax, Tanh
from .attention import CausalSelfAttention
from .container import Sequential
from .linear import Flatten, Linear
from .norm import LayerNorm

__all__ = ["ReLU", "Sigmoid", "Softmax", "Tanh", "Sequential", "Flatten", "Linear", "LayerNorm",
           "CausalSelfAttention"]
