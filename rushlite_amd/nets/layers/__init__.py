from .activation import ReLU, Sigmoid, Softmax, Tanh
from .container import Sequential
from .dropout import Dropout
from .linear import Flatten, Linear
from .transformer import LayerNorm, SelfAttention

__all__ = ["ReLU", "Sigmoid", "Softmax", "Tanh", "Sequential", "Dropout",
           "Flatten", "Linear", "LayerNorm", "SelfAttention"]
