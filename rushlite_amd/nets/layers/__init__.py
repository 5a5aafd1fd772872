from .activation import ReLU, Sigmoid, Softmax, Tanh
from .container import Sequential
from .dropout import Dropout
from .linear import Flatten, Linear
from .transformer import (GatedFeedForward, GatedLinear, LayerNorm, RandomDropout, Rotary, SelfAttention, VocabularyLoss,
                          packed_positions, rotary_frequencies)

__all__ = ["ReLU", "Sigmoid", "Softmax", "Tanh", "Sequential", "Dropout",
           "Flatten", "Linear", "LayerNorm", "SelfAttention", "GatedFeedForward", "GatedLinear",
           "RandomDropout", "Rotary", "VocabularyLoss", "packed_positions", "rotary_frequencies"]
