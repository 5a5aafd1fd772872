"""Random numbers on the device.

`Generator` is a counter-based generator whose count of calls lives on the device, so that a call recorded into an
`rsl.hip.Graph` draws afresh at every replay.  `dropout` keeps no mask: the backward pass forms it again from the call's
number.

    generator = rsl.Generator(seed=1)
    y = rsl.dropout(x, 0.1, generator, residual=r)      # r + what is kept of x / 0.9
"""
from __future__ import annotations

import numpy as np

from . import _C


class Generator:
    """What a call draws is a function of the seed and the number of the call."""

    def __init__(self, seed: int = 0, calls: int = 0):
        self.seed = int(seed) & 0xFFFFFFFFFFFFFFFF
        self._state = _C._Tensor(np.array([calls, 0], np.int64), [2], _C.device.hip, _C.dtype.int64)

    @property
    def calls(self) -> int:
        """Calls done, replays of recorded ones among them."""
        return int(self._state.numpy()[0])

    def state_dict(self) -> dict:
        return {"seed": self.seed, "calls": self.calls}

    def load_state_dict(self, state: dict) -> None:
        """In place: recorded calls go on from `calls`.  A recorded call keeps the seed it was recorded with."""
        self.seed = int(state["seed"]) & 0xFFFFFFFFFFFFFFFF
        self._state.copy(_C._Tensor(np.array([state["calls"], 0], np.int64), [2], _C.device.hip, _C.dtype.int64))


def dropout(x, rate: float, generator: Generator, residual=None):
    """residual + (kept ? x / (1 - rate) : 0): every value of x is dropped with probability `rate`."""
    return _C._dropout(x, residual, rate, generator.seed, generator._state)
