"""Optimizers over a model's parameters.

`AdamW` updates every parameter's buffer in place in one kernel.  Its states take 32 bits a value, or 8 bits in blocks of
256 that share a scale, rounded at random without bias.  The count of steps lives on the device, so a step recorded into
an `rsl.hip.Graph` advances it at every replay.

    opt = rsl.optim.AdamW(model, lr=1e-3, bits=8)
    loss.backward()
    opt.step()
    opt.zero_grad()
"""
from __future__ import annotations

import numpy as np

from . import _C
from .nets.Module import Module

_BLOCK = 256


def _tensor(array):
    return _C._Tensor(array, list(array.shape), _C.device.hip, getattr(_C.dtype, array.dtype.name))


class AdamW:
    """p = p (1 - lr weight_decay) - lr m^ / (sqrt(v^) + eps), with m and v the running means of the gradient and its
    square and m^, v^ corrected for their start at zero.

    `params`: a Module, whose frozen parameters (requires_grad off) are left as they are, or an iterable of Variables with
    requires_grad; float32 on the HIP device.  A Variable that comes more than once, as those of a shared layer do, is one
    parameter.  `weight_decay`: a number, or a function of a parameter that returns one (biases and norms are often left
    out).  `bits`: 32 or 8.
    `seed` chooses the random bits that 8-bit states are rounded with."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=32, seed=0):
        if bits not in (8, 32):
            raise ValueError(f"AdamW: states have 32 or 8 bits, not {bits}")
        found, memory = {}, {}
        if isinstance(params, Module):
            params = [p for p in params.parameters() if p.requires_grad]
        for i, p in enumerate(params):
            if not isinstance(p, _C.Variable) or not p.requires_grad:
                raise ValueError(f"AdamW: parameter {i} is not a Variable that requires a gradient")
            if _C._variable_id(p) in found:
                continue
            found[_C._variable_id(p)] = i, p
            p.realize()
            if np.prod(p.shape) and (other := memory.setdefault(_C._storage_ptr(p.data), i)) != i:
                raise ValueError(f"AdamW: parameters {other} and {i} are different Variables over the same memory")
        for i, p in found.values():
            if p.dtype != _C.dtype.float32 or p.device != _C.device.hip:
                raise ValueError(f"AdamW: parameter {i} is not float32 on the HIP device")
        self.params = [p for _, p in found.values()]
        self.lr, self.betas, self.eps, self.bits, self.seed = lr, tuple(betas), eps, bits, int(seed)
        decay = weight_decay if callable(weight_decay) else lambda p: weight_decay
        self._decay = [float(decay(p)) for p in self.params]
        self._step = _tensor(np.zeros(2, np.int64))
        self._states = [self._fresh(int(np.prod(p.shape, dtype=np.int64))) for p in self.params]

    def _fresh(self, n):
        if self.bits == 32:
            return tuple(_C.zeros([n]).data for _ in range(2)) + (None, None)
        codes, blocks = -(-n // 4), -(-n // _BLOCK)
        return (tuple(_C.zeros([codes], dtype=_C.dtype.int32).data for _ in range(2))
                + tuple(_C.zeros([blocks]).data for _ in range(2)))

    @property
    def steps(self) -> int:
        """Steps done, replays of recorded ones among them."""
        return int(self._step.numpy()[0])

    def step(self) -> None:
        """One update by the parameters' gradients (a gradient that was never formed is zero)."""
        _C._adamw(self.bits, [(p.data, p.grad, *s, d) for p, s, d in zip(self.params, self._states, self._decay)],
                  self.lr, *self.betas, self.eps, self.seed & 0xFFFFFFFFFFFFFFFF, self._step)

    def zero_grad(self) -> None:
        for p in self.params:
            p.zero_grad()

    def moments(self, i: int):
        """The first and second moment of parameter i as arrays of its shape."""
        p, (m, v, ms, vs) = self.params[i], self._states[i]
        if self.bits == 8:
            n = int(np.prod(p.shape, dtype=np.int64))
            m, v = _C._adamw_decode(True, m, ms, n), _C._adamw_decode(False, v, vs, n)
        return m.numpy().reshape(p.shape), v.numpy().reshape(p.shape)

    def state_dict(self) -> dict:
        """What a later run needs to go on: arrays, as they are held."""
        return {"bits": self.bits, "seed": self.seed, "step": self._step.numpy(),
                "states": [[None if t is None else t.numpy() for t in s] for s in self._states]}

    def load_state_dict(self, state: dict) -> None:
        held = state["states"]
        if state["bits"] != self.bits or len(held) != len(self._states):
            raise ValueError("AdamW: the state is of other parameters or another number of bits")
        for i, (mine, other) in enumerate(zip(self._states, held)):
            for t, a in zip(mine, other):
                if (t is None) != (a is None) or (t is not None and list(t.shape) != list(np.shape(a))):
                    raise ValueError(f"AdamW: the state of parameter {i} does not fit it")
        self.seed = int(state["seed"])
        # in place: a recorded step goes on reading the same buffers
        self._step.copy(_tensor(np.asarray(state["step"], np.int64)))
        for mine, other in zip(self._states, held):
            for t, a in zip(mine, other):
                if t is not None and np.size(a):
                    t.copy(_tensor(np.ascontiguousarray(a)))
