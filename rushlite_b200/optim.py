"""Optimizers: AdamW (the reference has none; its users write the SGD update
themselves)."""
from __future__ import annotations

from typing import Any, Iterable

import numpy as np

from . import _C
from ._C import Variable


class AdamW:
    """Adam with decoupled weight decay, one kernel launch for all parameters.

    Parameters are updated in place, so a training step with it can be
    recorded in a ``cuda.Graph``: the step count lives on the device and
    advances with every replay (the rates are recorded as they were).  A
    recorded step reads the gradients' memory as of its capture: record
    ``zero_grad()`` and the backward with it, since ``zero_grad()`` outside
    gives the parameters gradients that the recorded step does not see.  Every
    parameter must be a CUDA Variable of one dtype, float32 or float64, that
    requires a gradient; its moments have its dtype.  A parameter without
    a gradient from ``backward()`` takes a step with a gradient of 0.
    """

    def __init__(self, params: Iterable[Variable], lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01) -> None:
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW: no parameters")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("AdamW: a parameter appears twice")
        kinds = {p.dtype for p in self.params}
        if len(kinds) != 1 or not kinds <= {_C.dtype.float32, _C.dtype.float64}:
            raise ValueError("AdamW: all parameters must be float32, or all float64")
        for p in self.params:
            if p.device != _C.device.cuda or not p.requires_grad:
                raise ValueError("AdamW: parameters must be CUDA Variables that require a gradient")
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.exp_avg = [self._zeros_like(p) for p in self.params]
        self.exp_avg_sq = [self._zeros_like(p) for p in self.params]
        self._step = Variable(np.zeros(2, np.int64), dtype=_C.dtype.int64)
        self._moments = [v.data for v in self.exp_avg], [v.data for v in self.exp_avg_sq]

    @staticmethod
    def _zeros_like(p: Variable) -> Variable:
        kind = np.float32 if p.dtype == _C.dtype.float32 else np.float64
        return Variable(np.zeros(p.shape, kind), dtype=p.dtype)

    def step(self) -> None:
        """Updates every parameter from its gradient."""
        b1, b2 = self.betas
        _C.adamw_step(self.params, self._moments[0], self._moments[1], self._step.data, self.lr, b1, b2, self.eps,
                      self.weight_decay)

    def zero_grad(self) -> None:
        for p in self.params:
            p.zero_grad()

    def state_dict(self) -> dict[str, Any]:
        """The steps taken and both moments, as NumPy arrays (waits for the GPU)."""
        return {"step": int(self._step.numpy()[0]), "exp_avg": [v.numpy() for v in self.exp_avg],
                "exp_avg_sq": [v.numpy() for v in self.exp_avg_sq]}

    def load_state_dict(self, state: dict[str, Any]) -> None:
        """Takes over what state_dict() gave, into the buffers that recorded graphs already use."""
        for name, mine in (("exp_avg", self.exp_avg), ("exp_avg_sq", self.exp_avg_sq)):
            theirs = [np.asarray(a) for a in state[name]]
            if [list(a.shape) for a in theirs] != [list(v.shape) for v in mine]:
                raise ValueError(f"AdamW: {name} does not match the parameters' shapes")
        if int(state["step"]) < 0:
            raise ValueError("AdamW: step must not be negative")
        for name, mine in (("exp_avg", self.exp_avg), ("exp_avg_sq", self.exp_avg_sq)):
            for v, a in zip(mine, state[name]):
                v.data.copy(Variable(np.asarray(a), dtype=v.dtype).data)
        self._step.data.copy(Variable(np.array([int(state["step"]), 0], np.int64), dtype=_C.dtype.int64).data)
