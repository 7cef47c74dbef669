"""AdamW over the tensors of a model, in a few launches whatever their number."""
from __future__ import annotations

from array import array
from math import isfinite

from .backends import amd, amd_lm
from .core.tensor import Tensor


FP32_NORMAL = 2.0 ** -126, (2.0 - 2.0 ** -23) * 2.0 ** 127  # fp32's least and largest normal numbers


def _check_seed(seed):
    if type(seed) is not int or not 0 <= seed < 1 << 32:
        raise ValueError("the seed is an integer of 0 or more, below 2^32")


class AdamW:
    """``step()`` applies the gradients of ``parameters`` (float32 or bfloat16
    Tensors; those without a ``grad`` are left as they are):

        m' = beta1 m + (1 - beta1) g,  v' = beta2 v + (1 - beta2) g^2
        p' = p (1 - lr weight_decay) - lr m' / (1 - beta1^t) / (sqrt(v' / (1 - beta2^t)) + eps)

    ``bits`` 32 holds the moments in fp32, 8 in codes of 8 bits with an exponent
    for every 256 values, rounded up or down by chance (``seed``: the same run
    gives the same bits).  With ``max_norm`` gradients whose norm over all tensors
    exceeds it are scaled down to it, and a step whose norm is not finite changes
    nothing (t counts it all the same: nothing is read from the device); ``norm()``
    is the last step's.  Without it a gradient that is not finite makes its value NaN
    for good, and with 8 bits, from the next step on, all 256 values that share its
    moments' exponent.  ``lr`` may be changed between steps.  ``eps`` and each
    step's rate are fp32 in the kernels: eps is 2^-126 or more."""

    def __init__(self, parameters, lr=1e-3, *, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, bits=32, max_norm=None,
                 seed=0):
        parameters = tuple(dict.fromkeys(parameters))
        if not parameters or any(not isinstance(p, Tensor) or p.device != "amd" or p.dtype not in ("float32", "bfloat16")
                                 for p in parameters):
            raise ValueError("AdamW takes float32 or bfloat16 Tensors of the amd device")
        spans = sorted((p.storage.ptr, p.storage.ptr + p.storage.nbytes) for p in parameters if p.size)
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameters must not share memory: every value is stepped once")
        if bits not in (8, 32):
            raise ValueError("moments have 8 or 32 bits")
        _check_seed(seed)
        if len(betas) != 2 or any(not 0 <= b < 1 for b in betas):
            raise ValueError("betas lie in [0, 1)")
        if not FP32_NORMAL[0] <= eps <= FP32_NORMAL[1]:  # else 0 in the kernels, and a value without a gradient 0 / 0
            raise ValueError("eps is a normal number of fp32: 2^-126 (1.2e-38) or more")
        if max_norm is not None and not 0 < max_norm < float("inf"):
            raise ValueError("max_norm is a positive number")
        self.parameters, self.lr, self.betas, self.eps = parameters, lr, tuple(map(float, betas)), eps
        self.weight_decay, self.bits, self.max_norm, self.seed = weight_decay, bits, max_norm, seed
        self.steps = 0
        self._state = tuple(amd_lm.AdamWMoments(p.size, bits) for p in parameters)
        self._workspace = (None if max_norm is None else
                           amd_lm.adamw_workspace(len(parameters), sum(p.size for p in parameters)))
        self._norm = None

    def step(self):
        rate, decay = float(self.lr), float(self.weight_decay)
        if not (isfinite(rate) and rate >= 0 and isfinite(decay) and decay >= 0):
            raise ValueError("lr and weight_decay are numbers of 0 or more")
        tensors = [(p.storage, p.grad.storage, state, index)
                   for index, (p, state) in enumerate(zip(self.parameters, self._state)) if p.grad is not None]
        norm = amd_lm.adamw(tensors, self.bits, rate, *self.betas, self.eps, decay, self.steps + 1, seed=self.seed,
                            max_norm=self.max_norm, workspace=self._workspace)
        self.steps += 1
        self._norm = norm

    def norm(self):
        """The norm of all gradients of the last step, before it was cut (waits
        for the device); None without max_norm or before a step."""
        return None if self._norm is None else self._norm.tolist()[0]

    def zero_grad(self):
        for p in self.parameters:
            p.zero_grad()

    def _of(self, parameter):
        for p, state in zip(self.parameters, self._state):
            if p is parameter:
                return state
        raise ValueError("the optimizer does not hold this parameter")

    def moments(self, parameter):
        """(first, second) moments of one parameter as float32 Tensors: its own
        where they are held in 32 bits, the values that its codes stand for in 8."""
        state = self._of(parameter)
        return tuple(Tensor(x, shape=parameter.shape) for x in state.values())

    def state_dict(self):
        """Plain values (host arrays) from which ``load_state_dict`` goes on with
        the same bits."""
        return {"steps": self.steps, "bits": self.bits, "seed": self.seed,
                "moments": [[x.to_array() for x in state.storages()] for state in self._state]}

    def load_state_dict(self, state):
        """Goes on from a ``state_dict`` of an optimizer of the same tensors and bits;
        ValueError, and nothing changed, where it is not one."""
        try:
            steps, bits, seed, moments = (state[name] for name in ("steps", "bits", "seed", "moments"))
        except (KeyError, TypeError):
            raise ValueError("a state holds steps, bits, seed and moments") from None
        if bits != self.bits or not isinstance(moments, (list, tuple)) or len(moments) != len(self._state) \
                or type(steps) is not int or not 0 <= steps < (1 << 63) - 1:
            raise ValueError("the state is of another optimizer")
        _check_seed(seed)
        own = [state.storages() for state in self._state]
        for kept, given in zip(own, moments):
            if not isinstance(given, (list, tuple)) or len(given) != len(kept):
                raise ValueError("the state's moments are of another optimizer")
            # the items' type too: what is uploaded is as many bytes as the array has
            if any(not isinstance(values, array) or values.typecode != amd._TYPES[x.dtype][0] or len(values) != len(x)
                   for x, values in zip(kept, given)):
                raise ValueError("the state's moments are arrays of the sizes and item types of state_dict")
        for kept, given in zip(own, moments):
            for x, values in zip(kept, given):
                if len(x):
                    x.runtime.upload(x.ptr, values)
        self.steps, self.seed, self._norm = steps, seed, None
