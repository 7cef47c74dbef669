"""AdamW at the ends of what it takes: the least eps, parameters of both types, a bad
gradient and the steps behind it."""
import numpy as np
import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd
from qutai_amd.optim import AdamW
from tests.helpers import download, normal, stored, upload

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24


@pytest.mark.parametrize("bits", [8, 32])
def test_the_least_eps_leaves_values_without_a_gradient(bits):
    """A zero gradient's update is 0 / (0 + eps) = 0 with fp32's least normal eps too, and
    the others' first step is lr times their gradient's sign (m / sqrt(v) within four fp32
    roundings, and the parameter's)."""
    start = normal(1, 600)
    g = np.where(np.arange(600) % 3, normal(2, 600), 0.0).astype(np.float32)
    p = Tensor(upload(start, "float32"), shape=(600,), requires_grad=True)
    p.grad = Tensor(upload(g, "float32"), shape=(600,))
    AdamW([p], lr=1e-2, eps=2.0 ** -126, weight_decay=0.0, bits=bits).step()
    after = download(p.storage)
    assert np.array_equal(after[::3], start[::3])
    expected = start.astype(np.float64) - 1e-2 * np.sign(g)
    assert (np.abs(after - expected) <= UNIT * (np.abs(expected) + 8 * 1e-2)).all()
