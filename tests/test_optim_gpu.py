"""AdamW at the ends of what it takes: the least eps, parameters of both types, a bad
gradient and the steps behind it."""
import numpy as np
import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd
from qutai_amd.optim import AdamW
from tests.helpers import download, normal, stored, upload
from tests.test_adamw_gpu import Model

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


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("bits,lost", [(32, slice(600, 601)), (8, slice(512, 768))])
def test_what_a_bad_gradient_costs_for_good(bits, lost, bad):
    """Without max_norm an infinity or NaN among the gradients takes its own value with
    moments of 32 bits, with 8 bits from the next step on all 256 that share its moments'
    exponent; every other value goes on to the bit as if that gradient had been 0."""
    runs = []
    for value in (bad, 0.0):
        p = Tensor(upload(normal(3, 1024), "float32"), shape=(1024,), requires_grad=True)
        optimizer = AdamW([p], bits=bits, seed=2)
        for step in range(3):
            g = normal(10 + step, 1024)
            if step == 0:
                g[600] = value
            p.grad = Tensor(upload(g, "float32"), shape=(1024,))
            optimizer.step()
        runs.append([download(p.storage), *(download(x.storage) for x in optimizer.moments(p))])
    expected = np.zeros(1024, bool)
    expected[lost] = True
    for i, (got, clean) in enumerate(zip(*runs)):
        if i == 0 or bits == 8 or np.isnan(bad):  # fp32's moments of an infinity are infinite: 0.9 inf and more
            assert np.array_equal(np.isnan(got), expected), i
        assert np.array_equal(got[~expected], clean[~expected]) and not np.isfinite(got[expected]).any()


@pytest.mark.parametrize("bits", [8, 32])
def test_parameters_of_both_types(bits):
    """float32 and bfloat16 tensors in one optimizer, whose norm is that of all gradients."""
    sizes, types = [700, 513, 3, 4096], ["float32", "bfloat16", "bfloat16", "float32"]
    values = [stored(normal(20 + i, n), t) for i, (n, t) in enumerate(zip(sizes, types))]
    parameters = [Tensor(upload(x, t), shape=x.shape, requires_grad=True) for x, t in zip(values, types)]
    options = dict(lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1, max_norm=0.5, seed=6)
    optimizer, model = AdamW(parameters, **options, bits=bits), Model(values, bits, **options)
    for step in range(2):
        given = [stored(normal(40 + 10 * step + i, n), t) for i, (n, t) in enumerate(zip(sizes, types))]
        for p, g, t in zip(parameters, given, types):
            p.grad = Tensor(upload(g, t), shape=p.shape)
        optimizer.step()
        norm = model.step(given)
        assert abs(optimizer.norm() - norm) <= 1e-12 * norm
        for i, (p, t) in enumerate(zip(parameters, types)):
            got, value = download(p.storage), model.p[i]
            # a dozen fp32 roundings of a quotient of some ten times lr at most, and the parameter's own
            bound = 40 * UNIT * (np.abs(value) + 10 * options["lr"]) + (2.0 ** -8 * np.abs(value) if t == "bfloat16" else 0)
            assert (np.abs(got - value) <= bound).all(), (step, i)
            model.p[i] = got.astype(np.float64)  # each step on its own
            first, second = (download(x.storage) for x in optimizer.moments(p))
            if bits == 8:
                assert np.array_equal(first, model.m[i]) and np.array_equal(second, model.v[i]), (step, i)
