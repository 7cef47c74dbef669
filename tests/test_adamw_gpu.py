"""AdamW steps against their definition: moments of 32 bits within fp32's
roundings, codes of 8 bits to the bit; many tensors and few values, odd sizes and
addresses, bf16 parameters, clipped norms, missing gradients, saved states."""
from array import array

import numpy as np
import pytest

from oracle import reference as ora
from qutai_amd import Tensor
from qutai_amd.backends import amd
from qutai_amd.optim import AdamW
from tests.helpers import download, normal, stored, upload

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24
MASK = (1 << 32) - 1


def mixed(x):
    x = np.asarray(x, np.uint64) & np.uint64(MASK)
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0xBB67AE85)) & np.uint64(MASK)
    x ^= x >> np.uint64(13)
    x = (x * np.uint64(0x6A09E667)) & np.uint64(MASK)
    return x ^ (x >> np.uint64(16))


def rounding_bits(seed, step, tensor, count):
    key = mixed(mixed(mixed(seed) + np.uint64(step)) + np.uint64(tensor))
    bits = mixed(np.arange(count, dtype=np.uint64) * np.uint64(0x9E3779B9) + key)
    return (bits & np.uint64(0xFFFF)).astype(np.float64), (bits >> np.uint64(16)).astype(np.float64)


def held(values, bits, binades, positive):
    """What 8-bit codes with that many binades hold of float64 values."""
    out = np.zeros_like(values)
    for at in range(0, len(values), 256):
        x, b = np.abs(values[at:at + 256]), bits[at:at + 256]
        top = x.max()
        if not np.isfinite(top):
            out[at:at + 256] = np.nan
            continue
        fraction, exponent = np.frexp(top)
        E = max(int(exponent) - 1 + (fraction >= 0.9375), -64) if top > 0 else -64
        lowest = E - binades + 1
        mine = np.where(x > 0, np.maximum(np.frexp(x)[1] - 1, lowest), lowest)
        unit = np.ldexp(1.0, mine - 3)
        steps = np.floor(x / unit + b / 65536)
        if positive:
            steps = np.where((x > 0) & (steps == 0), 1, steps)
        out[at:at + 256] = np.where(values[at:at + 256] < 0, -1, 1) * steps * unit
    return out


class Model:
    """The definition in float64 (moments of 8 bits through their codes)."""

    def __init__(self, parameters, bits, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1, max_norm=None, seed=0):
        self.p = [p.astype(np.float64) for p in parameters]
        self.m, self.v = ([np.zeros(p.size) for p in parameters] for _ in range(2))
        self.size = [np.zeros(p.size) for p in parameters]  # of the terms that the first moment is a sum of
        self.bits, self.lr, self.betas, self.eps, self.decay = bits, lr, betas, eps, weight_decay
        self.max_norm, self.seed, self.t = max_norm, seed, 0

    def step(self, gradients):
        b1, b2 = self.betas
        self.t += 1
        norm = np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in gradients if g is not None))
        factor = self.max_norm / norm if self.max_norm and norm > self.max_norm else 1.0
        for i, g in enumerate(gradients):
            if g is None:
                continue
            g = g.astype(np.float64) * factor
            m, v = b1 * self.m[i] + (1 - b1) * g, b2 * self.v[i] + (1 - b2) * (g * g)
            update = m / (1 - b1 ** self.t) / (np.sqrt(v / (1 - b2 ** self.t)) + self.eps)
            self.p[i] = self.p[i] * (1 - self.lr * self.decay) - self.lr * update
            if self.bits == 8:
                low, high = rounding_bits(self.seed, self.t, i, g.size)
                m, v = held(m, low, 15, False), held(v, high, 31, True)
            self.m[i], self.v[i] = m, v
            self.size[i] = b1 * self.size[i] + (1 - b1) * np.abs(g)
        return norm


OPTIONS = dict(lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1)


def tensors(sizes, dtype, seed):
    values = [stored(normal(seed + i, n), dtype) for i, n in enumerate(sizes)]
    return values, [Tensor(upload(x, dtype), shape=(x.size,), requires_grad=True) for x in values]


def gradients(sizes, dtype, seed, parameters):
    found = []
    for i, (n, p) in enumerate(zip(sizes, parameters)):
        g = normal(seed + i, n, 10.0 ** -(i % 4)) * (np.random.default_rng(seed + i).random(n) < 0.8)
        g[n // 2:n // 2 + 300] = 0.0  # whole blocks of zeros
        g = stored(g, dtype)
        p.grad = Tensor(upload(g, dtype), shape=p.shape)
        found.append(g)
    return found


SIZES = [[1], [255], [256], [257, 3], [4096, 4097, 1], [70001, 5, 512, 12288], list(range(1, 120))]


@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_steps(sizes, dtype, bits, max_norm):
    values, parameters = tensors(sizes, dtype, 3)
    optimizer = AdamW(parameters, **OPTIONS, bits=bits, max_norm=max_norm, seed=11)
    model = Model(values, bits, **OPTIONS, max_norm=max_norm, seed=11)
    for t in range(3):
        given = gradients(sizes, dtype, 100 * (t + 1), parameters)
        optimizer.step()
        norm = model.step(given)
        if max_norm:
            assert abs(optimizer.norm() - norm) <= 1e-12 * norm
        for i, p in enumerate(parameters):
            got, before = download(p.storage), model.p[i]
            # update: a dozen fp32 roundings of a quotient that is at most some ten times lr, and the parameter's own
            assert np.abs(got - before).max() <= (40 * UNIT * (np.abs(before) + 10 * OPTIONS["lr"])).max() + (
                2.0 ** -8 * np.abs(before).max() if dtype == "bfloat16" else 0), (t, i)
            model.p[i] = got.astype(np.float64)  # each step on its own
            first, second = (download(x.storage) for x in optimizer.moments(p))
            if bits == 8:
                assert np.array_equal(first, model.m[i]) and np.array_equal(second, model.v[i]), (t, i)
            else:
                # a step multiplies a term by a constant (two roundings: its own and the product's; of a new term
                # the factor's and the clipped gradient's too) and rounds the sum, which is no larger than the sum
                # of the terms' magnitudes, however moments of two signs cancel: 5 roundings a step of that
                assert (np.abs(first - model.m[i]) <= 5 * UNIT * (t + 1) * model.size[i]).all(), (t, i)
                # all terms are positive; a square has its rounding and twice the clipped gradient's two
                assert (np.abs(second - model.v[i]) <= 8 * UNIT * (t + 1) * model.v[i] + 1e-38).all(), (t, i)


def test_views_at_odd_addresses():
    """Parameters, gradients and moments that are not 16-byte aligned."""
    block, grads = upload(normal(1, 3000), "float32"), upload(normal(2, 3000), "float32")
    spans = [(1, 700), (701, 2), (703, 1297)]
    parameters = [Tensor(amd.view(block, a, n), shape=(n,), requires_grad=True) for a, n in spans]
    for p, (a, n) in zip(parameters, spans):
        p.grad = Tensor(amd.view(grads, a, n), shape=(n,))
    before, given = download(block).astype(np.float64), download(grads)
    for bits in (32, 8):
        model = Model([download(block)[a:a + n] for a, n in spans], bits, **OPTIONS, seed=0)
        AdamW(parameters, **OPTIONS, bits=bits).step()
        model.step([given[a:a + n] for a, n in spans])
        after = download(block)
        for (a, n), value in zip(spans, model.p):
            assert np.abs(after[a:a + n] - value).max() <= 1e-5
    assert after[0] == before[0] and np.array_equal(after[2000:], before[2000:])


def test_missing_gradients_and_empty_tensors():
    values, parameters = tensors([10, 0, 300], "float32", 5)
    parameters[2].grad = Tensor(upload(normal(1, 300), "float32"), shape=(300,))
    parameters[1].grad = Tensor(amd.AMDStorage(0, "float32"), shape=(0,))
    for bits in (8, 32):
        optimizer = AdamW(parameters, bits=bits, max_norm=1.0)
        optimizer.step()
        assert np.array_equal(download(parameters[0].storage), values[0])
        assert not np.array_equal(download(parameters[2].storage), values[2])
        assert abs(optimizer.norm() - np.linalg.norm(normal(1, 300).astype(np.float64))) <= 1e-9
    optimizer.zero_grad()
    after = download(parameters[2].storage)
    optimizer.step()
    assert optimizer.norm() == 0.0 and np.array_equal(download(parameters[2].storage), after)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_norm_that_is_not_finite_leaves_everything(bits):
    values, parameters = tensors([300, 20], "float32", 7)
    optimizer = AdamW(parameters, bits=bits, max_norm=1.0)
    gradients([300, 20], "float32", 9, parameters)
    optimizer.step()
    before = [download(p.storage) for p in parameters] + [x.tolist() for p in parameters for x in optimizer.moments(p)]
    for bad in (np.nan, np.inf):
        given = gradients([300, 20], "float32", 10, parameters)
        given[1][3] = bad
        parameters[1].grad = Tensor(upload(given[1], "float32"), shape=(20,))
        optimizer.step()
        assert not np.isfinite(optimizer.norm())
        after = [download(p.storage) for p in parameters] + [x.tolist() for p in parameters for x in optimizer.moments(p)]
        assert all(np.array_equal(a, b) for a, b in zip(before, after))


def test_without_a_norm_a_bad_gradient_is_kept_to_its_place():
    for bits, spoiled in ((32, slice(600, 601)), (8, slice(512, 768))):
        _, parameters = tensors([1024], "float32", 7)
        g = normal(1, 1024)
        g[600] = np.nan
        parameters[0].grad = Tensor(upload(g, "float32"), shape=(1024,))
        optimizer = AdamW(parameters, bits=bits)
        optimizer.step()
        moments = download(optimizer.moments(parameters[0])[0].storage)
        bad = np.zeros(1024, bool)
        bad[spoiled] = True  # 8 bits: the block that shares its exponent
        assert np.array_equal(np.isnan(moments), bad)
        assert np.array_equal(np.isnan(download(parameters[0].storage)), np.arange(1024) == 600)


@pytest.mark.parametrize("scale", [1e-30, 1e-20, 1e18])
def test_extreme_gradients_in_8_bits(scale):
    """Values below the least exponent become zeros, large ones keep codes."""
    values, parameters = tensors([1000], "float32", 13)
    optimizer, model = AdamW(parameters, **OPTIONS, bits=8), Model(values, 8, **OPTIONS)
    for t in range(2):
        g = stored(normal(t + 1, 1000, scale), "float32")
        parameters[0].grad = Tensor(upload(g, "float32"), shape=(1000,))
        optimizer.step()
        model.step([g])
        first, second = (download(x.storage) for x in optimizer.moments(parameters[0]))
        assert np.array_equal(first, model.m[0].astype(np.float32)) and np.array_equal(second, model.v[0].astype(np.float32))
        assert np.isfinite(download(parameters[0].storage)).all()


def test_moments_of_8_bits_follow_small_changes():
    """With beta2 = 0.99 a step changes the second moment by 1%, a code is 6 to
    12%: rounded to nearest it would stay.  After 400 steps of gradients 1 the mean
    over 64 blocks is that of the definition; a code's rounding has a variance of at
    most 0.0125 steps of 0.125 a step, damped by 0.99 (deviation 0.04 for a value
    of 1), so the mean over 16384 is within 0.04 / 128 * 5 of 1 - 0.99^400, and
    after 400 more steps of gradients 0.5 within that of its value."""
    _, parameters = tensors([16384], "float32", 15)
    optimizer = AdamW(parameters, lr=0.0, betas=(0.9, 0.99), bits=8)
    target = 0.0
    for g in (1.0, 0.5):
        parameters[0].grad = Tensor(amd.full(16384, g, dtype="float32"), shape=(16384,))
        for _ in range(400):
            optimizer.step()
            target = 0.99 * target + 0.01 * g * g
        second = download(optimizer.moments(parameters[0])[1].storage).astype(np.float64)
        assert abs(second.mean() - target) <= 5 * second.std() / 128 + 1e-6 and second.std() <= 0.3 * target


@pytest.mark.parametrize("bits", [8, 32])
def test_saved_states_go_on_with_the_same_bits(bits):
    sizes = [700, 3]
    _, parameters = tensors(sizes, "float32", 21)
    optimizer = AdamW(parameters, **OPTIONS, bits=bits, seed=4)
    for t in range(2):
        gradients(sizes, "float32", 50 + t, parameters)
        optimizer.step()
    state, weights = optimizer.state_dict(), [download(p.storage) for p in parameters]
    others = [Tensor(upload(w, "float32"), shape=w.shape, requires_grad=True) for w in weights]
    second = AdamW(others, **OPTIONS, bits=bits)
    second.load_state_dict(state)
    for p, o in zip(parameters, others):
        o.grad = p.grad
    optimizer.step()
    second.step()
    assert all(np.array_equal(download(p.storage), download(o.storage)) for p, o in zip(parameters, others))
    assert all(a.to_array() == b.to_array() for s, t in zip(optimizer._state, second._state)
               for a, b in zip(s.storages(), t.storages()))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_tensor_beyond_32_bits(bits):
    """Equal values behind element 2^32 are stepped as those at the beginning (the rounding's
    hash takes an element's low 32 bits); the norm counts all of them."""
    size, steps = (1 << 32) + 4096, 2
    p = Tensor(amd.full(size, 0.5, dtype="float32"), shape=(size,), requires_grad=True)
    p.grad = Tensor(amd.full(size, 2.0 ** -10, dtype="float32"), shape=(size,))
    optimizer = AdamW([p], **OPTIONS, bits=bits, max_norm=1.0, seed=5)
    for _ in range(steps):
        optimizer.step()
    assert abs(optimizer.norm() - 2.0 ** -10 * size ** 0.5) <= 1e-9 * optimizer.norm()
    state = optimizer._of(p)
    if bits == 8:  # bytes, seen as words of eight
        ends = [(x, size // 8 - 512, 512) for x in (state.first, state.second)] + [(state.exponents, size // 128 // 8 - 4, 4)]
    else:
        ends = [(x, size - 4096, 4096) for x in (state.first, state.second)]
    for x, start, count in [(p.storage, size - 4096, 4096), *ends]:
        first, last = (amd.view(x, at, count).to_array() for at in (0, start))
        assert first == last and any(first)
    model = Model([np.full(4096, 0.5, np.float32)], bits, **OPTIONS, seed=5)
    for _ in range(steps):
        model.step([np.full(4096, 2.0 ** -10 / (2.0 ** -10 * size ** 0.5))])
    assert np.abs(download(amd.view(p.storage, 0, 4096)) - model.p[0]).max() <= 40 * UNIT * (0.5 + 10 * OPTIONS["lr"])
