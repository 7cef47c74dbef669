"""What an AdamW optimizer refuses before it touches the device: states of other
types and sizes, numbers that fp32 does not hold."""
from array import array
from types import SimpleNamespace

import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd_lm, amd_runtime
from qutai_amd.optim import AdamW
from tests.test_operators_host import built, fake

EINVAL = amd_runtime.QA_EINVAL

SIZES = (8, 300)


class Uploads:
    """A runtime that notes how many bytes it is told to write where."""

    def __init__(self):
        self.written = []

    def upload(self, ptr, buffer):
        self.written.append((ptr, memoryview(buffer).nbytes))

    def free(self, ptr):
        pass


@pytest.fixture(params=[32, 8])
def optimizer(request, monkeypatch):
    bits, runtime = request.param, Uploads()

    def moments(size, bits):
        words = [size] * 2 if bits == 32 else [(size + 7) // 8] * 2 + [(2 * ((size + 255) // 256) + 7) // 8]
        kept = [fake(n, "float32" if bits == 32 else "int64") for n in words]
        for x in kept:
            x.runtime = runtime
        return SimpleNamespace(size=size, bits=bits, storages=lambda: tuple(kept))

    monkeypatch.setattr(amd_lm, "AdamWMoments", moments)
    made = AdamW([Tensor(fake(n, "float32"), shape=(n,), requires_grad=True) for n in SIZES], bits=bits, seed=3)
    made.uploads = runtime
    return made


def state_of(optimizer, **change):
    kind = "f" if optimizer.bits == 32 else "q"
    moments = [[array(kind, bytes(x.nbytes)) for x in state.storages()] for state in optimizer._state]
    return {"steps": 5, "bits": optimizer.bits, "seed": 9, "moments": moments, **change}


def test_a_state_is_uploaded_whole(optimizer):
    optimizer.load_state_dict(state_of(optimizer))
    assert (optimizer.steps, optimizer.seed) == (5, 9)
    assert optimizer.uploads.written == [(x.ptr, x.nbytes) for s in optimizer._state for x in s.storages()]


@pytest.mark.parametrize("kind", ["d", "i", "H", "b", "other", list, bytes, memoryview])
def test_moments_of_another_item_type_write_nothing(optimizer, kind):
    """As many items of a wider type would be written past a moment's memory, of a narrower
    one leave part of it; the last tensor's last moment is wrong, so nothing of the others
    may have been written by then."""
    state = state_of(optimizer)
    last = state["moments"][-1][-1]
    if kind == "other":
        kind = "q" if optimizer.bits == 32 else "f"
    state["moments"][-1][-1] = array(kind, [0] * len(last)) if isinstance(kind, str) else kind(last)
    with pytest.raises(ValueError):
        optimizer.load_state_dict(state)
    assert not optimizer.uploads.written and (optimizer.steps, optimizer.seed) == (0, 3)


@pytest.mark.parametrize("change", [
    dict(steps=-1), dict(steps=2.0), dict(steps=True), dict(steps=1 << 63), dict(seed=-1), dict(seed=1 << 32), dict(seed=0.0),
    dict(seed=None), dict(bits=16), dict(moments=[]), dict(moments=None), dict(moments=[[], []]), dict(moments=[None, None])])
def test_states_of_other_optimizers_write_nothing(optimizer, change):
    with pytest.raises(ValueError):
        optimizer.load_state_dict(state_of(optimizer, **change))
    assert not optimizer.uploads.written and (optimizer.steps, optimizer.seed) == (0, 3)


@pytest.mark.parametrize("name", ["steps", "bits", "seed", "moments"])
def test_a_state_that_lacks_a_part_writes_nothing(optimizer, name):
    state = state_of(optimizer)
    del state[name]
    with pytest.raises(ValueError):
        optimizer.load_state_dict(state)
    assert not optimizer.uploads.written and (optimizer.steps, optimizer.seed) == (0, 3)


def test_moments_of_other_sizes_write_nothing(optimizer):
    for change in (lambda m: m[1].pop(), lambda m: m[1][-1].pop(), lambda m: m[1][-1].append(0), lambda m: m.reverse()):
        state = state_of(optimizer)
        change(state["moments"])
        with pytest.raises(ValueError):
            optimizer.load_state_dict(state)
    assert not optimizer.uploads.written and (optimizer.steps, optimizer.seed) == (0, 3)


LEAST, MOST = 2.0 ** -126, (2.0 - 2.0 ** -23) * 2.0 ** 127  # fp32's normal numbers


@pytest.mark.parametrize("eps", [5e-324, 7e-46, 1e-39, LEAST * (1 - 2.0 ** -52), 2.0 ** 128, 1e300, float("nan"), float("inf"), -1e-8])
def test_eps_that_fp32_does_not_hold_as_a_normal_number_is_refused(eps):
    """It would be 0 in the kernels (or its reciprocal infinite), and a value without a
    gradient 0 / 0."""
    parameter = Tensor(fake(8, "float32"), shape=(8,), requires_grad=True)
    with pytest.raises(ValueError):
        AdamW([parameter], eps=eps)


@built
def test_c_refuses_numbers_that_fp32_does_not_hold():
    """eps, the rate over 1 - beta1^step and the rate's decay are fp32 in the kernels."""
    import ctypes

    library, p = amd_runtime.load_library(), 4096
    row = (ctypes.c_int64 * 8)(p, p, p, p, p, 0, 0, 0)  # no values: nothing is launched

    def step(**change):
        a = dict(tensors=ctypes.addressof(row), count=1, bits=32, rate=1e-3, b1=0.9, b2=0.99, eps=1e-8, decay=0.0, step=1, seed=0,
                 max_norm=0.0, workspace=None, values=0, norm=None, stream=None)
        a.update(change)
        return library.qutai_amd_adamw(*a.values())

    for change in (dict(), dict(eps=LEAST), dict(eps=MOST), dict(rate=1e25), dict(rate=1e18, decay=1e20), dict(b1=1 - 2.0 ** -53, rate=1e20)):
        assert step(**change) == 0, change
    for change in (dict(eps=LEAST / 2), dict(eps=1e-46), dict(eps=2.0 ** 128), dict(eps=float("nan")),
                   dict(b1=1 - 2.0 ** -53, rate=1e25), dict(rate=1e19, decay=1e20)):
        assert step(**change) == EINVAL, change
