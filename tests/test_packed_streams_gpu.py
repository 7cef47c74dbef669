"""The operators of a training step over packed documents on a stream of their own,
and captured into a graph that is replayed between eager work: the results of the
default stream's calls, every time."""
import ctypes

import numpy as np
import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd, amd_lm
from qutai_amd.lm import Packing, Rotary
from tests.helpers import download, normal, upload

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, LENGTHS = 8, 2, [70, 1, 0, 300, 33]
TOTAL = sum(LENGTHS)


class Stream:
    """Library calls inside go to this stream."""

    def __init__(self, runtime):
        self.runtime, self.hip, self.handle = runtime, runtime.hip, ctypes.c_void_p()
        self.check(self.hip.hipStreamCreate(ctypes.byref(self.handle)))

    def check(self, status):
        assert status == 0, status

    def __enter__(self):
        self.runtime.call = lambda name, *arguments, mfma=False: self.check(
            self.runtime._functions[name](*arguments, self.handle))
        return self

    def __exit__(self, *failure):
        del self.runtime.call

    def wait(self):
        self.check(self.hip.hipStreamSynchronize(self.handle))

    def close(self):
        self.check(self.hip.hipStreamDestroy(self.handle))


@pytest.fixture
def stream():
    runtime = amd.get_runtime()
    runtime.synchronize()
    made = Stream(runtime)
    yield made
    made.wait()
    made.close()


def operands(dim):
    width = (HEADS + 2 * KV_HEADS) * dim
    return dict(qkv=upload(normal(1, TOTAL * width), "bfloat16"), g=upload(normal(2, TOTAL * HEADS * dim), "bfloat16"),
                p=upload(normal(3, 5000), "float32"), pg=upload(normal(4, 5000), "float32"))


def step(x, dim, packing, turns, moments, workspace):
    """Every operator once; what it wrote."""
    width, wide = (HEADS + 2 * KV_HEADS) * dim, HEADS * dim
    columns = dict(q_row=width, k_column=wide, k_row=width)
    place = dict(v_column=wide + KV_HEADS * dim, v_row=width)
    q, k = amd_lm.rotary(x["qkv"], x["qkv"], turns, 1, TOTAL, HEADS, KV_HEADS, dim, positions=packing.positions, **columns)
    dims = (packing, HEADS, KV_HEADS, dim)
    out, lse, rest = amd_lm.attention_packed(q, k, x["qkv"], *dims, **place, rest=True)
    grads = amd_lm.attention_packed_backward(x["g"], q, k, x["qkv"], out, lse, *dims, **place, rest=rest)
    back = amd_lm.rotary(grads[0], grads[1], turns, 1, TOTAL, HEADS, KV_HEADS, dim, positions=packing.positions, inverse=True)
    norm = amd_lm.adamw([(x["p"], x["pg"], moments, 0)], moments.bits, 1e-2, 0.9, 0.99, 1e-8, 0.1, 3, max_norm=0.5,
                        workspace=workspace)
    return q, k, out, lse, rest, *grads, *back, norm


@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 32)])
def test_a_stream_of_its_own(stream, dim, bits):
    packing, turns = Packing(LENGTHS), Rotary(dim, layout="half")
    x, moments, workspace = operands(dim), amd_lm.AdamWMoments(5000, bits), amd_lm.adamw_workspace(1, 5000)
    start = x["p"].copy()
    expected = [download(y) for y in step(x, dim, packing, turns, moments, workspace)]
    after, held = download(x["p"]), [y.to_array() for y in moments.storages()]
    amd.copy_into(x["p"], start)
    again = amd_lm.AdamWMoments(5000, bits)
    amd.synchronize()
    with stream:
        found = step(x, dim, packing, turns, again, workspace)
        stream.wait()
    assert all(np.array_equal(a, download(b), equal_nan=True) for a, b in zip(expected, found))
    assert np.array_equal(after, download(x["p"])) and held == [y.to_array() for y in again.storages()]


@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 32)])
def test_replayed_graphs(stream, dim, bits):
    packing, turns = Packing(LENGTHS), Rotary(dim, layout="half")
    x, moments, workspace = operands(dim), amd_lm.AdamWMoments(5000, bits), amd_lm.adamw_workspace(1, 5000)
    start = x["p"].copy()
    # eager steps: what each replay has to give, and memory in the pool for the captured one
    expected = []
    for _ in range(3):
        found = step(x, dim, packing, turns, moments, workspace)
        expected.append(([download(y) for y in found], download(x["p"]), [y.to_array() for y in moments.storages()]))
    del found
    amd.copy_into(x["p"], start)
    again, hip = amd_lm.AdamWMoments(5000, bits), stream.hip
    amd.synchronize()
    graph, runner = ctypes.c_void_p(), ctypes.c_void_p()
    with stream:
        stream.check(hip.hipStreamBeginCapture(stream.handle, 2))
        try:
            found = step(x, dim, packing, turns, again, workspace)
        finally:
            status = hip.hipStreamEndCapture(stream.handle, ctypes.byref(graph))
        stream.check(status)
    stream.check(hip.hipGraphInstantiate(ctypes.byref(runner), graph, None, None, 0))
    for values, after, held in expected:
        stream.check(hip.hipGraphLaunch(runner, stream.handle))
        stream.wait()
        assert all(np.array_equal(a, download(b)) for a, b in zip(values, found))
        assert np.array_equal(after, download(x["p"])) and held == [y.to_array() for y in again.storages()]
        step(operands(dim), dim, packing, turns, amd_lm.AdamWMoments(5000, bits), amd_lm.adamw_workspace(1, 5000))  # eager
        amd.synchronize()
    stream.check(hip.hipGraphExecDestroy(runner))
    stream.check(hip.hipGraphDestroy(graph))


def test_steps_of_two_optimizers_between_each_other():
    from qutai_amd.optim import AdamW

    values = [normal(i, 700) for i in range(2)]
    alone, together = [], []
    for mixed in (False, True):
        parameters = [Tensor(upload(v, "float32"), shape=(700,), requires_grad=True) for v in values]
        optimizers = [AdamW([p], bits=8, max_norm=0.1, seed=i) for i, p in enumerate(parameters)]
        order = [0, 1, 0, 1, 1, 0] if mixed else [0, 0, 0, 1, 1, 1]
        for i in order:
            parameters[i].grad = Tensor(upload(normal(9 + i + 2 * optimizers[i].steps, 700), "float32"), shape=(700,))
            optimizers[i].step()
        (together if mixed else alone).extend(download(p.storage) for p in parameters)
    assert all(np.array_equal(a, b) for a, b in zip(alone, together))
