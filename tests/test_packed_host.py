"""Packings, rotary frequencies and the refusals of the operators of a training
step over packed documents, before any device call."""
from math import log, pi
from pathlib import Path
from types import SimpleNamespace

import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd, amd_lm, amd_runtime
from qutai_amd.lm import Config, Packing, Rotary
from qutai_amd.lm.layers import attention, rotary
from qutai_amd.optim import AdamW
from tests.test_operators_host import LIBRARY, built, fake

EINVAL, EWORKSPACE = amd_runtime.QA_EINVAL, amd_runtime.QA_EWORKSPACE


def test_packing_places(monkeypatch):
    monkeypatch.setattr(amd, "storage", lambda values, dtype: list(values))
    packing = Packing([3, 0, 300, 1], total=310)
    assert (packing.starts, packing.used, packing.total, packing.longest) == ((0, 3, 3, 303), 304, 310, 300)
    lengths_at = {0: 3, 3: 300, 303: 1}

    def tiles(rows, order):
        table, count = packing.tiles(rows, order)
        found = [(word & 0xFFFFFFFF, word >> 32, n) for word, n in zip(table[:count], table[count:])]
        assert len(table) == 2 * count and all(lengths_at[start] == n for start, _, n in found)
        return found

    for rows in (4, 32, 64, 128, 256):
        for order in ("end", "start", "length"):
            found = tiles(rows, order)
            covered = [start + t for start, first, n in found for t in range(first, min(first + rows, n))]
            assert sorted(covered) == list(range(304)) and all(first % rows == 0 for _, first, _ in found)
    assert [first for _, first, _ in tiles(128, "end")] == [256, 128, 0, 0, 0]
    assert [(start, first) for start, first, _ in tiles(128, "start")] == [(3, 0), (3, 128), (3, 256), (0, 0), (303, 0)]
    assert [start for start, _, _ in tiles(128, "length")] == [3, 3, 3, 0, 303]


def test_packing_of_large_starts(monkeypatch):
    monkeypatch.setattr(amd, "storage", lambda values, dtype: list(values))
    table, count = Packing([1 << 30, 5]).tiles(1 << 29, "end")
    assert [(w & 0xFFFFFFFF, w >> 32) for w in table[:count]] == [(0, 1 << 29), (0, 0), (1 << 30, 0)]


def test_positions_that_failed_are_made_again(monkeypatch):
    """Positions whose kernel could not be sent (an upload inside a capture) are not
    kept as if they were there."""
    packing, sent = Packing([2, 3]), []
    block, starts = fake(5, "int64"), fake(2, "int64")
    block.runtime.call = lambda name, *arguments: sent.append(name)
    monkeypatch.setattr(amd, "AMDStorage", lambda size, dtype: block)

    def failing(values, dtype):
        raise RuntimeError("no upload here")

    monkeypatch.setattr(amd, "storage", failing)
    for _ in range(2):
        with pytest.raises(RuntimeError):
            packing.positions
    monkeypatch.setattr(amd, "storage", lambda values, dtype: starts)
    assert packing.positions is block and packing.positions is block and sent == ["qutai_amd_positions"]


@pytest.mark.parametrize("lengths,total", [([-1], None), ([1.0], None), ([True], None), ([4], 3), ([1 << 31], None),
                                           ([2], 2.0)])
def test_packing_refusals(lengths, total):
    with pytest.raises(ValueError):
        Packing(lengths, total)


def test_rotary_frequencies():
    plain = Rotary(64)
    assert plain.frequencies[0] == 1.0 and abs(plain.frequencies[31] - 10000.0 ** (-62 / 64)) < 1e-18
    assert plain.magnitude == 1.0 and plain.rotary_dim == 64
    halves = Rotary(64, scaling={"kind": "linear", "factor": 2.0})
    assert all(a == b / 2 for a, b in zip(halves.frequencies, plain.frequencies))
    base = Rotary(64, scaling={"kind": "base", "factor": 8.0})
    assert base.frequencies[0] == 1.0 and abs(base.frequencies[31] * 8 / plain.frequencies[31] - 1) < 1e-12
    parts = Rotary(64, scaling={"kind": "parts", "factor": 8.0, "original_length": 1024})
    assert abs(parts.magnitude - (0.1 * log(8.0) + 1)) < 1e-15
    for f, p in zip(plain.frequencies, parts.frequencies):
        turns = 1024 * f / (2 * pi)
        assert p == f if turns >= 32 else p <= f
        assert abs(p * 8 / f - 1) < 1e-12 if turns <= 1 else p > f / 8


@pytest.mark.parametrize("change", [
    dict(dim=0), dict(dim=258), dict(dim=64.0), dict(rotary_dim=3), dict(rotary_dim=66), dict(rotary_dim=0), dict(layout="other"),
    dict(theta=0), dict(theta=float("inf")), dict(scaling="linear"), dict(scaling={"kind": "other", "factor": 2}),
    dict(scaling={"kind": "linear"}), dict(scaling={"kind": "linear", "factor": 0}),
    dict(scaling={"kind": "linear", "factor": 2, "low": 1}), dict(scaling={"kind": "parts", "factor": 2}),
    dict(scaling={"kind": "parts", "factor": 2, "original_length": 8, "low": 4, "high": 4}),
    dict(scaling={"kind": "parts", "factor": 2, "original_length": 8, "magnitude": 0}),
    dict(rotary_dim=2, scaling={"kind": "base", "factor": 2})])
def test_rotary_refusals(change):
    with pytest.raises(ValueError):
        Rotary(**{"dim": 64, **change})


def test_configurations():
    plain = Config()
    assert plain.rotary() is None and not {"rope_layout", "rope_dim", "rope_scaling"} & set(plain.to_dict())
    other = Config(rope_layout="half", rope_dim=32, rope_scaling={"kind": "linear", "factor": 2.0})
    assert Config(**other.to_dict()) == other and other.rotary().rotary_dim == 32
    for change in (dict(rope_layout="x"), dict(rope_dim=31), dict(rope_dim=128), dict(rope_scaling={"kind": "x"})):
        with pytest.raises(ValueError):
            Config(**change)


def rotary_call(**change):
    a = dict(q=fake(6 * 4 * 8, "bfloat16"), k=fake(6 * 2 * 8, "bfloat16"), rotary=Rotary(8), batch=2, time=3, heads=4,
             kv_heads=2, dim=8)
    a.update(change)
    return amd_lm.rotary(**a)


@pytest.mark.parametrize("change", [
    dict(dim=16), dict(heads=0, kv_heads=0), dict(time=-1), dict(q=fake(8, "bfloat16")), dict(q=fake(192, "float32")),
    dict(q=fake(192, "float64"), k=fake(96, "float64")), dict(q_row=31), dict(q_column=1), dict(k_column=-1),
    dict(positions=fake(6, "float32")), dict(positions=fake(5, "int64")), dict(positions=fake(6, "int64"), offset=1),
    dict(positions=fake(6, "int64"), starts=fake(2, "int64")), dict(starts=fake(3, "int64")), dict(inverse=2),
    dict(out=fake(6 * 40, "bfloat16"), out_row=40), dict(out=fake(6 * 48, "bfloat16"), out_row=48, out_k_column=31),
    dict(out=fake(6 * 48, "float32"), out_row=48)])
def test_rotary_operator_refusals(change):
    with pytest.raises(ValueError):
        rotary_call(**change)


def test_rotary_refuses_a_moved_result_in_its_input():
    block = fake(6 * 64, "bfloat16")
    with pytest.raises(ValueError):
        rotary_call(q=block, k=block, q_row=64, k_column=32, k_row=64, out=block, out_row=64, out_q_column=8, out_k_column=40)


def packed_call(backward=False, **change):
    packing = change.pop("packing", Packing([2, 4]))
    a = dict(q=fake(6 * 32, "bfloat16"), k=fake(6 * 16, "bfloat16"), v=fake(6 * 16, "bfloat16"), packing=packing, heads=4,
             kv_heads=2, dim=8)
    if backward:
        a.update(gradient=fake(6 * 32, "bfloat16"), out=fake(6 * 32, "bfloat16"), lse=fake(24, "float32"))
    a.update(change)
    return (amd_lm.attention_packed_backward if backward else amd_lm.attention_packed)(**a)


WRONG = [dict(dim=0), dict(dim=264), dict(heads=3), dict(kv_heads=0), dict(q=fake(6 * 32 - 1, "bfloat16")),
         dict(v=fake(6 * 16, "float32")), dict(q=fake(192, "int64"), k=fake(96, "int64"), v=fake(96, "int64")),
         dict(packing=Packing([2, 5])), dict(q_row=31), dict(k_column=1), dict(v_column=-8)]


@pytest.mark.parametrize("change", WRONG)
def test_packed_attention_refusals(change):
    with pytest.raises(ValueError):
        packed_call(**change)


@pytest.mark.parametrize("change", WRONG + [
    dict(gradient=fake(6 * 32, "float32")), dict(gradient=fake(6 * 31, "bfloat16")), dict(lse=fake(24, "bfloat16")),
    dict(lse=fake(23, "float32")), dict(out=fake(6, "bfloat16")), dict(into=fake(6 * 64, "bfloat16")),
    dict(rest=fake(6, "bfloat16")), dict(rest=fake(6 * 32, "float32"))])
def test_packed_backward_refusals(change):
    with pytest.raises(ValueError):
        packed_call(True, **change)


def test_packed_backward_refuses_overlaps():
    block = fake(6 * 64, "bfloat16")
    place = dict(q=block, k=block, v=block, q_row=64, k_column=32, k_row=64, v_column=48, v_row=64)
    with pytest.raises(ValueError):
        packed_call(True, **place, into=block)
    with pytest.raises(ValueError):  # columns that share values
        packed_call(True, **{**place, "v_column": 40}, into=fake(6 * 64, "bfloat16"))


def test_layer_functions_refuse_shapes():
    q, k = (Tensor(fake(6 * n, "float32"), shape=(1, 6, n)) for n in (32, 16))
    with pytest.raises(ValueError):
        attention(q, k, k, 4, 2, Packing([3, 4]))
    with pytest.raises(ValueError):
        rotary(q, q, 4, 2, Rotary(8))


def parameter(size=8, dtype="float32"):
    return Tensor(fake(size, dtype), shape=(size,), requires_grad=True)


@pytest.mark.parametrize("change", [
    dict(parameters=[]), dict(parameters=[parameter(dtype="float64")]), dict(parameters=[1.0]), dict(bits=16),
    dict(seed=-1), dict(seed=1 << 32), dict(seed=1.0), dict(betas=(0.9,)), dict(betas=(1.0, 0.9)), dict(eps=0),
    dict(max_norm=0), dict(max_norm=float("inf"))])
def test_adamw_refusals(change):
    with pytest.raises(ValueError):
        AdamW(**{"parameters": [parameter()], **change})


def test_adamw_refuses_parameters_that_share_memory(monkeypatch):
    monkeypatch.setattr(amd_lm, "AdamWMoments", lambda size, bits: SimpleNamespace(size=size, bits=bits))
    p, inside, behind = parameter(64), fake(8, "float32"), fake(8, "float32")
    inside.ptr, behind.ptr = p.storage.ptr + 4 * 60, p.storage.ptr + 4 * 64
    with pytest.raises(ValueError):
        AdamW([p, Tensor(p.storage, shape=(64,), requires_grad=True)])
    with pytest.raises(ValueError):
        AdamW([Tensor(inside, shape=(8,), requires_grad=True), p])
    assert len(AdamW([p, Tensor(behind, shape=(8,), requires_grad=True), p]).parameters) == 2  # the same one once


def test_adamw_step_refusals(monkeypatch):
    monkeypatch.setattr(amd_lm, "AdamWMoments", lambda size, bits: SimpleNamespace(size=size, bits=bits))
    p = parameter()
    optimizer = AdamW([p])
    for grad in (fake(7, "float32"), fake(8, "bfloat16")):  # other sizes, other types
        p.grad = Tensor(grad, shape=(grad.size,))
        with pytest.raises(ValueError):
            optimizer.step()
    p.grad = Tensor(fake(8, "float32"), shape=(8,))
    for lr in (-1.0, float("nan"), float("inf")):
        optimizer.lr = lr
        with pytest.raises(ValueError):
            optimizer.step()
    assert optimizer.steps == 0
    with pytest.raises(ValueError):
        optimizer.moments(parameter())


@built
def test_c_entry_points_refuse():
    """The C entry points' own checks (pointers that are never followed)."""
    import ctypes

    library, p = amd_runtime.load_library(), 4096
    turns = (ctypes.c_double * 4)(1, 1, 1, 1)

    def turn(**change):
        a = dict(q=p, k=p, qo=p, ko=p, turns=ctypes.addressof(turns), positions=None, starts=None, offset=0, batch=2, time=3,
                 heads=4, kv=2, dim=8, rotary=8, qr=32, kr=16, qor=32, kor=16, half=1, magnitude=1.0, inverse=0, dtype=5,
                 stream=None)
        a.update(change)
        return library.qutai_amd_rotary(*a.values())

    for change in (dict(batch=-1), dict(heads=0, kv=0), dict(dim=258), dict(dim=0), dict(rotary=7), dict(rotary=10),
                   dict(turns=None), dict(dtype=1), dict(magnitude=0.0), dict(magnitude=float("nan")), dict(qr=31),
                   dict(kor=15), dict(q=None), dict(ko=None), dict(batch=1 << 30, time=4)):
        assert turn(**change) == EINVAL, change
    assert turn(batch=0) == 0

    for wrong in ((None, 1, 5, 5, p), (p, 0, 5, 5, p), (p, 1, 6, 5, p), (p, 1, -1, 5, p), (p, 1, 5, 1 << 31, p), (p, 1, 5, 5, None)):
        assert library.qutai_amd_positions(*wrong, None) == EINVAL, wrong
    assert library.qutai_amd_positions(None, 0, 0, 0, None, None) == 0

    def forward(**change):
        a = dict(q=p, k=p, v=p, out=p, lse=p, rest=None, tiles=p, count=2, rows=64, tokens=200, sequences=3, longest=1000, heads=4, kv=2, dim=64, qr=256, kr=128,
                 vr=128, dtype=5, scale=0.125, causal=1, stream=None)
        a.update(change)
        return library.qutai_amd_attention_packed_fwd(*a.values())

    wrong = (dict(heads=3), dict(kv=0), dict(dim=0), dict(dim=264), dict(qr=255), dict(kr=127), dict(vr=64), dict(dtype=4),
             dict(scale=0.0), dict(scale=float("nan")), dict(rows=100), dict(rows=0), dict(q=None), dict(lse=None),
             dict(tiles=None), dict(count=-1), dict(count=1 << 40), dict(tokens=-1), dict(sequences=-1), dict(longest=-1), dict(tokens=1 << 31), dict(q=p + 2), dict(qr=1 << 30), dict(dim=20))
    for change in wrong:
        assert forward(**change) == EINVAL, change
    assert forward(count=0) == 0
    assert forward(rest=p, dim=136, qr=544, kr=272, vr=272) == EINVAL and forward(rest=p, rows=4) == EINVAL
    for dtype, dim, rows in ((5, 20, 4), (0, 160, 4), (0, 64, 128), (5, 64, 64)):
        assert library.qutai_amd_attention_packed_rows(50000, 9, 1000, 4, 2, dim, dtype, 1, 0.1, 0) == rows
    assert library.qutai_amd_attention_packed_rows(50000, 9, 1000, 4, 2, 64, 5, 0, 0.1, 0) == 4
    assert library.qutai_amd_attention_packed_rows(50000, 9, 1000, 4, 2, 64, 4, 1, 0.1, 0) == 0

    row = (ctypes.c_int64 * 8)(p, p, p, p, p, 8, 0, 0)

    def step(values=None, **change):
        table = (ctypes.c_int64 * 8)(*(values or row))
        a = dict(tensors=ctypes.addressof(table), count=1, bits=32, rate=1e-3, b1=0.9, b2=0.99, eps=1e-8, decay=0.0, step=1,
                 seed=0, max_norm=0.0, workspace=None, values=0, norm=None, stream=None)
        a.update(change)
        return library.qutai_amd_adamw(*a.values())

    for change in (dict(bits=16), dict(b1=1.0), dict(b2=-0.1), dict(eps=0.0), dict(step=0), dict(rate=-1.0),
                   dict(rate=float("nan")), dict(decay=-1.0), dict(max_norm=-1.0), dict(count=-1), dict(tensors=None),
                   dict(values=(0, p, p, p, p, 8, 0, 0)), dict(values=(p, 0, p, p, p, 8, 0, 0)),
                   dict(values=(p, p, p, p, 0, 8, 0, 0), bits=8), dict(values=(p, p, p, p, p, -1, 0, 0)),
                   dict(values=(p, p, p, p, p, 8, 4, 0)), dict(values=(p + 1, p, p, p, p, 8, 0, 0)),
                   dict(values=(p, p, p + 2, p, p, 8, 0, 0))):
        assert step(**change) == EINVAL, change
    assert step(max_norm=1.0) == EWORKSPACE
    assert step(values=(0, 0, 0, 0, 0, 0, 0, 0)) == 0 and step(count=0) == 0
    assert library.qutai_amd_adamw_workspace(-1, 8) == 0 and library.qutai_amd_adamw_workspace(49, 8) == 2048
    assert library.qutai_amd_adamw_moments(p, p, None, p, p, 8, None) == EINVAL
    assert library.qutai_amd_adamw_moments(p, p, p, p, p, -1, None) == EINVAL


@built
def test_workspace_of_the_key_pass():
    """Asked for where a group's heads work side by side: fp32 or wide bf16 heads that
    share keys, few key tiles; nothing for sizes that are none."""
    import ctypes

    library = ctypes.CDLL(str(LIBRARY))
    ask = library.qutai_amd_attention_packed_workspace
    ask.restype, ask.argtypes = ctypes.c_size_t, amd_runtime.SIGNATURES["qutai_amd_attention_packed_workspace"]
    assert ask(1000, 3, 8, 2, 64, 0, 128) == 2 * 4 * 1000 * 2 * 64 * 4 and ask(1000, 3, 4, 1, 136, 5, 128) == 2 * 4 * 1000 * 136 * 4
    for sizes in ((1000, 3, 8, 8, 64, 0, 128), (1000, 3, 8, 2, 64, 5, 64), (1000, 3, 8, 2, 64, 0, 4), (1 << 20, 3, 8, 2, 64, 0, 128),
                  (100000, 90000, 8, 2, 64, 0, 128), (0, 0, 8, 2, 64, 0, 128), (-1, 3, 8, 2, 64, 0, 128), (1000, -3, 8, 2, 64, 0, 128),
                  (1000, 3, 8, 3, 64, 0, 128), (1000, 3, 0, 2, 64, 0, 128), (1000, 3, 8, 0, 64, 0, 128), (1000, 3, 8, 2, 0, 0, 128),
                  (1000, 3, 8, 2, 264, 0, 128), (1000, 3, 8, 2, 64, 4, 128)):
        assert ask(*sizes) == 0, sizes
