"""Rotary positions against the formulas in float64: both layouts, parts of the
head, every scaling, positions for each token, each sequence or all, far out, rows
that are not whole 16-byte chunks, columns of wider matrices and in place."""
from math import exp, log, pi

import numpy as np
import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd, amd_lm
from qutai_amd.lm import Packing, Rotary
from qutai_amd.lm.layers import rotary
from tests.helpers import download, normal, stored, upload

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24
STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}
PARTS = {"kind": "parts", "factor": 8.0, "original_length": 256}

CASES = [
    # dtype, tokens, heads, kv_heads, dim, rotary_dim, layout, scaling, stacked
    ("bfloat16", 1, 1, 1, 64, 64, "half", None, False),
    ("bfloat16", 67, 16, 4, 64, 64, "half", PARTS, True),
    ("bfloat16", 67, 16, 4, 64, 64, "interleaved", {"kind": "linear", "factor": 4.0}, True),
    ("bfloat16", 33, 8, 2, 128, 64, "half", {"kind": "base", "factor": 8.0}, True),
    ("bfloat16", 33, 8, 2, 128, 32, "interleaved", PARTS, False),
    ("bfloat16", 9, 3, 1, 80, 40, "half", None, True),
    ("bfloat16", 9, 3, 3, 80, 24, "interleaved", None, False),
    ("bfloat16", 5, 2, 1, 6, 2, "half", None, True),
    ("bfloat16", 5, 2, 1, 7, 4, "interleaved", None, False),
    ("bfloat16", 17, 2, 2, 256, 256, "half", None, False),
    ("bfloat16", 300, 5, 1, 96, 96, "half", None, True),
    ("float32", 1, 1, 1, 2, 2, "half", None, False),
    ("float32", 50, 12, 12, 80, 40, "interleaved", {"kind": "base", "factor": 2.0}, False),
    ("float32", 50, 4, 2, 80, 40, "half", PARTS, True),
    ("float32", 21, 3, 1, 128, 128, "half", {"kind": "linear", "factor": 7.5}, True),
    ("float32", 21, 3, 1, 36, 12, "interleaved", None, True),
    ("float32", 4, 2, 1, 256, 100, "half", None, False),
    ("bfloat16", 12, 0, 3, 64, 64, "half", None, False),
    ("bfloat16", 12, 3, 0, 64, 16, "interleaved", None, False),
]


def frequencies(rotary_dim, scaling, theta=10000.0):
    """(radians a position of every pair, magnitude), from the definition."""
    kind, factor = (scaling["kind"], scaling["factor"]) if scaling else (None, 1.0)
    found = []
    for i in range(rotary_dim // 2):
        share = 2 * i / rotary_dim
        f = exp(-share * log(theta))
        if kind == "base":
            f = exp(-share * (log(theta) + log(factor) * rotary_dim / (rotary_dim - 2)))
        if kind == "linear":
            f /= factor
        if kind == "parts":
            turns = scaling["original_length"] * f / (2 * pi)
            kept = min(1.0, max(0.0, (turns - 1.0) / 31.0))
            f = kept * f + (1 - kept) * f / factor
        found.append(f)
    return np.array(found), 0.1 * log(factor) + 1 if kind == "parts" else 1.0


def turned(x, places, rotary_dim, layout, scaling, sign=1):
    """(the turned heads of (tokens, heads, dim), their bound without the last rounding)."""
    f, magnitude = frequencies(rotary_dim, scaling)
    angle = places[:, None, None] * f
    c, s = magnitude * np.cos(angle), sign * magnitude * np.sin(angle)
    first, second = ((slice(0, rotary_dim // 2), slice(rotary_dim // 2, rotary_dim)) if layout == "half"
                     else (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)))
    y, bound = x.copy(), np.zeros(x.shape)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    # sine and cosine: 2 units of their own, the angle's rounding to first order, its fp64 reduction
    # (2^-53 of the turns), the magnitude; two products and a sum
    off = (np.abs(a) + np.abs(b)) * magnitude * (9 * UNIT + 2 * pi * 2.0 ** -51 * places[:, None, None] * f)
    bound[..., first], bound[..., second] = off, off
    return y, bound


def within(got, value, bound, dtype):
    bound = bound + STEP[dtype] * (np.abs(value) + bound)
    off = np.abs(got.reshape(value.shape) - value) - bound
    assert (off <= 0).all(), f"{off.max():.3g} beyond the bound at {np.unravel_index(off.argmax(), off.shape)}"


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:7])) + (c[7]["kind"] if c[7] else ""))
def test_turned_heads(case, inverse):
    dtype, tokens, heads, kv_heads, dim, rotary_dim, layout, scaling, stacked = case
    seed = 10 * CASES.index(case)
    q, k = (stored(normal(seed + i, (tokens, n, dim)), dtype) for i, n in enumerate((heads, kv_heads)))
    places = np.random.default_rng(seed).integers(0, 200000, tokens)
    positions = amd.storage(places.tolist(), dtype="int64")
    turns = Rotary(dim, rotary_dim=rotary_dim, layout=layout, scaling=scaling)
    dims = (turns, 1, tokens, heads, kv_heads, dim)
    expected = [turned(x, places, rotary_dim, layout, scaling, -1 if inverse else 1) for x in (q, k)]
    if not stacked:
        got = amd_lm.rotary(*(upload(x, dtype) if x.size else None for x in (q, k)), *dims, positions=positions,
                            inverse=inverse)
        for x, (value, bound) in zip(got, expected):
            if x is not None:
                within(download(x), value, bound, dtype)
        assert [x is None for x in got] == [heads == 0, kv_heads == 0]
        return
    # columns of one matrix whose other columns stay as they are, out of place and in place
    width = (heads + 2 * kv_heads) * dim + 8
    matrix = stored(normal(seed + 5, (tokens, width)), dtype)
    at = heads * dim + 8
    matrix[:, :heads * dim], matrix[:, at:at + kv_heads * dim] = q.reshape(tokens, -1), k.reshape(tokens, -1)
    block = upload(matrix, dtype)
    got = amd_lm.rotary(block, block, *dims, positions=positions, inverse=inverse, q_row=width, k_column=at, k_row=width)
    for x, (value, bound) in zip(got, expected):
        within(download(x), value, bound, dtype)
    amd_lm.rotary(block, block, *dims, positions=positions, inverse=inverse, q_row=width, k_column=at, k_row=width,
                  out=block, out_row=width, out_k_column=at)
    after = download(block).reshape(tokens, width)
    assert np.array_equal(after[:, :heads * dim], download(got[0]).reshape(tokens, -1))
    assert np.array_equal(after[:, at:at + kv_heads * dim], download(got[1]).reshape(tokens, -1))
    others = np.r_[heads * dim:at, at + kv_heads * dim:width]
    assert np.array_equal(after[:, others], matrix[:, others])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions_of_sequences(layout):
    """offset + starts + t is the position of a token of a batch."""
    batch, time, heads, kv_heads, dim = 3, 5, 4, 2, 64
    q, k = (stored(normal(i, (batch * time, n, dim)), "float32") for i, n in enumerate((heads, kv_heads)))
    starts = [0, 1000, 70000]
    turns = Rotary(dim, layout=layout)
    got = amd_lm.rotary(upload(q, "float32"), upload(k, "float32"), turns, batch, time, heads, kv_heads, dim, offset=7,
                        starts=amd.storage(starts, dtype="int64"))
    places = np.array([7 + s + t for s in starts for t in range(time)])
    for x, y in zip((q, k), got):
        within(download(y), *turned(x, places, dim, layout, None), "float32")


def test_default_is_the_decoders_rope():
    batch, time, heads, dim = 2, 40, 4, 64
    x = upload(normal(3, batch * time * heads * dim), "float32")
    own, _ = amd_lm.rotary(x, None, Rotary(dim), batch, time, heads, 0, dim, offset=3)
    assert np.abs(download(own) - download(amd_lm.rope(x, batch, time, heads, dim, 10000.0, 3))).max() <= 4e-6


def test_far_positions_keep_their_angles():
    """2^40 + 1 positions on, an angle of fp32 holds nothing; pairs still turn by
    their frequency (the turns' 53 bits leave 2^-11 of a turn there)."""
    turns, place = Rotary(4, theta=2.0 ** 20, layout="half"), 2 ** 24 + 1
    got, _ = amd_lm.rotary(upload(np.array([1.0, 1.0, 0.0, 0.0]), "float32"), None, turns, 1, 1, 1, 0, 4, offset=place)
    f = np.array([1.0, 2.0 ** -10]) * place
    assert np.abs(download(got) - np.r_[np.cos(f), np.sin(f)]).max() <= 1e-6


def test_inverse_turns_back_and_gradients():
    heads, kv_heads, dim, lengths = 4, 2, 64, [5, 1, 9]
    packing, turns = Packing(lengths), Rotary(64, rotary_dim=32, layout="half", scaling=PARTS)
    q, k = (Tensor(upload(normal(i, 15 * n * dim), "float32"), shape=(1, 15, n * dim), requires_grad=True)
            for i, n in enumerate((heads, kv_heads)))
    out = rotary(q, k, heads, kv_heads, turns, positions=packing.positions)
    places = np.concatenate([np.arange(n) for n in lengths])
    for i, (x, y) in enumerate(zip((q, k), out)):
        g = normal(7 + i, y.size)
        y.backward(Tensor(upload(g, "float32"), shape=y.shape))
        value, bound = turned(g.astype(np.float64).reshape(15, -1, dim), places, 32, "half", PARTS, -1)
        within(download(x.grad.storage), value, bound, "float32")
        # the turn is linear: <turned x, g> = <x, gradient>
        left = download(y.storage).astype(np.float64) @ g
        right = download(x.storage).astype(np.float64) @ download(x.grad.storage)
        assert abs(left - right) <= 1e-5 * np.abs(g).sum()


def test_no_tokens():
    turns = Rotary(64)
    empty = amd.AMDStorage(0, "float32")
    assert [x.size for x in amd_lm.rotary(empty, empty, turns, 0, 5, 2, 1, 64)] == [0, 0]


@pytest.mark.parametrize("lengths,total", [([1], 1), ([0, 3, 0, 0, 2, 0], 9), ([], 4), ([0, 0], 0), (list(range(130)), None),
                                           ([70000, 1, 5], 70100)])
def test_places_of_packed_tokens(lengths, total):
    packing = Packing(lengths, total)
    places = [t for n in lengths for t in range(n)]
    assert packing.positions.tolist() == places + [0] * (packing.total - len(places))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_beyond_32_bits(dtype):
    """In place in a matrix of more than 2^32 values: what the same rows give side by side."""
    rows, row, heads, dim = 17000, 1 << 18, 3, 64
    x, turns, columns = upload(normal(5, rows * heads * dim), dtype), Rotary(dim, layout="half", scaling=PARTS), (128, row - 192)
    block = amd.AMDStorage(rows * row, dtype)
    for column in columns:
        amd_lm.copy_rows(x, rows, heads * dim, out=block, out_column=column, out_row=row)
    dims = (turns, 1, rows, heads, heads, dim)
    near = amd_lm.rotary(x, x, *dims)
    amd_lm.rotary(block, block, *dims, q_column=columns[0], q_row=row, k_column=columns[1], k_row=row, out=block, out_row=row,
                  out_q_column=columns[0], out_k_column=columns[1])
    for y, column in zip(near, columns):
        assert np.array_equal(download(y), download(amd_lm.copy_rows(block, rows, heads * dim, column=column, row=row)))
