"""Attention of packed sequences, forward and backward, against the formulas in
float64: lengths of zero and one, around the tiles' ends and of many tiles, heads
shared and not, every width and type, with and without the causal mask, operands
that are columns of wider matrices, infinities in a neighbouring sequence."""
import numpy as np
import pytest

from qutai_amd.backends import amd, amd_lm
from qutai_amd.lm import Packing
from tests.helpers import download, normal, stored, upload

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24  # half a step of fp32
STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}

CASES = [
    # dtype, lengths, heads, kv_heads, dim, causal, stacked
    ("bfloat16", [1], 1, 1, 64, True, False),
    ("bfloat16", [0, 1, 0, 2, 3], 4, 2, 64, True, True),
    ("bfloat16", [31, 32, 33, 1], 4, 1, 64, True, True),
    ("bfloat16", [63, 64, 65], 4, 4, 64, False, False),
    ("bfloat16", [127, 128, 129], 2, 1, 64, True, True),
    ("bfloat16", [255, 1, 256, 257], 2, 2, 64, True, False),
    ("bfloat16", [300, 7, 520], 6, 2, 64, True, True),
    ("bfloat16", [700, 3], 8, 1, 64, False, True),
    ("bfloat16", [5, 130, 64], 5, 5, 64, True, True),
    ("bfloat16", [33, 290], 3, 1, 64, True, False),
    ("bfloat16", [65, 129, 40], 16, 1, 64, True, False),
    ("bfloat16", [1, 64, 200], 4, 1, 128, True, True),
    ("bfloat16", [257, 31], 2, 2, 128, False, False),
    ("bfloat16", [400, 9], 8, 2, 128, True, True),
    ("bfloat16", [100, 30], 4, 2, 96, True, True),
    ("bfloat16", [97, 161], 3, 3, 80, False, False),
    ("bfloat16", [70, 129], 4, 2, 40, True, True),
    ("bfloat16", [70, 5], 2, 1, 32, True, False),
    ("bfloat16", [70, 35], 2, 1, 8, True, False),
    ("bfloat16", [40, 140], 2, 1, 136, True, True),
    ("bfloat16", [140, 20], 2, 1, 256, False, False),
    ("bfloat16", [9, 30], 2, 1, 20, True, True),
    ("bfloat16", [9, 30], 2, 1, 7, False, False),
    ("bfloat16", [90, 200], 4, 1, 128, True, True),
    ("bfloat16", [129, 64], 6, 1, 128, False, False),
    ("bfloat16", [129, 64], 3, 1, 128, True, False),
    ("bfloat16", [150, 77], 8, 2, 64, False, True),
    ("bfloat16", [8, 3, 1, 7], 4, 2, 64, True, True),
    ("bfloat16", [8, 3, 1, 7], 4, 2, 128, True, False),
    ("float32", [1, 0, 2, 5], 4, 2, 64, True, True),
    ("float32", [20, 21, 3], 4, 2, 64, False, True),
    ("float32", [64, 129, 33], 4, 2, 64, True, True),
    ("float32", [200, 31], 3, 3, 80, False, False),
    ("float32", [140, 65], 2, 1, 128, True, True),
    ("float32", [40, 20], 2, 1, 36, True, False),
    ("float32", [10, 33], 2, 1, 10, True, True),
    ("float32", [20, 7], 2, 1, 160, False, False),
    ("bfloat16", [150, 77, 1], 8, 2, 96, True, True),
    ("bfloat16", [150, 64], 6, 1, 72, False, False),
    ("bfloat16", [33, 64, 130], 4, 4, 88, True, False),
    ("bfloat16", [150, 77, 1], 8, 2, 32, True, True),
    ("bfloat16", [150, 64], 6, 1, 24, False, True),
    ("bfloat16", [33, 64, 130], 3, 3, 16, False, False),
]


def inputs(case, seed):
    dtype, lengths, heads, kv_heads, dim, causal, stacked = case
    total = sum(lengths)
    q, k, v, g = (stored(normal(seed + i, (total, n, dim), scale), dtype)
                  for i, (n, scale) in enumerate(((heads, 1.5), (kv_heads, 1.0), (kv_heads, 1.0), (heads, 1.0))))
    return q, k, v, g


def reference(q, k, v, g, lengths, causal, dtype, exact_rest, weight=None):
    """{name: (value, bound)}: the formulas in float64, and how far roundings may
    take a kernel that holds scores, statistics and sums in fp32 and rounds bf16's
    probabilities and dS to bf16 (fp32's keep 2^-24 of theirs)."""
    total, heads, dim = q.shape
    kv_heads, scale = k.shape[1], q.shape[2] ** -0.5
    group, step = heads // k.shape[1], STEP[dtype]
    if weight is None:  # a probability's or dS's rounding
        weight = 2.0 ** -8 if dtype == "bfloat16" else 8 * UNIT
    out = {n: (np.zeros(s), np.zeros(s)) for n, s in (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    lse = np.zeros((total, heads)), np.zeros((total, heads))
    start = 0
    for n in lengths:
        rows = slice(start, start + n)
        seen = np.tril(np.ones((n, n), bool)) if causal else np.ones((n, n), bool)
        for h in range(heads if n else 0):
            c = h // group
            Q, K, V, G = q[rows, h], k[rows, c], v[rows, c], g[rows, h]
            s = Q @ K.T * scale
            # the score's sum of dim products, its scaling, the exponent's product and the exponential
            s_bound = (dim + 8) * UNIT * (np.abs(Q) @ np.abs(K).T) * scale + 4 * UNIT * np.abs(s)
            s = np.where(seen, s, -np.inf)
            top = s.max(1, keepdims=True)
            e = np.exp(s - top)
            p = e / e.sum(1, keepdims=True)
            off = np.where(seen, s_bound, 0).max(1, keepdims=True) + 8 * UNIT + 2 * UNIT * np.abs(top)
            p_rel = 2 * off + (n + 4) * UNIT  # of a probability in fp32: its own score, and the sum's
            lse[0][rows, h] = (top + np.log(e.sum(1, keepdims=True)))[:, 0]
            lse[1][rows, h] = (p_rel + 4 * UNIT * (1 + np.abs(lse[0][rows, h][:, None])))[:, 0]
            o = p @ V
            o_bound = (p @ np.abs(V)) * (p_rel + weight + (n + 2) * UNIT)
            out["out"][0][rows, h] = o
            out["out"][1][rows, h] = o_bound + step * (np.abs(o) + o_bound)
            dp = G @ V.T
            dp_bound = (dim + 4) * UNIT * (np.abs(G) @ np.abs(V).T)
            delta = (G * o).sum(1, keepdims=True)
            left = 2.0 ** -16 if exact_rest and dtype == "bfloat16" else step  # of what the backward knows of out
            d_bound = (np.abs(G) * (o_bound + left * (np.abs(o) + o_bound))).sum(1, keepdims=True) \
                + (dim + 4) * UNIT * (np.abs(G) * np.abs(o)).sum(1, keepdims=True)
            ds = p * (dp - delta)
            rel = 2 * p_rel + lse[1][rows, h][:, None] + weight
            ds_bound = np.abs(ds) * rel + p * (dp_bound + d_bound) * (1 + rel) + 4 * UNIT * p * (np.abs(dp) + np.abs(delta))
            dq = ds @ K * scale
            out["dq"][0][rows, h] = dq
            out["dq"][1][rows, h] = (ds_bound + (n + 4) * UNIT * np.abs(ds)) @ np.abs(K) * scale * (1 + step) + step * np.abs(dq)
            out["dk"][0][rows, c] += ds.T @ Q * scale
            out["dk"][1][rows, c] += (ds_bound + (n * group + 4) * UNIT * np.abs(ds)).T @ np.abs(Q) * scale * (1 + step)
            out["dv"][0][rows, c] += p.T @ G
            out["dv"][1][rows, c] += (p * (rel + (n * group + 4) * UNIT)).T @ np.abs(G) * (1 + step)
        start += n
    for name in ("dk", "dv"):
        out[name] = out[name][0], out[name][1] + step * np.abs(out[name][0])
    return {**out, "lse": lse}


def within(name, got, value, bound):
    off = np.abs(got.reshape(value.shape) - value) - bound
    assert np.isfinite(got).all(), f"{name} is not finite"
    assert (off <= 0).all(), f"{name}: {off.max():.3g} beyond its bound at {np.unravel_index(off.argmax(), off.shape)}"


def run(case, q, k, v, g, total=None):
    dtype, lengths, heads, kv_heads, dim, causal, stacked = case
    rows = q.shape[0]
    packing = Packing(lengths, total=rows)
    if stacked:
        width = (heads + 2 * kv_heads) * dim
        block = upload(np.concatenate([x.reshape(rows, -1) for x in (q, k, v)], 1).reshape(-1), dtype)
        stores = (block,) * 3
        place = dict(q_row=width, k_column=heads * dim, k_row=width, v_column=(heads + kv_heads) * dim, v_row=width)
    else:
        stores, place = tuple(upload(x, dtype) for x in (q, k, v)), {}
    dims = (packing, heads, kv_heads, dim)
    out, lse, rest = amd_lm.attention_packed(*stores, *dims, causal=causal, rest=True, **place)
    gradient = upload(g, dtype)
    grads = amd_lm.attention_packed_backward(gradient, *stores, out, lse, *dims, causal=causal, rest=rest, **place)
    result = dict(zip(("dq", "dk", "dv"), map(download, grads)), out=download(out), lse=download(lse))
    if stacked:  # the same gradients in columns of one block
        into = amd.full(rows * width, 7.0, dtype=dtype)
        amd_lm.attention_packed_backward(gradient, *stores, out, lse, *dims, causal=causal, rest=rest, **place, into=into)
        columns = np.concatenate([result[n].reshape(rows, -1) for n in ("dq", "dk", "dv")], 1)
        assert np.array_equal(download(into).reshape(rows, width), columns)
    return result, rest


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_forward_and_gradients(case):
    dtype, lengths, heads, kv_heads, dim, causal, _ = case
    q, k, v, g = inputs(case, 100 + CASES.index(case))
    got, rest = run(case, q, k, v, g)
    for name, (value, bound) in reference(q, k, v, g, lengths, causal, dtype, rest is not None).items():
        within(name, got[name], value, bound)


@pytest.mark.parametrize("dtype,dim", [("bfloat16", 64), ("bfloat16", 128), ("bfloat16", 20), ("float32", 64)])
def test_rows_behind_the_last_sequence_are_zero(dtype, dim):
    case = (dtype, [40, 3], 4, 2, dim, True, True)
    q, k, v, g = (np.concatenate((x, np.full((5, *x.shape[1:]), np.nan))) for x in inputs(case, 5))
    got, rest = run(case, q, k, v, g)
    for name, (value, bound) in reference(*(x[:43] for x in (q, k, v, g)), [40, 3], True, dtype, rest is not None).items():
        value, bound = (np.concatenate((x, np.zeros((5, *x.shape[1:])))) for x in (value, bound))
        within(name, got[name], value, bound)


@pytest.mark.parametrize("dtype,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64)])
def test_a_sequence_does_not_see_its_neighbours(dtype, dim):
    case = (dtype, [70, 33, 50], 4, 2, dim, False, False)
    q, k, v, g = inputs(case, 9)
    clean, _ = run(case, q, k, v, g)
    for x, value in ((k, np.inf), (v, np.nan), (q, -np.inf), (g, np.nan)):
        x[70:103] = value
    got, _ = run(case, q, k, v, g)
    for name, value in clean.items():
        rows, other = got[name].reshape(153, -1), value.reshape(153, -1)
        assert np.array_equal(rows[:70], other[:70]) and np.array_equal(rows[103:], other[103:])
        assert not np.isfinite(rows[70:103]).all()


@pytest.mark.parametrize("dtype,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64)])
def test_later_tokens_do_not_change_earlier_ones(dtype, dim):
    case = (dtype, [140], 4, 2, dim, True, False)
    q, k, v, g = inputs(case, 11)
    value, bound = reference(q[:100], k[:100], v[:100], g[:100], [100], True, dtype, False)["out"]
    k[100:], v[100:] = np.inf, np.nan
    got, _ = run(case, q, k, v, g)
    within("out", got["out"].reshape(140, -1)[:100], value, bound)
    assert np.isnan(got["out"].reshape(140, -1)[100:]).any(1).all()


def test_large_scores_and_equal_ones():
    """Scores of thousands: one key takes a row; equal keys share it."""
    case = ("bfloat16", [80], 2, 1, 64, True, False)
    q, k, v, g = inputs(case, 13)
    q *= 64
    got, rest = run(case, q, k, v, g)
    expected = reference(q, k, v, g, [80], True, "bfloat16", rest is not None)
    within("out", got["out"], *expected["out"])
    k[:] = k[:1]
    got, rest = run(case, q, k, v, g)
    within("out", got["out"], *reference(q, k, v, g, [80], True, "bfloat16", rest is not None)["out"])


def test_the_same_bits_every_time():
    case = ("bfloat16", [300, 65, 513], 8, 2, 64, True, True)
    operands = inputs(case, 17)
    first, _ = run(case, *operands)
    again, _ = run(case, *operands)
    assert all(np.array_equal(first[n], again[n]) for n in first)


@pytest.mark.parametrize("dtype,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 80)])
def test_rectangles_agree_with_attention(dtype, dim):
    """Sequences of one length are what ``attention`` computes of a batch."""
    batch, time, heads, kv_heads = 3, 150, 4, 2
    case = (dtype, [time] * batch, heads, kv_heads, dim, True, False)
    q, k, v, g = inputs(case, 19)
    got, _ = run(case, q, k, v, g)
    stores = [upload(x, dtype) for x in (q, k, v)]
    out, lse = amd_lm.attention(*stores, batch, time, heads, kv_heads, dim)
    grads = amd_lm.attention_backward(upload(g, dtype), *stores, out, lse, batch, time, heads, kv_heads, dim)
    bounds = reference(q, k, v, g, [time] * batch, True, dtype, False)
    for name, x in (("out", out), ("lse", lse), *zip(("dq", "dk", "dv"), grads)):
        value, bound = bounds[name]
        within(name, got[name], download(x).reshape(value.shape), 2 * bound)


@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [
    ([1, 2, 3, 5, 0, 8] * 100, 4, 2, 64), ([9, 2, 3, 5, 0, 8] * 100, 4, 1, 64), ([9, 40] * 150, 8, 4, 128),
    ([65, 2] * 140, 4, 4, 64), ([65, 2] * 140, 8, 4, 96), ([65, 2] * 140, 4, 4, 80),
    ([65, 2] * 140, 8, 4, 32), ([65, 2] * 140, 4, 4, 24)])
def test_many_short_sequences(lengths, heads, kv_heads, dim):
    case = ("bfloat16", lengths, heads, kv_heads, dim, True, True)
    q, k, v, g = inputs(case, 23)
    got, rest = run(case, q, k, v, g)
    for name, (value, bound) in reference(q, k, v, g, lengths, True, "bfloat16", rest is not None).items():
        within(name, got[name], value, bound)


def test_nothing_to_attend():
    for lengths, total in (([], 0), ([0, 0], 0), ([], 3)):
        packing = Packing(lengths, total=total)
        q = upload(np.ones(total * 4 * 64), "bfloat16")
        k, v = (upload(np.ones(total * 2 * 64), "bfloat16") for _ in range(2))
        out, lse = amd_lm.attention_packed(q, k, v, packing, 4, 2, 64)
        assert out.size == q.size and not download(out).any()
        grads = amd_lm.attention_packed_backward(q, q, k, v, out, lse, packing, 4, 2, 64)
        assert [x.size for x in grads] == [q.size, k.size, v.size] and not any(download(x).any() for x in grads)


def test_gradients_against_differences():
    """d loss / d x of the recorded layer function, loss = sum of out * g."""
    from qutai_amd import Tensor
    from qutai_amd.lm.layers import attention

    lengths, heads, kv_heads, dim = [3, 9, 6], 4, 2, 8
    case = ("float32", lengths, heads, kv_heads, dim, True, False)
    q, k, v, g = inputs(case, 29)
    packing = Packing(lengths)

    def value(arrays, recorded=False):
        tensors = [Tensor(upload(x, "float32"), shape=(1, 18, x.shape[1] * dim), requires_grad=True) for x in arrays]
        out = attention(*tensors, heads, kv_heads, packing)
        if recorded:
            out.backward(Tensor(upload(g, "float32"), shape=out.shape))
            return [download(t.grad.storage) for t in tensors]
        return float(download(out.storage) @ g.reshape(-1))

    grads = value((q, k, v), True)
    rng = np.random.default_rng(31)
    for which, x in enumerate((q, k, v)):
        step = 1e-2 * rng.standard_normal(x.shape)
        ahead, behind = ([a + s * step if i == which else a for i, a in enumerate((q, k, v))] for s in (1, -1))
        slope = (value(ahead) - value(behind)) / 2
        # third derivatives of a softmax of scores of order 1 times 1e-6 a step, and fp32's sums of 18 * 32 values
        assert abs(slope - grads[which] @ step.reshape(-1)) <= 2e-4 * (np.abs(grads[which]) @ np.abs(step).reshape(-1)) + 1e-5


@pytest.mark.parametrize("apart,dtype,lengths,heads,kv_heads,dim", [
    (True, "float32", [330, 0, 41], 8, 1, 64), (True, "float32", [130, 129], 6, 2, 128), (True, "bfloat16", [200, 30], 4, 1, 136),
    (False, "float32", [330, 41], 2, 2, 64), (False, "float32", [21 + i % 9 for i in range(70)], 16, 8, 32),
    (False, "bfloat16", [21 + i % 9 for i in range(70)], 16, 8, 136)])
@pytest.mark.parametrize("causal", [True, False])
def test_heads_of_a_group_side_by_side(apart, dtype, lengths, heads, kv_heads, dim, causal):
    """The key pass of few tiles, whose heads' sums are added up by a kernel of their own,
    and of many; the rows behind the sequences stay zero, the same sums come every time."""
    runtime = amd.get_runtime()
    packing = Packing(lengths)
    need = packing.plan(2, heads, kv_heads, dim, amd.code(dtype), True, dim ** -0.5, causal)[3]
    assert bool(need) == apart and need % (8 * packing.total * dim) == 0
    case = dtype, lengths, heads, kv_heads, dim, causal, True
    q, k, v, g = inputs(case, 31)
    behind = [np.concatenate([x, np.full((3, *x.shape[1:]), 5.0)]) for x in (q, k, v, g)]
    result, rest = run(case, *behind)
    expected = reference(q, k, v, g, lengths, causal, dtype, rest is not None)
    for name, (value, bound) in expected.items():
        got = result[name].reshape(len(behind[0]), *value.shape[1:])
        within(name, got[:-3], value, bound)
        assert not got[-3:].any()
    again, _ = run(case, *behind)
    assert all(np.array_equal(result[name], again[name]) for name in result)
    assert runtime.lib.qutai_amd_attention_packed_workspace(*packing.extent[:2], heads, kv_heads, dim, amd.code(dtype), 4) == 0


@pytest.mark.parametrize("dtype,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64), ("bfloat16", 136)])
def test_rows_beyond_32_bits(dtype, dim):
    """Columns of matrices of more than 2^32 values: what the same rows give side by side."""
    lengths, heads, kv_heads, row = [700] * 24 + [1, 80], 4, 2, 1 << 18
    rows, wide, narrow = sum(lengths), heads * dim, kv_heads * dim
    assert rows * row > 1 << 32
    packing = Packing(lengths)
    q, k, v, g = (upload(normal(41 + i, rows * n * dim), dtype) for i, n in enumerate((heads, kv_heads, kv_heads, heads)))
    columns = (row - wide, 64, 4096)
    block = amd.AMDStorage(rows * row, dtype)
    for x, width, column in zip((q, k, v), (wide, narrow, narrow), columns):
        amd_lm.copy_rows(x, rows, width, out=block, out_column=column, out_row=row)
    place = dict(zip(("q_column", "k_column", "v_column"), columns), q_row=row, k_row=row, v_row=row)
    dims = (packing, heads, kv_heads, dim)
    near = amd_lm.attention_packed(q, k, v, *dims, rest=True)
    far = amd_lm.attention_packed(block, block, block, *dims, **place, rest=True)
    into = amd.AMDStorage(rows * row, dtype)
    expected = amd_lm.attention_packed_backward(g, q, k, v, *near[:2], *dims, rest=near[2])
    amd_lm.attention_packed_backward(g, block, block, block, *far[:2], *dims, rest=far[2], **place, into=into)
    found = [amd_lm.copy_rows(into, rows, width, column=column, row=row) for width, column in zip((wide, narrow, narrow), columns)]
    for x, y in zip((*near[:2], *expected), (*far[:2], *found)):
        x, y = download(x), download(y)
        assert np.isfinite(x).all() and x.any() and np.array_equal(x, y)


@pytest.mark.parametrize("dtype,dim", [("bfloat16", 64), ("bfloat16", 128), ("float32", 64), ("bfloat16", 20)])
def test_scales_and_a_packing_used_for_all(dtype, dim):
    """Twice the queries at half the scale are the same scores: the same results, and half of
    dQ's.  One packing serves every type, width, mask and scale."""
    packing, heads, kv_heads = Packing([90, 3, 200]), 4, 2
    for other in (32, 64, 80):  # tables and plans of other calls
        x, y = (upload(normal(3, 293 * n * other), "float32") for n in (1, 1))
        amd_lm.attention_packed_backward(x, x, y, y, *amd_lm.attention_packed(x, y, y, packing, 1, 1, other, causal=False),
                                         packing, 1, 1, other, causal=False)
    q, k, v, g = (stored(normal(51 + i, (293, n, dim)), dtype) for i, n in enumerate((heads, kv_heads, kv_heads, heads)))
    for scale in (0.7, 2.0 ** -20, 8.0):
        results = []
        for factor, rows in ((1.0, packing), (2.0, packing), (2.0, Packing([90, 3, 200]))):
            stores, dims = [upload(x, dtype) for x in (q * factor, k, v)], (rows, heads, kv_heads, dim)
            out, lse, rest = amd_lm.attention_packed(*stores, *dims, scale=scale / factor, rest=True)
            grads = amd_lm.attention_packed_backward(upload(g, dtype), *stores, out, lse, *dims, scale=scale / factor, rest=rest)
            dq, dk, dv = map(download, grads)
            results.append([download(out), download(lse), dq * factor, dk, dv])
        # a factor of two changes no rounding but of what lies below fp32's least normal number, 2^-126: each of the at
        # most 6 x 2 x 293 products in a sum moves by that at most, times the scale (8: less than 2^15 in all)
        for x in results[1:]:
            assert all(np.isfinite(a).all() and np.abs(a - b).max() <= 2.0 ** -111 for a, b in zip(results[0], x))


@pytest.mark.parametrize("heads,kv_heads,dim,causal", [
    (4, 2, 64, True), (3, 1, 64, False), (8, 2, 128, True), (2, 2, 128, False), (6, 3, 96, True), (4, 4, 80, False), (8, 2, 32, True),
    (3, 3, 24, False)])
def test_short_sequences_keep_more_of_probabilities(heads, kv_heads, dim, causal):
    """No sequence of more than 64 tokens: probabilities and dS in two bf16 parts, the second
    of what the first left, so 2^-8 of 2^-8 is lost."""
    lengths = [64, 1, 0, 33, 2, 9, 64, 31, 32, 47]
    case = ("bfloat16", lengths, heads, kv_heads, dim, causal, True)
    q, k, v, g = inputs(case, 61)
    got, rest = run(case, q, k, v, g)
    assert rest is not None
    for name, (value, bound) in reference(q, k, v, g, lengths, causal, "bfloat16", True, 2.0 ** -16).items():
        within(name, got[name], value, bound)
