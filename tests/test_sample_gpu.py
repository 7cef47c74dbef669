"""Tokens sampled from logits against the definition in float64: each filter
alone and together, ties across every cut, rows of -inf, +inf and NaN, numbers at
both ends, vocabularies around a lane, a wave and a step of the workgroup."""
import numpy as np
import pytest

from qutai_amd.backends import amd, amd_lm
from tests.helpers import download, stored, upload

pytestmark = pytest.mark.gpu


def kept_weights(row, temperature, top_k, top_p, min_p):
    """Weights by index, 0 where a token is not kept."""
    row = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    order = np.argsort(-row, kind="stable")
    top = row[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(row == top, 1.0, np.exp((row - top) / temperature))
    w[row == -np.inf] = 0
    kept = order[:top_k] if top_k else order
    if top_p < 1:
        before = np.concatenate(([0.0], np.cumsum(w[kept])[:-1]))
        kept = kept[(before < top_p * w[kept].sum()) | (np.arange(len(kept)) == 0)]
    kept = kept[w[kept] >= min_p]
    out = np.zeros(len(row))
    out[kept] = w[kept]
    return out


def expected(row, u, temperature, top_k, top_p, min_p):
    """[(token, probability)]: more than one only where 64-bit sums cannot tell."""
    clean = np.where(np.isnan(row), -np.inf, row)
    if clean.max() == -np.inf:
        return [(-1, 0.0)]
    if temperature == 0:
        return [(int(clean.argmax()), 1.0)]
    found = set()
    for nudge in (1 - 1e-9, 1, 1 + 1e-9):
        w = kept_weights(row, temperature, top_k, top_p * nudge if top_p < 1 else 1.0, min_p)
        sums = np.cumsum(w)
        for slack in (-1e-10, 0, 1e-10):
            over = np.nonzero((sums > (min(max(u, 0.0), 1.0) + slack) * sums[-1]) & (w > 0))[0]
            token = over[0] if len(over) else np.nonzero(w)[0][-1]
            found.add((int(token), float(w[token] / sums[-1])))
    return sorted(found)


def check(logits, uniforms, dtype="float32", wide=False, **parameters):
    logits = stored(logits, dtype)
    rows, vocab = logits.shape
    if not wide:
        uniforms = np.asarray(uniforms, dtype=np.float32)
    given = {n: p if np.isscalar(p) else amd.storage(list(map(int, p)), dtype="int64") if n == "top_k" else upload(p, "float32")
             for n, p in parameters.items()}
    source = upload(logits, dtype)
    tokens, probabilities = amd_lm.sample(source, upload(uniforms, "float64" if wide else "float32"), rows, vocab, **given)
    tokens, probabilities = download(tokens), download(probabilities)
    names = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    for r in range(rows):
        # (a float32 storage's numbers are what the kernel sees)
        p = {n: v if n not in parameters else parameters[n] if np.isscalar(parameters[n])
             else (int if n == "top_k" else lambda x: float(np.float32(x)))(parameters[n][r]) for n, v in names.items()}
        allowed = expected(logits[r], float(uniforms[r]), **p)
        near = [(t, c) for t, c in allowed if t == tokens[r]]
        assert near, (r, p, int(tokens[r]), allowed)
        assert any(abs(probabilities[r] - c) <= 2.0 ** -23 * c for _, c in near)
    return tokens


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=1), dict(top_k=5), dict(top_p=0.3), dict(top_p=0.0),
            dict(min_p=0.2), dict(temperature=1.3, top_k=20, top_p=0.8, min_p=0.02), dict(temperature=2.5, top_p=0.99),
            dict(top_k=10 ** 9, top_p=0.9999), dict(temperature=1e-3, top_p=0.5), dict(min_p=1.0), dict(temperature=50.0, top_k=400)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 65, 1000, 4096, 4097, 8192, 8193, 33000])
def test_filters_match_float64(dtype, vocab):
    rng = np.random.default_rng(vocab)
    for i, setting in enumerate(SETTINGS):
        rows = 4 if vocab < 8192 else 2
        logits = rng.standard_normal((rows, vocab)) * 3
        logits[:, rng.random(vocab) < 0.05] = -np.inf
        check(logits, rng.random(rows), dtype, **setting)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_ties(dtype):
    """Equal logits at every cut: all tokens alike, a few levels, both zeros."""
    rng = np.random.default_rng(0)
    for vocab in (10, 100, 5000):
        rows = 6
        for logits in (np.zeros((rows, vocab)), rng.integers(-2, 3, (rows, vocab)).astype(float),
                       np.where(rng.random((rows, vocab)) < 0.5, 0.0, -0.0)):
            for setting in (dict(), dict(top_k=3), dict(top_k=vocab // 2, top_p=0.37), dict(top_p=0.61), dict(min_p=0.3),
                            dict(temperature=0.0), dict(top_k=vocab // 3, top_p=0.9, min_p=0.1)):
                check(logits, rng.random(rows), dtype, **setting)


def test_numbers_cover_the_tokens_in_order():
    """Evenly spread numbers hit every token as often as its share."""
    logits = np.log(np.array([1.0, 4.0, 0.0, 2.0, 1.0]) + 1e-300)
    n = 800
    tokens = check(np.tile(logits, (n, 1)), (np.arange(n) + 0.5) / n, wide=True)
    assert np.array_equal(tokens, np.repeat([0, 1, 3, 4], [100, 400, 200, 100]))


def test_both_ends_and_outside():
    logits = np.tile(np.array([-np.inf, 0.0, 1.0, -1.0, -np.inf]), (6, 1))
    tokens = check(logits, np.array([0.0, 1.0 - 2.0 ** -53, 1.0, 7.0, -3.0, 0.5]), wide=True)
    assert list(tokens[:5]) == [1, 3, 3, 3, 1]
    # a number that is not one counts as 0
    nan = amd_lm.sample(upload(logits[:1], "float32"), upload(np.array([np.nan]), "float32"), 1, 5)[0]
    assert download(nan)[0] == 1


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("setting", [dict(), dict(temperature=0.0), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.5),
                                     dict(top_k=3, top_p=0.9)])
def test_rows_without_a_finite_logit(dtype, setting):
    logits = np.full((5, 9), -np.inf)
    logits[1, 3], logits[1, 5] = np.inf, np.inf
    logits[1, 6] = 4.0
    logits[2] = np.nan
    logits[3, 4], logits[3, 2] = -3.0, np.nan
    logits[4] = np.arange(9)
    logits[4, 8] = np.nan
    tokens = check(logits, np.full(5, 0.9), dtype, **setting)
    assert tokens[0] == -1 and tokens[2] == -1 and tokens[3] == 4 and tokens[1] in (3, 5)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [300, 9000])
def test_magnitudes_of_every_size(dtype, vocab):
    """Logits around zero of magnitudes far apart, where a cut may lie among the
    smallest; a wide and a narrow temperature; NaN of both signs."""
    rng = np.random.default_rng(vocab)
    tiny = rng.choice([-1.0, 1.0], (4, vocab)) * 2.0 ** rng.integers(-40, 4, (4, vocab))
    tiny[:, rng.random(vocab) < 0.1] = 0.0
    tiny[1] = np.where(rng.random(vocab) < 0.5, -np.abs(tiny[1]), -0.0)  # the largest is zero
    tiny[2] *= 2.0 ** -60  # all of them next to nothing
    tiny[3, rng.random(vocab) < 0.2] = -np.inf
    for setting in (dict(), dict(top_k=vocab // 2), dict(top_p=0.5), dict(top_k=vocab // 2, top_p=0.7), dict(min_p=0.9),
                    dict(temperature=0.01, top_p=0.6), dict(temperature=300.0, top_k=vocab // 3), dict(top_k=vocab - 1)):
        check(tiny, rng.random(4), dtype, **setting)
    broken = rng.standard_normal((2, vocab))
    broken[:, ::3] = np.nan
    broken[:, 1::6] = np.copysign(np.nan, -1.0)
    for setting in (dict(), dict(top_k=5), dict(top_k=vocab - 3, top_p=0.9), dict(top_p=0.4)):
        check(broken, rng.random(2), dtype, **setting)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [50, 32768, 100001])
def test_parameters_of_every_row(dtype, vocab):
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 50000 else 8
    check(rng.standard_normal((rows, vocab)) * 2.5, rng.random(rows), dtype,
          temperature=np.where(rng.random(rows) < 0.2, 0.0, rng.random(rows) + 0.3), top_k=rng.integers(0, 40, rows),
          top_p=np.where(rng.random(rows) < 0.3, 1.0, rng.random(rows)), min_p=rng.random(rows) * 0.1)


def test_the_largest_vocabulary():
    rng = np.random.default_rng(2)
    for dtype in ("float32", "bfloat16"):
        for setting in (dict(), dict(top_p=0.9), dict(top_k=1000, temperature=0.9)):
            check(rng.standard_normal((1, 1 << 20)), rng.random(1), dtype, **setting)


def test_no_rows():
    empty = amd.AMDStorage(0, "float32")
    tokens, probabilities = amd_lm.sample(empty, empty, 0, 10)
    assert tokens.size == 0 and probabilities.size == 0 and tokens.dtype == "int64"


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_parameters_of_rows_that_are_not_numbers(dtype):
    """NaN: a temperature of 0, no top_p, a min_p of 1."""
    rng = np.random.default_rng(3)
    logits, nan = stored(rng.standard_normal((6, 40)), dtype), float("nan")
    given = dict(temperature=[nan, 1.0, 1.0, nan, 0.7, 1.0], top_p=[1.0, nan, 1.0, nan, 0.4, 2.0], min_p=[0.0, 0.0, nan, nan, -1.0, 3.0])
    meant = dict(temperature=[0.0, 1.0, 1.0, 0.0, 0.7, 1.0], top_p=[1.0, 1.0, 1.0, 1.0, 0.4, 1.0], min_p=[0.0, 0.0, 1.0, 1.0, 0.0, 1.0])
    results = [amd_lm.sample(upload(logits, dtype), upload(np.full(6, 0.6), "float32"), 6, 40,
                             **{n: upload(np.array(v), "float32") for n, v in p.items()}) for p in (given, meant)]
    assert all(a.to_array() == b.to_array() for a, b in zip(*results))
    assert list(download(results[0][0])[[0, 2, 3, 5]]) == list(logits[[0, 2, 3, 5]].argmax(1))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [4097, 140000])
def test_infinities_and_ties_in_long_rows(dtype, vocab):
    """+inf in a few places and in more than top_k keeps, NaN in a third, and all
    logits alike, in rows longer than the list of candidates and than the registers."""
    rng = np.random.default_rng(vocab)
    rows = rng.standard_normal((4, vocab)) * 3
    rows[0, rng.integers(0, vocab, 3)] = np.inf
    rows[1, rng.integers(0, vocab, 900)] = np.inf
    rows[2, ::3] = np.nan
    rows[3] = -7.25
    for setting in (dict(), dict(top_k=5), dict(top_k=700, top_p=0.4), dict(top_p=0.5), dict(min_p=1.0), dict(temperature=0.0)):
        check(rows, rng.random(4), dtype, **setting)
