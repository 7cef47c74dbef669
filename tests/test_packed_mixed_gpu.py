"""Packed attention of short documents beside long ones: what a document's probabilities
and dS keep goes by its own length, not by its neighbours'."""
import numpy as np
import pytest

from tests.test_attention_packed_gpu import inputs, reference, run, within

pytestmark = pytest.mark.gpu

SHORT = [6, 64, 1, 33, 2, 0, 9, 47]


@pytest.mark.parametrize("heads,kv_heads,dim,causal,many", [
    # every shape of the key pass: few tiles of groups of four and two, many (repeated) of each
    (4, 1, 64, True, 1), (4, 2, 64, False, 1), (3, 1, 64, True, 1), (8, 2, 128, True, 1), (4, 2, 128, True, 1), (3, 3, 128, False, 1),
    (8, 2, 96, True, 1), (4, 2, 80, False, 1), (2, 2, 72, True, 1), (8, 2, 32, True, 1), (3, 3, 24, False, 1),
    (4, 1, 64, True, 60), (8, 4, 128, True, 60), (3, 3, 96, False, 60)])
@pytest.mark.parametrize("long", [65, 200])
def test_short_documents_beside_a_long_one(heads, kv_heads, dim, causal, many, long):
    """Documents of up to 64 tokens take probabilities and dS in two bf16 parts, of which
    2^-8 of 2^-8 is lost, whatever lies beside them; the long one's take one part."""
    lengths = SHORT[:4] + [long] + SHORT[4:] * many
    case = ("bfloat16", lengths, heads, kv_heads, dim, causal, True)
    q, k, v, g = inputs(case, 71)
    got, rest = run(case, q, k, v, g)
    assert rest is not None
    start = 0
    at = {}  # rows of the short documents and of the long one
    for n in lengths:
        at.setdefault(n == long, []).extend(range(start, start + n))
        start += n
    for is_long, rows in at.items():
        bounds = reference(*(x[rows] for x in (q, k, v, g)), [long] if is_long else [n for n in lengths if n != long], causal,
                           "bfloat16", True, 2.0 ** -8 if is_long else 2.0 ** -16)
        for name, (value, bound) in bounds.items():
            whole = got[name].reshape(len(q), *value.shape[1:])
            within(name, whole[rows], value, bound)


@pytest.mark.parametrize("dim,causal", [(64, True), (64, False), (128, True), (40, False)])
def test_out_does_not_depend_on_the_neighbours(dim, causal):
    """A document's out, lse and dQ are the same bits alone, beside shorter documents and
    beside a long one (dK and dV sum their heads in an order that goes by the batch)."""
    heads, kv_heads, document = 4, 2, 37
    case = ("bfloat16", [document, 200, 5], heads, kv_heads, dim, causal, False)
    q, k, v, g = inputs(case, 73)
    results = []
    for lengths in ([document], [document, 5], [document, 200, 5]):
        rows = slice(0, sum(lengths))
        got, _ = run(("bfloat16", lengths, heads, kv_heads, dim, causal, False), *(x[rows] for x in (q, k, v, g)))
        results.append({n: got[n].reshape(sum(lengths), -1)[:document] for n in ("out", "lse", "dq")})
    for other in results[1:]:
        assert all(np.array_equal(results[0][n], other[n]) for n in other)
