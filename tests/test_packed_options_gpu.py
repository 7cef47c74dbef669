"""Packed attention with operands at addresses of their own, many tiles, and what it counts
as a launch on the matrix cores."""
import numpy as np
import pytest

from qutai_amd.backends import amd, amd_lm
from qutai_amd.lm import Packing
from tests.helpers import download, normal, stored, upload

pytestmark = pytest.mark.gpu


def shifted(values, dtype, shift=1):
    """A storage of these values whose address is no multiple of 16 bytes."""
    flat = np.concatenate([np.zeros(shift), np.asarray(values).reshape(-1)])
    return amd.view(upload(flat, dtype), shift, flat.size - shift)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", ["rest", "out", "gradient", "k"])
def test_operands_at_any_address(which, dim):
    """An operand that is not 16-byte aligned: the same bits for the rest of out, which is
    copied; gradients within the roundings of two kernels for the others, whose rows are
    then worked on one at a time without the rest."""
    packing, heads, kv_heads, dtype = Packing([70, 3, 31]), 4, 2, "bfloat16"
    q, k, v, g = (stored(normal(81 + i, (104, n, dim)), dtype) for i, n in enumerate((heads, kv_heads, kv_heads, heads)))
    stores, dims = [upload(x, dtype) for x in (q, k, v)], (packing, heads, kv_heads, dim)
    out, lse, rest = amd_lm.attention_packed(*stores, *dims, rest=True)
    operands = dict(gradient=upload(g, dtype), q=stores[0], k=stores[1], v=stores[2], out=out, lse=lse)
    expected = [download(x) for x in amd_lm.attention_packed_backward(**operands, packing=packing, heads=heads, kv_heads=kv_heads,
                                                                      dim=dim, rest=rest)]
    if which == "rest":
        rest = shifted(download(rest), dtype)
        assert rest.ptr % 16
    else:
        operands[which] = shifted(download(operands[which]), dtype)
    got = [download(x) for x in amd_lm.attention_packed_backward(**operands, packing=packing, heads=heads, kv_heads=kv_heads, dim=dim,
                                                                 rest=rest)]
    for a, b in zip(got, expected):
        # one wave per row knows out as bf16 alone, whose half step of 2^-8 is an error of delta and so of every dS
        assert np.array_equal(a, b) if which == "rest" else np.abs(a - b).max() <= 2.0 ** -5 * np.abs(b).max()


def test_many_sequences_of_many_heads():
    """More tiles times heads than workgroups fit a launch, of heads that share workgroups:
    sequences of one token, whose out is their value, and whose dV is their heads' gradient
    summed (four bf16 terms in fp32, rounded to bf16)."""
    count, heads, kv_heads, dim = 140000, 64, 16, 8
    assert count * heads >= 1 << 23
    packing = Packing([1] * count)
    q, k, v, g = (stored(np.tile(normal(91 + i, 1000 * n * dim), count // 1000), "bfloat16")
                  for i, n in enumerate((heads, kv_heads, kv_heads, heads)))
    stores, dims = [upload(x, "bfloat16") for x in (q, k, v)], (packing, heads, kv_heads, dim)
    out, lse, rest = amd_lm.attention_packed(*stores, *dims, rest=True)
    expected = np.repeat(v.reshape(count, kv_heads, 1, dim), heads // kv_heads, 2)
    assert np.array_equal(download(out), expected.reshape(-1))
    dq, dk, dv = amd_lm.attention_packed_backward(upload(g, "bfloat16"), *stores, out, lse, *dims, rest=rest)
    terms = g.astype(np.float64).reshape(count, kv_heads, heads // kv_heads, dim)
    total = terms.sum(2).reshape(-1)
    assert (np.abs(download(dv) - total) <= 2.0 ** -8 * np.abs(total) + 2.0 ** -22 * np.abs(terms).sum(2).reshape(-1)).all()
    # dS is what two fp32 sums of the same 8 products, of up to 60 in all, leave: 8 x 2^-24 x 60 each; times |q| or |k| of up
    # to 5, the scale of 0.36 and the four heads of dK: 4e-4 at most
    assert np.abs(download(dq)).max() <= 4e-4 and np.abs(download(dk)).max() <= 4e-4


@pytest.mark.parametrize("dtype,dim,lengths,shift,forward,backward", [
    ("bfloat16", 64, [70, 3], 0, True, True), ("bfloat16", 64, [70, 3], 1, False, False), ("bfloat16", 20, [70, 3], 0, False, False),
    ("bfloat16", 64, [2, 3], 0, True, True),  # queries in tiles, keys one at a time
    ("bfloat16", 136, [70, 3], 0, True, True), ("bfloat16", 136, [20, 3], 0, False, False),
    ("float32", 64, [70, 3], 0, True, True), ("float32", 64, [20, 3], 0, False, False), ("float32", 160, [70, 3], 0, False, False)])
def test_what_counts_as_a_launch_on_the_matrix_cores(dtype, dim, lengths, shift, forward, backward):
    """The calls whose rows are worked on in tiles, in one of the passes at least."""
    runtime, packing, heads, kv_heads = amd.get_runtime(), Packing(lengths), 4, 2
    q, k, v, g = (shifted(normal(95 + i, packing.total * n * dim), dtype, shift)
                  for i, n in enumerate((heads, kv_heads, kv_heads, heads)))
    dims = (packing, heads, kv_heads, dim)
    before = runtime.mfma_launches
    out, lse = amd_lm.attention_packed(q, k, v, *dims)
    assert runtime.mfma_launches - before == forward
    before = runtime.mfma_launches
    amd_lm.attention_packed_backward(g, q, k, v, out, lse, *dims)
    assert runtime.mfma_launches - before == backward
