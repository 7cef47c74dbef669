"""The quantised key and value cache: the values that its codes stand for are the
definition's exactly (ties, tiny and huge rows, infinities and NaN among them),
positions and counts of each sequence are kept to, and attention over it agrees
with float64 attention of those values."""
import numpy as np
import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd, amd_lm
from qutai_amd.nn import MultiHeadAttention, QuantizedKVCache
from tests.helpers import download, stored, upload

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24  # half a step of fp32


def held(x, bits):
    """The float64 values that codes of ``bits`` stand for, for rows (..., dim)."""
    x = np.asarray(x, dtype=np.float64)
    most, group = (127, x.shape[-1]) if bits == 8 else (7, 32)
    out = np.empty_like(x)
    for start in range(0, x.shape[-1], group):
        part = x[..., start:start + group]
        with np.errstate(invalid="ignore"):
            amax = np.abs(part).max(-1, keepdims=True)
            fraction, exponent = np.frexp(amax / most)
            scale = np.maximum(np.ldexp(np.ceil(fraction * 256), exponent - 8), 2.0 ** -100)
            scale = np.where(np.isfinite(amax), scale, np.nan)
            out[..., start:start + group] = np.rint(part / scale) * scale
    return out


def as_tensor(x, dtype):
    return Tensor(upload(x, dtype), shape=x.shape)


def read(cache, dtype="float32"):
    return [download(x.storage).reshape(x.shape) for x in cache.read(dtype)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch,new,kv_heads,dim", [(1, 1, 1, 1), (2, 3, 2, 5), (1, 4, 3, 32), (2, 5, 1, 40), (3, 2, 2, 64),
                                                    (1, 7, 2, 80), (2, 3, 1, 96), (1, 9, 2, 128), (1, 3, 3, 160), (2, 2, 1, 256)])
def test_written_values_are_the_definitions(bits, dtype, batch, new, kv_heads, dim):
    rng = np.random.default_rng(dim + new)
    k, v = (stored(rng.standard_normal((batch, new, kv_heads, dim)) * 3, dtype) for _ in range(2))
    cache = QuantizedKVCache(new + 2, bits=bits)
    cache.append(as_tensor(k, dtype), as_tensor(v, dtype))
    assert cache.lengths == (new,) * batch
    for got, x in zip(read(cache), (k, v)):
        assert np.array_equal(got, held(x, bits).transpose(0, 2, 1, 3))
    for got, x in zip(read(cache, "bfloat16"), (k, v)):
        assert np.array_equal(got, stored(held(x, bits), "bfloat16").transpose(0, 2, 1, 3))


@pytest.mark.parametrize("bits", [8, 4])
def test_ties_extremes_and_what_is_not_finite(bits):
    most = 127 if bits == 8 else 7
    dim = 32
    rows = np.zeros((12, dim))
    halves = np.arange(dim) % most - 0.5  # codes halfway between two, scale 1: half to even
    rows[0], rows[1] = halves, -halves
    rows[0, 0] = rows[1, 0] = most
    rows[2] = 1e38 * np.cos(np.arange(dim))
    rows[3] = 1e-38 * np.cos(np.arange(dim))  # below the smallest scale: zeros
    rows[4] = 2.0 ** -100 * np.arange(dim) / 4
    rows[6, 3], rows[7, 4], rows[8, 5] = np.inf, -np.inf, np.nan
    rows[8, 6] = 1.0
    rows[9] = np.nextafter(np.float32(most), np.float32(0)) * np.ones(dim)
    rows[10] = np.nextafter(np.float32(most), np.float32(1e9)) * np.ones(dim)  # just above: the next scale
    rows[11] = np.random.default_rng(0).standard_normal(dim) * np.float32(3.4e38) / 6
    x = rows.astype(np.float32)[None, :, None]
    cache = QuantizedKVCache(12, bits=bits)
    cache.append(as_tensor(x, "float32"), as_tensor(-x, "float32"))
    expected = held(x, bits).transpose(0, 2, 1, 3)
    keys, values = read(cache)
    assert np.array_equal(keys, expected, equal_nan=True) and np.array_equal(values, -expected, equal_nan=True)
    assert np.isnan(keys[0, 0, 6:9]).all() and not np.isnan(np.delete(keys, (6, 7, 8), axis=2)).any()
    assert (keys[0, 0, 3] == 0).all() and (keys[0, 0, 5] == 0).all()


def test_lengths_counts_and_truncation():
    rng = np.random.default_rng(4)
    cache, kept = QuantizedKVCache(16), [np.zeros((0, 2, 8)) for _ in range(3)]

    def add(new, counts=None):
        x = stored(rng.standard_normal((3, new, 2, 8)), "float32")
        cache.append(as_tensor(x, "float32"), as_tensor(2 * x, "float32"), counts)
        for b, n in enumerate((new,) * 3 if counts is None else counts):
            kept[b] = np.concatenate((kept[b], x[b, :n]))
        check()

    def check():
        assert cache.lengths == tuple(len(x) for x in kept)
        keys, values = read(cache)
        for b, x in enumerate(kept):
            expected = held(x, 8).transpose(1, 0, 2)
            assert np.array_equal(keys[b, :, :len(x)], expected) and np.array_equal(values[b, :, :len(x)], 2 * expected)
            assert (keys[b, :, len(x):] == 0).all() and (values[b, :, len(x):] == 0).all()

    add(4, (4, 0, 2))
    add(1)
    add(3, [1, 3, 0])
    add(2)
    cache.truncate((3, 1, 4))
    kept[:] = [x[:n] for x, n in zip(kept, (3, 1, 4))]
    check()
    add(5)
    cache.truncate(2)
    kept[:] = [x[:2] for x in kept]
    check()
    add(14)
    with pytest.raises(ValueError):
        add(1)
    for counts in ((1, 2), (2, 0, 0), (-1, 0, 0), (1.0, 1, 1)):
        cache.truncate(0)
        with pytest.raises(ValueError):
            cache.append(*(as_tensor(np.ones((3, 1, 2, 8)), "float32") for _ in range(2)), counts)
    for lengths in (1, (0, 0, 1), (0, 0)):
        with pytest.raises(ValueError):
            cache.truncate(lengths)


def test_columns_of_a_product_and_positions_outside():
    """Keys and values as columns of wider rows; positions before 0 and from the
    capacity on are not written."""
    rng = np.random.default_rng(6)
    batch, new, heads, dim, capacity = 2, 3, 2, 24, 8
    row = 3 * heads * dim + 5
    block = stored(rng.standard_normal((batch * new, row)), "bfloat16")
    for start, starts in ((0, None), (6, None), (-1, [0, 8])):
        cache = amd_lm.QuantizedCache(batch, heads, dim, capacity, 8)
        for codes in (cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales):
            codes.runtime.call("qutai_amd_fill", codes.ptr, codes.nbytes // 4, 0.0, amd.code("float32"))
        source = upload(block, "bfloat16")
        amd_lm.cache_quantize(cache, source, source, new, start=start,
                              starts=None if starts is None else amd.storage(starts, dtype="int64"),
                              key_column=heads * dim + 2, key_row=row, value_column=2 * heads * dim + 5, value_row=row)
        got = amd_lm.cache_dequantize(cache, capacity)
        for values, column in zip(got, (heads * dim + 2, 2 * heads * dim + 5)):
            x = held(block[:, column:column + heads * dim].reshape(batch, new, heads, dim), 8)
            expected = np.zeros((batch, capacity, heads, dim))
            for b in range(batch):
                for t in range(new):
                    at = start + t + (0 if starts is None else starts[b])
                    if 0 <= at < capacity:
                        expected[b, at] = x[b, t]
            assert np.array_equal(download(values).reshape(batch, heads, capacity, dim), expected.transpose(0, 2, 1, 3))


ATTEND = [
    # dtype, bits, batch, heads, kv_heads, dim, past (one for all, or each), new
    ("float32", 8, 1, 1, 1, 1, 0, 1), ("float32", 8, 2, 3, 3, 5, 6, 2), ("float32", 4, 1, 4, 2, 32, 40, 1),
    ("float32", 8, 2, 2, 1, 64, 129, 3), ("float32", 4, 1, 2, 2, 80, (63,), 4), ("float32", 8, 1, 4, 2, 128, 700, 1),
    ("float32", 4, 2, 2, 1, 256, (64, 3), 2), ("float32", 8, 3, 8, 8, 64, (1000, 0, 17), 1), ("float32", 8, 1, 2, 1, 96, 0, 70),
    ("bfloat16", 8, 1, 16, 4, 64, 1000, 1), ("bfloat16", 8, 4, 8, 2, 64, (5, 31, 32, 33), 1), ("bfloat16", 4, 2, 8, 2, 128, (300, 511), 1),
    ("bfloat16", 8, 1, 32, 1, 64, 65, 1), ("bfloat16", 8, 2, 5, 1, 40, 127, 7), ("bfloat16", 4, 1, 24, 2, 64, 2000, 3),
    ("bfloat16", 8, 1, 4, 4, 256, 515, 2), ("bfloat16", 4, 1, 4, 4, 192, 15, 2), ("bfloat16", 8, 2, 4, 1, 128, 0, 130),
    ("bfloat16", 8, 1, 8, 2, 64, 100, 67), ("bfloat16", 4, 2, 4, 2, 32, (0, 90), 33), ("bfloat16", 8, 1, 2, 2, 64, 9000, 1),
    ("bfloat16", 4, 1, 2, 1, 96, 5000, 1), ("float32", 4, 1, 3, 1, 160, 33, 20),
]


def raised_scales(x):
    """24 times an upper bound of each value's scale where codes have 4 bits: the
    largest code of a group is 6.5 at least (its scale is the smallest that
    holds it, 2^-7 too large at most), so a sixth of the largest value."""
    out = np.empty_like(x)
    for start in range(0, x.shape[-1], 32):
        out[..., start:start + 32] = 4 * np.abs(x[..., start:start + 32]).max(-1, keepdims=True)
    return out


def check_attention(out, q, k, v, starts, counts, scale, dtype, bits=8):
    """out (batch, new, heads, dim) against float64 attention over the held k, v
    (batch, kv_heads, length, dim).  The bf16 kernels hold codes of 4 bits as
    code + 24 and take the 24 off a product of 32 channels, or of a block of 32
    keys, again: 16 additions (of 8 products each, and of two parts) are then
    rounded at up to 24 scales, not at the codes' own size."""
    batch, new, heads, dim = q.shape
    group = heads // k.shape[1]
    # a weight reaches the value product as two bf16 parts (half a step of 16 bits together) or three
    parts = 2.0 ** -16 if dtype == "bfloat16" else 4 * UNIT
    for b in range(batch):
        n, total = counts[b], starts[b] + counts[b]
        assert (out[b, n:] == 0).all()
        if not n:
            continue
        for h in range(heads):
            keys, values = k[b, h // group, :total], v[b, h // group, :total]
            s = q[b, :n, h] @ keys.T * scale
            hidden = np.arange(total)[None] > starts[b] + np.arange(n)[:, None]
            s[hidden] = -np.inf
            x = s - s.max(axis=1, keepdims=True)
            p = np.exp(x)
            p /= p.sum(axis=1, keepdims=True)
            expected = p @ values
            # a score's roundings (padded width, both scales, parts of q), the exponential's argument and itself
            size = np.abs(q[b, :n, h]) @ np.abs(keys).T * scale
            arg = np.where(hidden, 0.0, np.abs(x))
            moved = UNIT * ((dim + 40) * (size + size.max(axis=1, keepdims=True)) + 4 * arg + 8) + parts
            raised = dtype == "bfloat16" and bits == 4
            if raised:
                moved += 16 * UNIT * scale * np.abs(q[b, :n, h]) @ raised_scales(keys).T
            bound = (p * (moved + (p * moved).sum(axis=1, keepdims=True) + 2 * (total + 40) * UNIT)) @ np.abs(values)
            bound += 4 * UNIT * np.abs(expected)
            if raised:
                bound += 16 * UNIT * p @ raised_scales(values)
            if dtype == "bfloat16":
                bound += 2.0 ** -8 * (np.abs(expected) + bound)
            assert (np.abs(out[b, :n, h] - expected) <= bound).all(), (b, h)


@pytest.mark.parametrize("dtype,bits,batch,heads,kv_heads,dim,past,new", ATTEND)
def test_attention_matches_float64(dtype, bits, batch, heads, kv_heads, dim, past, new):
    rng = np.random.default_rng(dim + new + heads)
    starts = (past,) * batch if isinstance(past, int) else past
    longest = max(starts)
    cache = QuantizedKVCache(longest + new + 3, bits=bits)
    if longest:
        old = [as_tensor(rng.standard_normal((batch, longest, kv_heads, dim)), dtype) for _ in range(2)]
        cache.append(*old, starts)
    else:
        cache.reserve(batch, kv_heads, dim)
    fresh = [as_tensor(rng.standard_normal((batch, new, kv_heads, dim)), dtype) for _ in range(2)]
    q = stored(rng.standard_normal((batch, new, heads, dim)) * 2, dtype)
    for counts in ((new,) * batch, tuple(max(0, new - b - 1) for b in range(batch))):
        cache.truncate(starts)
        cache.append(*fresh, counts)
        out = cache.attend(as_tensor(q, dtype))
        assert out.dtype == dtype and out.shape == q.shape
        k, v = read(cache) if cache.length else [np.zeros((batch, kv_heads, 0, dim))] * 2
        check_attention(download(out.storage).reshape(q.shape), q, k, v, starts, counts, dim ** -0.5, dtype, bits)


PAIRS = [("bfloat16", 8, 64), ("bfloat16", 4, 64), ("bfloat16", 4, 128), ("bfloat16", 8, 128), ("bfloat16", 4, 256),
         ("bfloat16", 8, 192), ("float32", 8, 64)]


@pytest.mark.parametrize("dtype,bits,dim", PAIRS)
@pytest.mark.parametrize("heads,new", [(3, 1), (1, 4), (2, 2)])
def test_sequences_that_end_around_blocks_and_pairs_of_them(dtype, bits, dim, heads, new):
    """Four rows or fewer: two blocks of 32 keys beside each other, the second of
    which may hold nothing, at a split's end and at the capacity's."""
    past = (0, 30, 31, 32, 33, 62, 63, 64, 65, 95, 96, 97, 255, 256, 287, 288, 289, 511, 512 - new)
    test_attention_matches_float64(dtype, bits, len(past), heads, 1, dim, past, new)


@pytest.mark.parametrize("bits,dim", [(4, 256), (4, 200), (8, 256)])
def test_many_rows_of_wide_heads(bits, dim):
    test_attention_matches_float64("bfloat16", bits, 2, 4, 2, dim, (70, 129), 37)


@pytest.mark.parametrize("bits", [8, 4])
def test_what_lies_behind_a_sequence_does_not_leak(bits):
    """Scales of NaN and infinity behind the visible positions, and a poisoned
    position that only later queries see."""
    rng = np.random.default_rng(8)
    cache = QuantizedKVCache(100, bits=bits)
    junk = np.full((2, 100, 1, 64), np.nan)
    cache.append(as_tensor(junk, "float32"), as_tensor(junk, "float32"))
    cache.truncate(0)
    k, v = (stored(rng.standard_normal((2, 37, 1, 64)), "float32") for _ in range(2))
    cache.append(as_tensor(k, "float32"), as_tensor(v, "float32"), (37, 11))
    q = stored(rng.standard_normal((2, 37, 2, 64)), "float32")
    out = download(cache.attend(as_tensor(q, "float32")).storage).reshape(q.shape)
    check_attention(out, q, *read(cache), (0, 0), (37, 11), 0.125, "float32")
    k[0, 20] = np.inf
    cache.truncate(0)
    cache.append(as_tensor(k, "float32"), as_tensor(v, "float32"))
    out = download(cache.attend(as_tensor(q, "float32")).storage).reshape(q.shape)
    assert np.isfinite(out[0, :20]).all() and np.isnan(out[0, 20:]).all() and np.isfinite(out[1]).all()


def test_large_scores_and_scales():
    """Scores of some thousands, and rows of values whose scales lie 2^80 apart."""
    rng = np.random.default_rng(9)
    k, v = (stored(rng.standard_normal((1, 90, 1, 32)) * 30, "float32") for _ in range(2))
    v *= np.where(np.arange(90) % 3 == 0, 2.0 ** 60, 2.0 ** -20)[None, :, None, None]
    q = stored(rng.standard_normal((1, 1, 4, 32)) * 30, "float32")
    cache = QuantizedKVCache(91)
    cache.append(as_tensor(k[:, :89], "float32"), as_tensor(v[:, :89], "float32"))
    cache.append(as_tensor(k[:, 89:], "float32"), as_tensor(v[:, 89:], "float32"))
    out = download(cache.attend(as_tensor(q, "float32")).storage).reshape(q.shape)
    check_attention(out, q, *read(cache), (89,), (1,), 32 ** -0.5, "float32")


@pytest.mark.parametrize("bits", [8, 4])
def test_the_largest_magnitudes(bits):
    """fp32's largest number: 8 bits hold it; with 4 bits 7 times the scale that
    holds what lies above 3.396e38 is beyond fp32, and infinity."""
    most = float(np.finfo(np.float32).max)
    x = np.zeros((1, 3, 1, 32), dtype=np.float32)
    x[0, :, 0, 3] = most, 3.3961e38, -3.39e38
    cache = QuantizedKVCache(3, bits=bits)
    cache.append(as_tensor(x, "float32"), as_tensor(x, "float32"))
    exact = held(x, bits)
    expected = np.where(np.abs(exact) > most, np.copysign(np.inf, exact), exact).transpose(0, 2, 1, 3)
    assert all(np.array_equal(got, expected) for got in read(cache))
    assert np.isfinite(expected).all() == (bits == 8) and np.isfinite(expected[0, 0, 1:]).all()


@pytest.mark.parametrize("dtype,bits", [("float32", 8), ("float32", 4), ("bfloat16", 8), ("bfloat16", 4)])
def test_sums_of_large_values_stay_in_range(dtype, bits):
    """Values of 1e27, keys whose scores rise by less than 2^8 along the sequence,
    so that weights above 1 are summed."""
    rng = np.random.default_rng(16)
    k, v = np.zeros((1, 3000, 1, 32)), 1e27 * (1 - 0.2 * rng.random((1, 3000, 1, 32)))
    k[..., 0] = np.linspace(0, 30, 3000)[None, :, None]
    cache = QuantizedKVCache(3000, bits=bits)
    cache.append(as_tensor(k[:, :2999], dtype), as_tensor(v[:, :2999], dtype))
    cache.append(as_tensor(k[:, 2999:], dtype), as_tensor(v[:, 2999:], dtype))
    q = np.zeros((1, 1, 2, 32))
    q[..., 0] = 1.0
    out = download(cache.attend(as_tensor(q, dtype)).storage).reshape(q.shape)
    check_attention(out, q, *read(cache), (2999,), (1,), 32 ** -0.5, dtype, bits)


@pytest.mark.parametrize("bits", [8, 4])
def test_rows_beyond_four_gigabytes(bits):
    """The last heads' codes lie behind the 32-bit offsets."""
    rng = np.random.default_rng(10)
    heads, capacity = (66, 1 << 18) if bits == 8 else (132, 1 << 18)
    cache = QuantizedKVCache(capacity, bits=bits)
    k, v = (stored(rng.standard_normal((1, 3, heads, 256)), "bfloat16") for _ in range(2))
    cache.append(as_tensor(k[:, :2], "bfloat16"), as_tensor(v[:, :2], "bfloat16"))
    cache.append(as_tensor(k[:, 2:], "bfloat16"), as_tensor(v[:, 2:], "bfloat16"))
    assert cache.codes.key_codes.nbytes > 1 << 32
    for got, x in zip(read(cache), (k, v)):
        assert np.array_equal(got, held(x, bits).transpose(0, 2, 1, 3))
    q = stored(rng.standard_normal((1, 1, heads, 256)), "bfloat16")
    out = download(cache.attend(as_tensor(q, "bfloat16")).storage).reshape(q.shape)
    check_attention(out, q, *read(cache), (2,), (1,), 1 / 16, "bfloat16", bits)


@pytest.mark.parametrize("bits,dtype", [(8, "bfloat16"), (4, "bfloat16"), (8, "float32")])
def test_decoding_over_the_length_at_which_the_split_changes(bits, dtype):
    """512 (sequence, head) pairs, one position at a time past 4096 keys, from
    where on each takes twice the ranges."""
    rng = np.random.default_rng(15)
    batch, kv_heads, dim, past = 64, 8, 8, 4094
    cache = QuantizedKVCache(4100, bits=bits)
    old = [rng.standard_normal((batch, past, kv_heads, dim), dtype=np.float32) for _ in range(2)]
    cache.append(*(as_tensor(x, dtype) for x in old), (past,) + tuple(range(past - 63, past)))
    starts = cache.lengths
    steps = []
    for _ in range(4):
        cache.append(*(as_tensor(rng.standard_normal((batch, 1, kv_heads, dim)), dtype) for _ in range(2)))
        q = stored(rng.standard_normal((batch, 1, 2 * kv_heads, dim)) * 2, dtype)
        steps.append((q, download(cache.attend(as_tensor(q, dtype)).storage).reshape(q.shape)))
    some = [0, 1, 30, 63]
    k, v = (x[some] for x in read(cache))
    for i, (q, out) in enumerate(steps):
        check_attention(out[some], q[some], k, v, [starts[b] + i for b in some], (1,) * 4, dim ** -0.5, dtype, bits)


def test_no_new_positions_and_counts_of_the_library():
    """An append of nothing; counts above the new positions and below none, as the
    library's callers may pass them."""
    rng = np.random.default_rng(14)
    cache = QuantizedKVCache(40)
    k, v = (stored(rng.standard_normal((3, 6, 2, 32)), "float32") for _ in range(2))
    cache.append(as_tensor(k, "float32"), as_tensor(v, "float32"))
    empty = Tensor(amd.AMDStorage(0, "float32"), shape=(3, 0, 2, 32))
    cache.append(empty, empty)
    assert cache.lengths == (6, 6, 6) and cache.attend(empty).shape == (3, 0, 2, 32)
    q = stored(rng.standard_normal((3, 6, 4, 32)), "float32")
    counts = amd.storage([1 << 62, -(1 << 62), 4], dtype="int64")
    out = amd_lm.attention_quantized(cache.codes, upload(q, "float32"), 6, 4, counts=counts, longest=6)
    check_attention(download(out).reshape(q.shape), q, *read(cache), (0, 0, 0), (6, 0, 4), 32 ** -0.5, "float32")


@pytest.mark.parametrize("dtype,bits,dim", [("bfloat16", 8, 64), ("float32", 4, 256), ("bfloat16", 4, 5)])
def test_attention_counts_as_a_launch_on_the_matrix_cores(dtype, bits, dim):
    cache, runtime = QuantizedKVCache(8, bits=bits), amd.get_runtime()
    x = as_tensor(np.ones((1, 2, 1, dim)), dtype)
    cache.append(x, x)
    before = runtime.mfma_launches
    cache.attend(x)
    assert runtime.mfma_launches == before + 1


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(3)
    cache = QuantizedKVCache(4000)
    cache.append(*(as_tensor(rng.standard_normal((2, 3999, 2, 64)), "bfloat16") for _ in range(2)), (3999, 1234))
    cache.append(*(as_tensor(rng.standard_normal((2, 1, 2, 64)), "bfloat16") for _ in range(2)))
    q = as_tensor(rng.standard_normal((2, 1, 8, 64)), "bfloat16")
    first = cache.attend(q).storage.to_array()
    assert all(cache.attend(q).storage.to_array() == first for _ in range(4))


@pytest.mark.parametrize("bits,dtype", [(8, "float32"), (8, "bfloat16"), (4, "float32")])
def test_multi_head_attention_over_a_quantised_cache(bits, dtype):
    """The layer's inference with a quantised cache, in parts of 5, 1 and 3
    positions, against its own products over the values that the cache holds."""
    rng = np.random.default_rng(12)
    layer = MultiHeadAttention(32, 4, causal=True, seed=1, dtype=dtype)
    cache = QuantizedKVCache(9, bits=bits)
    for new in (5, 1, 3):
        x = stored(rng.standard_normal((2, new, 32)), dtype)
        start = cache.length
        y = layer(as_tensor(x, dtype), cache=cache)
        assert cache.length == start + new and not y.requires_grad
        q = layer.query(as_tensor(x, dtype))
        q = download(q.storage).reshape(2, new, 4, 8)
        k, v = read(cache)
        out = np.empty((2, new, 4, 8))
        for b in range(2):
            for h in range(4):
                s = q[b, :, h] @ k[b, h].T * 8 ** -0.5
                s[np.arange(start + new)[None] > start + np.arange(new)[:, None]] = -np.inf
                p = np.exp(s - s.max(1, keepdims=True))
                out[b, :, h] = p / p.sum(1, keepdims=True) @ v[b, h]
        w = download(layer.output.weight.storage).reshape(32, 32)
        expected = stored(out.reshape(2, new, 32), dtype) @ w + download(layer.output.bias.storage)
        # bf16: the mixed rows' and the result's roundings; fp32: sums of a few hundred terms
        limit = 3 * 2.0 ** -8 if dtype == "bfloat16" else 400 * UNIT
        scale = np.abs(out.reshape(2, new, 32)) @ np.abs(w) + np.abs(expected)
        assert (np.abs(download(y.storage).reshape(2, new, 32) - expected) <= limit * scale).all()
    with pytest.raises(ValueError):
        MultiHeadAttention(32, 4, seed=1, dtype=dtype)(as_tensor(x, dtype), cache=cache)
    with pytest.raises(ValueError):
        layer(as_tensor(x, dtype), cache=cache)  # the capacity is used up


def test_attend_refuses():
    cache = QuantizedKVCache(8)
    with pytest.raises(ValueError):
        cache.read()
    with pytest.raises(ValueError):
        cache.attend(as_tensor(np.ones((1, 1, 2, 8)), "float32"))
    ones = as_tensor(np.ones((1, 2, 2, 8)), "float32")
    cache.append(ones, ones)
    for shape in ((1, 1, 2, 8), (2, 2, 2, 8), (1, 2, 3, 8), (1, 2, 2, 4)):
        with pytest.raises(ValueError):
            cache.attend(as_tensor(np.ones(shape), "float32"))
    for bad in ((np.ones((1, 2, 1, 8)),) * 2, (np.ones((1, 2, 2, 8)), np.ones((1, 1, 2, 8))), (np.ones((2, 2, 8)),) * 2):
        with pytest.raises(ValueError):
            cache.append(*(as_tensor(x, "float32") for x in bad))
    cache.truncate(1)
    with pytest.raises(ValueError):
        cache.attend(ones)
