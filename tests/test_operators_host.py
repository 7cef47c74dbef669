"""Arguments that the decoder operators refuse, before any device call: the
Python checks, and the C entry points' own (stand-in pointers that are never
followed)."""
from itertools import count
from math import prod
from pathlib import Path
from types import SimpleNamespace

import pytest

from qutai_amd import Tensor
from qutai_amd.backends import amd, amd_lm, amd_runtime
from qutai_amd.lm import Config, decoder, qk_norm_rope
from qutai_amd.nn import QuantizedKVCache

LIBRARY = Path(__file__).resolve().parent.parent / "qutai_amd" / "libqutai_amd.so"
built = pytest.mark.skipif(not LIBRARY.exists(), reason="libqutai_amd.so not built")
FAKE = 1 << 20


ADDRESSES = count(FAKE, FAKE)


class _Runtime:
    def free(self, ptr):
        pass


def fake(size, dtype):
    """A storage shell with no device allocation, each at an address of its own."""
    storage = object.__new__(amd.AMDStorage)
    storage.dtype, storage._size, storage.ptr, storage.runtime = dtype, size, next(ADDRESSES), _Runtime()
    return storage


def qk_call(**change):
    a = dict(q=fake(2 * 3 * 4 * 8, "bfloat16"), k=fake(2 * 3 * 2 * 8, "bfloat16"), q_weight=fake(8, "float32"),
             k_weight=fake(8, "float32"), batch=2, time=3, heads=4, kv_heads=2, dim=8, theta=1e4, eps=1e-6)
    a.update(change)
    return amd_lm.qk_norm_rope(**a)


@pytest.mark.parametrize("change", [
    dict(dim=7), dict(dim=0), dict(dim=258), dict(heads=0, kv_heads=0), dict(heads=-1), dict(batch=-1), dict(time=-2),
    dict(q=fake(8, "bfloat16")), dict(k=fake(96, "float32")), dict(q=fake(192, "int64"), k=fake(96, "int64")),
    dict(q_weight=None), dict(k_weight=None), dict(q_weight=fake(8, "bfloat16")), dict(k_weight=fake(7, "float32")),
    dict(starts=fake(2, "float32")), dict(starts=fake(3, "int64")), dict(q_column=1), dict(q_row=31), dict(k_column=-1),
])
def test_qk_norm_rope_refuses(change):
    with pytest.raises(ValueError):
        qk_call(**change)


@pytest.mark.parametrize("q,k,heads,kv_heads", [
    ((2, 3, 32), (1, 6, 16), 4, 2), ((2, 3, 32), (3, 2, 16), 4, 2), ((2, 3, 32), (2, 3, 16), 4, 4), ((2, 3, 32), (2, 3, 24), 4, 2),
    ((2, 3, 32), (2, 6, 16), 4, 2), ((2, 3, 34), (2, 3, 16), 4, 2), ((6, 32), (6, 16), 4, 2), ((2, 3, 32), (6, 16), 4, 2),
    ((2, 3, 32), (2, 3, 16), 0, 2),
])
def test_recorded_qk_norm_rope_refuses_other_shapes(q, k, heads, kv_heads):
    """Keys of as many values in other sequences or positions among them, which
    would be turned by the positions of the queries."""
    q, k, *weights = (Tensor(fake(prod(shape), "float32"), shape=shape) for shape in (q, k, (8,), (8,)))
    with pytest.raises(ValueError, match="qk_norm_rope takes q"):
        qk_norm_rope(q, k, *weights, heads, kv_heads, 1e4, 1e-6)


def test_qk_norm_rope_backward_refuses():
    def call(**change):
        a = dict(gq=fake(192, "bfloat16"), gk=fake(96, "bfloat16"), q=fake(192, "bfloat16"), k=fake(96, "bfloat16"),
                 q_weight=fake(8, "float32"), k_weight=fake(8, "float32"), batch=2, time=3, heads=4, kv_heads=2, dim=8,
                 theta=1e4, eps=1e-6)
        a.update(change)
        return amd_lm.qk_norm_rope_backward(**a)

    for change in (dict(gq=fake(191, "bfloat16")), dict(gk=fake(96, "float32")),
                   dict(out=fake(288, "bfloat16")),  # q and k are apart: one row does not hold both
                   dict(q=fake(6 * 48, "bfloat16"), k=fake(6 * 48, "bfloat16"), q_row=48, k_column=8, k_row=48,
                        out=fake(6 * 48, "bfloat16"))):  # overlapping columns
        with pytest.raises(ValueError):
            call(**change)


@built
def test_qk_norm_rope_entry_points_refuse():
    library = amd_runtime.load_library()

    def forward(q=FAKE, k=FAKE, wq=FAKE, wk=FAKE, q_out=FAKE, k_out=FAKE, starts=None, offset=0, batch=2, time=3,
                heads=4, kv_heads=2, dim=8, q_row=32, k_row=16, theta=1e4, eps=1e-6, dtype=5):
        return library.qutai_amd_qk_norm_rope(q, k, wq, wk, q_out, k_out, starts, offset, batch, time, heads, kv_heads,
                                              dim, q_row, k_row, theta, eps, dtype, None)

    for change in (dict(dim=7), dict(dim=258), dict(dim=0), dict(heads=0, kv_heads=0), dict(heads=-4), dict(batch=-1),
                   dict(time=-1), dict(q_row=31), dict(k_row=15), dict(theta=0.0), dict(theta=float("nan")),
                   dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=1), dict(dtype=4), dict(q=None), dict(k_out=None),
                   dict(wq=None), dict(wk=None), dict(batch=1 << 30, time=1 << 30), dict(offset=1 << 60),
                   dict(q_row=1 << 50), dict(batch=1 << 25, q_row=1 << 40)):
        assert forward(**change) == amd_runtime.QA_EINVAL, change
    assert forward(batch=0, q=None, k=None) == 0  # nothing to do
    back = library.qutai_amd_qk_norm_rope_backward
    rest = (None, 0, 2, 3, 4, 2, 8, 32, 16, 32, 16, 1e4, 1e-6, 5)
    p = FAKE
    assert back(p, p, p, p, p, p, p, p, p, p, *rest, None, 0, None) == amd_runtime.QA_EWORKSPACE
    assert back(p, p, p, p, p, p, p, p, p, p, *rest, p, 7, None) == amd_runtime.QA_EWORKSPACE
    assert back(None, p, p, p, p, p, p, p, p, p, *rest, p, 1 << 20, None) == amd_runtime.QA_EINVAL
    assert back(p, p, p, p, None, None, p, p, p, p, *rest, p, 1 << 20, None) == amd_runtime.QA_EINVAL
    assert library.qutai_amd_qk_norm_rope_workspace(0) == 0 and library.qutai_amd_qk_norm_rope_workspace(64) > 0


def test_config_with_normed_heads():
    plain, normed = Config(d_model=64, n_heads=4, n_kv_heads=2), Config(d_model=64, n_heads=4, n_kv_heads=2, qk_norm=True)
    assert "qk_norm" not in plain.to_dict() and normed.to_dict()["qk_norm"] is True
    assert Config(**normed.to_dict()) == normed and Config(**plain.to_dict()) == plain
    extra = normed.parameter_counts()["total_parameters"] - plain.parameter_counts()["total_parameters"]
    assert extra == plain.n_layers * 2 * 16
    with pytest.raises(ValueError):
        Config(qk_norm=1)


# ---- the quantised cache -----------------------------------------------------------

def fake_cache(batch=2, kv_heads=2, dim=8, capacity=10, bits=8):
    cache = object.__new__(amd_lm.QuantizedCache)
    cache.batch, cache.kv_heads, cache.dim, cache.capacity, cache.bits = batch, kv_heads, dim, capacity, bits
    return cache


def test_a_cache_of_impossible_sizes_is_refused():
    for sizes in ((2, 2, 8, 10, 2), (0, 2, 8, 10, 8), (2, 0, 8, 10, 8), (2, 2, 0, 10, 8), (2, 2, 257, 10, 8), (2, 2, 8, 0, 4)):
        with pytest.raises(ValueError):
            amd_lm.QuantizedCache(*sizes)
    for arguments in ((0, 8), (-3, 8), (8, 16), (2.0, 8)):
        with pytest.raises(ValueError):
            QuantizedKVCache(arguments[0], bits=arguments[1])
    cache = QuantizedKVCache(8)
    cache.truncate(0)
    assert cache.length == 0
    for lengths in (1, (1, 0)):
        with pytest.raises(ValueError):
            cache.truncate(lengths)


@pytest.mark.parametrize("change", [
    dict(new=-1), dict(keys=fake(96, "float32")), dict(keys=fake(96, "int64"), values=fake(96, "int64")),
    dict(values=fake(95, "bfloat16")), dict(key_column=1), dict(value_row=15), dict(starts=fake(3, "int64")),
    dict(counts=fake(2, "float32")),
])
def test_cache_quantize_refuses(change):
    a = dict(cache=fake_cache(), keys=fake(96, "bfloat16"), values=fake(96, "bfloat16"), new=3)
    with pytest.raises(ValueError):
        amd_lm.cache_quantize(**{**a, **change})


@pytest.mark.parametrize("change", [
    dict(q=fake(192, "int64")), dict(q=fake(191, "float32")), dict(heads=3), dict(heads=0), dict(new=-1), dict(longest=11),
    dict(starts=fake(1, "int64")), dict(counts=fake(2, "bfloat16")),
])
def test_attention_quantized_refuses(change):
    a = dict(cache=fake_cache(), q=fake(2 * 3 * 4 * 8, "float32"), new=3, heads=4)
    with pytest.raises(ValueError):
        amd_lm.attention_quantized(**{**a, **change})


def test_cache_dequantize_refuses():
    for change in (dict(length=11), dict(length=-1), dict(length=4, dtype="float64"), dict(length=4, lengths=fake(3, "int64"))):
        with pytest.raises(ValueError):
            amd_lm.cache_dequantize(fake_cache(), **change)


@built
def test_cache_entry_points_refuse():
    library, p = amd_runtime.load_library(), FAKE

    def write(key_codes=p, start=0, batch=2, new=3, heads=2, dim=8, capacity=10, key_row=16, value_row=16, bits=8, dtype=5,
              keys=p):
        return library.qutai_amd_cache_quantize(keys, p, key_codes, p, p, p, None, None, start, batch, new, heads, dim,
                                                capacity, key_row, value_row, bits, dtype, None)

    for change in (dict(key_codes=p + 8), dict(start=1 << 60), dict(batch=-1), dict(new=-1), dict(heads=0), dict(dim=257),
                   dict(dim=0), dict(capacity=0), dict(key_row=15), dict(value_row=15), dict(bits=5), dict(dtype=0 + 4),
                   dict(keys=None), dict(batch=1 << 13, new=1 << 13), dict(key_codes=None), dict(capacity=1 << 40)):
        assert write(**change) == amd_runtime.QA_EINVAL, change
    assert write(batch=0) == 0 and write(new=0) == 0

    def read(shift=0, batch=2, heads=2, dim=8, capacity=10, length=4, bits=8, dtype=5, codes=p, out=p):
        return library.qutai_amd_cache_dequantize(codes, p, p, p, out, p, None, shift, batch, heads, dim, capacity, length,
                                                  bits, dtype, None)

    for change in (dict(length=11), dict(length=-1), dict(bits=16), dict(dtype=1), dict(codes=None), dict(codes=p + 4),
                   dict(dim=300), dict(shift=1 << 50), dict(out=None),
                   dict(batch=1 << 12, capacity=1 << 20, length=1 << 18)):
        assert read(**change) == amd_runtime.QA_EINVAL, change

    def attend(q=p, start=0, batch=2, new=3, heads=4, kv_heads=2, dim=8, capacity=1024, longest=1000, bits=8, dtype=5,
               scale=1.0, codes=p, less=0):
        size = library.qutai_amd_attention_quantized_workspace_size(batch, new, heads, kv_heads, dim, longest, dtype) - less
        return library.qutai_amd_attention_quantized(q, codes, p, p, p, p, None, None, start, batch, new, heads, kv_heads,
                                                     dim, capacity, longest, bits, dtype, scale, p, max(size, 0), None)

    for change in (dict(q=None), dict(start=-(1 << 50)), dict(batch=-1), dict(new=-1), dict(heads=3), dict(kv_heads=0),
                   dict(dim=0), dict(dim=257), dict(capacity=0), dict(capacity=1000), dict(longest=1025), dict(bits=3), dict(dtype=4),
                   dict(scale=0.0), dict(scale=float("nan")), dict(codes=p + 8), dict(batch=1 << 12, new=1 << 12)):
        assert attend(**change) == amd_runtime.QA_EINVAL, change
    assert attend(batch=0) == 0 and attend(new=0) == 0
    assert attend(less=4) == amd_runtime.QA_EWORKSPACE
    pitch = library.qutai_amd_cache_pitch
    assert [pitch(d) for d in (0, 1, 32, 33, 80, 100, 129, 193, 256, 257)] == [0, 32, 32, 64, 96, 128, 192, 256, 256, 0]


@built
@pytest.mark.parametrize("scale", [1e-300, 9e-31, -1.0, 2e30])
def test_attention_scales_that_fp32_does_not_hold_are_refused(scale):
    # (below 1e-38 a masked score's -inf would be multiplied by zero)
    library, p = amd_runtime.load_library(), FAKE
    assert library.qutai_amd_attention_quantized(p, p, p, p, p, p, None, None, 3, 2, 3, 4, 2, 8, 32, 32, 8, 5, scale, p,
                                                 1 << 30, None) == amd_runtime.QA_EINVAL


@pytest.mark.parametrize("new, counts", [(5, None), (5, (5, 1)), (3, (1,)), (3, (4, 1)), (3, 4)])
def test_a_refused_first_append_settles_nothing(new, counts):
    cache = QuantizedKVCache(4)
    with pytest.raises(ValueError):
        cache.append_rows(None, None, 2, new, 4, 64, counts)
    assert cache.codes is None and cache.lengths == () and cache.length == 0


@pytest.mark.parametrize("keys, values, columns", [
    (fake(96, "float64"), fake(96, "float64"), {}), (fake(96, "int64"), fake(96, "int64"), {}),
    (fake(96, "float32"), fake(96, "bfloat16"), {}), (fake(95, "float32"), fake(96, "float32"), {}),
    (fake(96, "float32"), fake(96, "float32"), dict(key_row=15)), (fake(96, "float32"), fake(96, "float32"), dict(value_column=1)),
    (fake(96, "float32"), fake(96, "float32"), dict(value_column=-1, value_row=17)),
])
def test_a_first_append_of_wrong_rows_settles_nothing(keys, values, columns, monkeypatch):
    reserved = []
    monkeypatch.setattr(amd_lm, "QuantizedCache", lambda *sizes: reserved.append(sizes) or fake_cache())
    cache = QuantizedKVCache(4)
    with pytest.raises(ValueError):
        cache.append_rows(keys, values, 2, 3, 2, 8, **columns)
    assert not reserved and cache.codes is None and cache.lengths == ()


def stand_in(batch, kv_heads, dim, capacity, bits):
    return SimpleNamespace(batch=batch, kv_heads=kv_heads, dim=dim, capacity=capacity, bits=bits)


def test_an_append_that_the_library_refuses_changes_nothing(monkeypatch):
    refuse = []
    monkeypatch.setattr(amd_lm, "QuantizedCache", stand_in)

    def quantize(*arguments, **options):
        if refuse:
            raise ValueError("refused")

    monkeypatch.setattr(amd_lm, "cache_quantize", quantize)
    rows = fake(2 * 3 * 2 * 8, "float32")
    cache = QuantizedKVCache(32)
    refuse.append(True)
    with pytest.raises(ValueError):
        cache.append_rows(rows, rows, 2, 3, 2, 8)
    assert cache.codes is None and cache.lengths == () and cache.length == 0
    refuse.clear()
    cache.append_rows(rows, rows, 1, 3, 2, 8)  # other sizes than those refused
    refuse.append(True)
    with pytest.raises(ValueError):
        cache.append_rows(rows, rows, 1, 3, 2, 8)
    assert cache.lengths == (3,) and cache._last[:2] == (3, 0)


@pytest.mark.parametrize("failing", [0, 1, 2])
def test_a_decode_step_that_fails_leaves_the_caches(failing, monkeypatch):
    """Three blocks, of which one raises behind its append."""
    monkeypatch.setattr(amd_lm, "QuantizedCache", stand_in)
    monkeypatch.setattr(amd_lm, "cache_quantize", lambda *arguments, **options: None)
    monkeypatch.setattr(decoder, "embed", lambda ids, weight, shape: None)
    rows = fake(2 * 3 * 2 * 8, "float32")

    class FailingBlock:
        fails = False

        def decode(self, hidden, cache, counts):
            cache.append_rows(rows, rows, 2, 3, 2, 8)
            if self.fails:
                raise RuntimeError("out of memory")

    model = object.__new__(decoder.Decoder)
    model.config, model.blocks = Config(max_seq_len=16, n_layers=3), [FailingBlock() for _ in range(3)]
    model.embedding = SimpleNamespace(weight=None)
    caches = model.caches()
    model.blocks[failing].fails = True
    for held in ((), (5, 5)):
        with pytest.raises(RuntimeError):
            model.decode([[1, 2, 3], [4, 5, 6]], caches)
        assert all(c.lengths == held and (c.codes is None) == (held == ()) for c in caches)
        for c in caches:
            c.append_rows(rows, rows, 2, 3, 2, 8)
            c.append_rows(rows, rows, 2, 2, 2, 8)


def test_blocks_do_not_share_a_cache(monkeypatch):
    """One cache for two blocks: each would append behind the other's positions."""
    monkeypatch.setattr(amd_lm, "QuantizedCache", stand_in)
    appended = []
    monkeypatch.setattr(decoder, "embed", lambda ids, weight, shape: None)
    model = object.__new__(decoder.Decoder)
    model.config, model.embedding = Config(max_seq_len=16, n_layers=2), SimpleNamespace(weight=None)
    model.blocks = [SimpleNamespace(decode=lambda hidden, cache, counts: appended.append(cache))] * 2
    cache = model.caches()[0]
    with pytest.raises(ValueError, match="of its own"):
        model.decode([[1, 2]], (cache, cache))
    assert not appended


def around_changes_of_plan():
    """Lengths before, at and behind each multiple of 2048 (where ranges of keys
    change) and every length around a power of two, in order."""
    lengths = set(range(300))
    for n in range(2048, 66000, 2048):
        lengths.update(range(n - 140, n + 3, 1 if n & (n - 1) == 0 else 20), (n - 1, n, n + 1))
    return sorted(lengths)


@built
@pytest.mark.parametrize("dtype", [0, 5])
@pytest.mark.parametrize("sequences,heads,kv_heads,dim", [(8, 16, 8, 64), (16, 32, 8, 128), (32, 32, 8, 128), (40, 32, 8, 128),
                                                          (64, 32, 8, 128), (128, 16, 4, 64), (128, 32, 8, 32), (1, 16, 4, 256)])
def test_a_growing_cache_never_keeps_too_small_a_workspace(sequences, heads, kv_heads, dim, dtype):
    """The size that the runtime keeps, while the longest sequence grows over
    every change of plan and shrinks again, against the library's own, which
    never falls where the length grows."""
    runtime = object.__new__(amd_runtime.Runtime)
    runtime._closed, runtime._attention_workspaces = True, {}
    runtime.lib = amd_runtime.load_library()
    size = runtime.lib.qutai_amd_attention_quantized_workspace_size
    lengths = around_changes_of_plan()
    for longest in (*lengths, *reversed(lengths)):
        for new in (1, 2):
            arguments = sequences, new, heads, kv_heads, dim, longest, dtype
            assert runtime.attention_workspace(*arguments) >= size(*arguments), arguments
    sizes = [size(sequences, 1, heads, kv_heads, dim, longest, dtype) for longest in lengths]
    assert sizes == sorted(sizes)


# ---- sampling ------------------------------------------------------------------------

@pytest.mark.parametrize("change", [
    dict(logits=fake(40, "float64")), dict(logits=fake(39, "float32")), dict(uniforms=fake(4, "bfloat16")),
    dict(uniforms=fake(5, "float32")), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 21), dict(temperature=-1.0),
    dict(temperature=float("inf")), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=1.5), dict(top_k=True),
    dict(top_p=1.1), dict(top_p=-0.1), dict(min_p=2), dict(min_p=float("nan")), dict(top_k=fake(4, "float32")),
    dict(temperature=fake(3, "float32")), dict(top_p=fake(4, "float64")), dict(min_p="0"),
])
def test_sample_refuses(change):
    a = dict(logits=fake(40, "float32"), uniforms=fake(4, "float32"), rows=4, vocab=10)
    with pytest.raises(ValueError):
        amd_lm.sample(**{**a, **change})


@built
def test_sample_entry_point_refuses():
    library, p = amd_runtime.load_library(), FAKE

    def call(logits=p, uniforms=p, tokens=p, probabilities=p, rows=4, vocab=10, temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, dtype=0, uniform_dtype=0):
        return library.qutai_amd_sample(logits, uniforms, tokens, probabilities, rows, vocab, None, temperature, None, top_k,
                                        None, top_p, None, min_p, dtype, uniform_dtype, None)

    for change in (dict(logits=None), dict(uniforms=None), dict(tokens=None), dict(probabilities=None), dict(rows=-1),
                   dict(rows=1 << 22), dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(temperature=-1.0),
                   dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_p=-1.0),
                   dict(top_p=float("nan")), dict(min_p=1.5), dict(min_p=float("nan")), dict(dtype=1), dict(uniform_dtype=5)):
        assert call(**change) == amd_runtime.QA_EINVAL, change
    assert call(rows=0, logits=None) == 0
