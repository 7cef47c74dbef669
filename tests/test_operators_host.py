"""Arguments that the decoder operators refuse, before any device call: the
Python checks, and the C entry points' own (stand-in pointers that are never
followed)."""
from itertools import count
from pathlib import Path

import pytest

from qutai_amd.backends import amd, amd_lm, amd_runtime
from qutai_amd.lm import Config

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
