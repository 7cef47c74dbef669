"""What a Rotary and a Config refuse: numbers that overflow and descriptions that are none
are ValueErrors, whatever their type."""
from types import SimpleNamespace

import pytest

from qutai_amd.backends import amd_lm
from qutai_amd.lm import Config, Rotary
from tests.test_operators_host import fake

HUGE = 10 ** 400  # an integer that no float holds


@pytest.mark.parametrize("change", [
    dict(scaling={"kind": "base", "factor": 1e200}, rotary_dim=4),  # the factor's square
    dict(scaling={"kind": "base", "factor": HUGE}), dict(scaling={"kind": "linear", "factor": HUGE}),
    dict(scaling={"kind": "linear", "factor": 5e-324}), dict(theta=HUGE), dict(theta=1e300, scaling={"kind": "base", "factor": 1e300}),
    dict(theta=1e300, scaling={"kind": "base", "factor": 1e100}), dict(theta=5e-324, scaling={"kind": "linear", "factor": 1e-300}), dict(scaling={"kind": ["linear"], "factor": 2}),
    dict(scaling={"kind": {}, "factor": 2}), dict(layout=["half"]), dict(theta="1"), dict(theta=None), dict(theta=True),
    dict(scaling={"kind": "parts", "factor": 2, "original_length": HUGE}),
    dict(scaling={"kind": "parts", "factor": 2, "original_length": 8, "low": -HUGE}),
    dict(scaling={"kind": "parts", "factor": 2, "original_length": 8, "low": -0.5}),
    dict(scaling={"kind": "parts", "factor": 2, "original_length": 8, "magnitude": 1e31}),
    dict(scaling={"kind": "parts", "factor": 2, "original_length": 8, "magnitude": 1e-60})])
def test_rotary_refuses_with_a_value_error(change):
    with pytest.raises(ValueError):
        Rotary(**{"dim": 64, **change})


@pytest.mark.parametrize("change", [dict(rope_scaling={"kind": "base", "factor": 1e200}, rope_dim=4),
                                    dict(rope_scaling={"kind": ["linear"], "factor": 2}), dict(rope_layout=["half"])])
def test_config_refuses_with_a_value_error(change):
    with pytest.raises(ValueError):
        Config(**change)


@pytest.mark.parametrize("offset", [1 << 63, -(1 << 63) - 1, 1 << 200, 0.5, float("inf"), float("nan"), "1", None])
def test_an_offset_that_no_int64_holds_is_refused(offset):
    """It would arrive at the kernel as another position."""
    q, k = fake(6 * 4 * 8, "bfloat16"), fake(6 * 2 * 8, "bfloat16")
    with pytest.raises(ValueError):
        amd_lm.rotary(q, k, Rotary(8), 2, 3, 4, 2, 8, offset=offset)


def test_a_whole_number_of_any_type_is_an_offset(monkeypatch):
    sent = []
    monkeypatch.setattr(amd_lm, "get_runtime", lambda: SimpleNamespace(call=lambda name, *arguments: sent.append(arguments[7])))
    block = fake(6 * 48, "bfloat16")
    for offset in (7, 7.0, True + 6):
        amd_lm.rotary(block, block, Rotary(8), 2, 3, 4, 2, 8, offset=offset, q_row=48, k_column=32, k_row=48, out=block, out_row=48)
    assert sent == [7] * 3 and all(type(x) is int for x in sent)
