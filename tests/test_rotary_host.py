"""What a Rotary and a Config refuse: numbers that overflow and descriptions that are none
are ValueErrors, whatever their type."""
import pytest

from qutai_amd.lm import Config, Rotary

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
