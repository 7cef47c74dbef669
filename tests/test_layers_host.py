"""Options of the lm layer functions that exclude each other, refused before any device
call."""
import pytest

from qutai_amd import Tensor
from qutai_amd.lm import Rotary, qk_norm_rope
from qutai_amd.lm.layers import rotary
from tests.test_operators_host import fake


@pytest.mark.parametrize("function", ["qk_norm_rope", "rotary"])
def test_positions_take_the_place_of_an_offset(function):
    """One position for every token says where it is; an offset beside it says otherwise."""
    q, k, *weights = (Tensor(fake(n, "float32"), shape=shape)
                      for n, shape in ((192, (2, 3, 32)), (96, (2, 3, 16)), (8, (8,)), (8, (8,))))
    where = dict(offset=5, positions=fake(6, "int64"))
    with pytest.raises(ValueError, match="positions"):
        if function == "rotary":
            rotary(q, k, 4, 2, Rotary(8), **where)
        else:
            qk_norm_rope(q, k, *weights, 4, 2, 1e4, 1e-6, **where)
