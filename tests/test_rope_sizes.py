"""CPU: what cos and sin are multiplied by where a context is stretched by parts
of its pairs' numbers: 0.1 ln(factor) + 1 from a factor of 1 on, and 1 for a
context that is not stretched (Peng et al., 2023)."""
import math

import pytest

from quantibbler_amd.gpu import Rope


@pytest.mark.parametrize("factor,size", [(4e-5, 1.0), (0.25, 1.0), (0.999, 1.0), (1.0, 1.0), (1.5, 0.1 * math.log(1.5) + 1),
                                         (16.0, 0.1 * math.log(16.0) + 1), (1e6, 0.1 * math.log(1e6) + 1)])
def test_the_size_is_of_stretched_contexts_alone(factor, size):
    rope = Rope(128, 10000.0, scaling={"kind": "yarn", "factor": factor, "original_len": 4096})
    assert rope._rope.size == size
    for kind in ("linear", "base", "ramp"):
        more = {"original_len": 4096} if kind == "ramp" else {}
        assert Rope(128, 10000.0, scaling={"kind": kind, "factor": factor, **more})._rope.size == 1.0
