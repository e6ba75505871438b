"""Corners of the frequency scalings, on the CPU."""
import math

import pytest

from llm_inference_optimization_b200 import rotary


@pytest.mark.parametrize("factor,want", [(0.25, 1.0), (0.9, 1.0), (1.0, 1.0), (4.0, 0.1 * math.log(4.0) + 1.0)])
def test_yarn_attention_factor_is_one_up_to_factors_of_one(factor, want):
    """The published rule: 1 for factors up to 1, 0.1 ln(factor) + 1 above; a factor that is given is taken as it is."""
    sc = {"type": "yarn", "factor": factor, "original_max_position": 4096}
    assert rotary.frequencies(64, 10000.0, sc)[1] == pytest.approx(want, rel=1e-15)
    assert rotary.frequencies(64, 10000.0, sc | {"attention_factor": 0.7})[1] == 0.7
