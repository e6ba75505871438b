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


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": None}, {"type": "ntk", "factor": "four"}, {"type": "linear", "factor": [4.0]},
                                     {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": None, "original_max_position": 8192},
                                     {"type": "yarn", "factor": 4.0, "original_max_position": None},
                                     {"type": "yarn", "factor": 4.0, "original_max_position": 4096, "beta_fast": "fast"}])
def test_values_that_are_no_numbers_are_refused(scaling):
    with pytest.raises(RuntimeError, match="numbers"):
        rotary.frequencies(64, 10000.0, scaling)


def test_optional_values_may_be_none():
    sc = {"type": "yarn", "factor": 4.0, "original_max_position": 4096}
    assert rotary.frequencies(64, 10000.0, sc | {"beta_fast": None, "attention_factor": None}) == rotary.frequencies(64, 10000.0, sc)
