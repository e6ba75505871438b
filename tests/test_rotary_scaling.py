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


@pytest.mark.parametrize("theta,dim", [(10000.0, 64), (500000.0, 128), (1e6, 80)])
def test_fixed_point_frequencies_are_off_by_their_rounding(theta, dim):
    """Against 60 digits: 2^-51 of the frequency (four roundings of 2^-53: the power, 2 pi, its product, the quotient) and half a unit of
    the 64-bit fraction.  That, times the position, is what an angle is off by."""
    from decimal import Decimal, localcontext
    r = rotary.RotaryEmbedding(dim, theta, device="cpu")
    with localcontext() as c:
        c.prec = 60
        pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
        for i, t in enumerate(r.turns.tolist()):
            true = (Decimal(theta).ln() * Decimal(-2 * i) / Decimal(dim)).exp() / (2 * pi)
            off = abs(Decimal(t % (1 << 64)) / Decimal(2) ** 64 - true)
            assert off <= true * Decimal(2) ** -51 + Decimal(2) ** -65
