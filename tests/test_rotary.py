"""Rotary frequencies and argument checks, on the CPU."""
import math

import pytest
import torch

import llm_inference_optimization_b200 as skv
from llm_inference_optimization_b200 import _lib, rotary


def test_plain_linear_and_ntk_frequencies():
    f, a = rotary.frequencies(64, 10000.0)
    assert a == 1.0 and len(f) == 32 and f[0] == 1.0 and f[31] == pytest.approx(10000.0 ** (-62 / 64), rel=1e-15)
    g, _ = rotary.frequencies(64, 10000.0, {"type": "linear", "factor": 4.0})
    assert all(y == x / 4 for x, y in zip(f, g))
    h, _ = rotary.frequencies(64, 10000.0, {"type": "ntk", "factor": 4.0})
    assert h[0] == 1.0 and h[31] == pytest.approx(f[31] / 4, rel=1e-12)      # the slowest pair slows by the factor


def test_llama3_keeps_fast_pairs_and_divides_slow_ones():
    sc = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position": 8192}
    f, _ = rotary.frequencies(128, 500000.0)
    g, a = rotary.frequencies(128, 500000.0, sc)
    assert a == 1.0
    for x, y in zip(f, g):
        wave = 2 * math.pi / x
        if wave < 8192 / 4:
            assert y == x
        elif wave > 8192:
            assert y == pytest.approx(x / 8, rel=1e-15)
        else:
            s = (8192 / wave - 1) / 3
            assert y == pytest.approx((1 - s) * x / 8 + s * x, rel=1e-13)


def test_yarn_ramp_and_attention_factor():
    f, _ = rotary.frequencies(64, 10000.0)
    g, a = rotary.frequencies(64, 10000.0, {"type": "yarn", "factor": 16.0, "original_max_position": 4096})
    assert a == pytest.approx(0.1 * math.log(16) + 1)
    assert g[0] == f[0] and g[31] == pytest.approx(f[31] / 16, rel=1e-15)
    assert all(x / 16 <= y * (1 + 1e-12) and y <= x * (1 + 1e-12) for x, y in zip(f, g))
    _, b = rotary.frequencies(64, 10000.0, {"type": "yarn", "factor": 16.0, "original_max_position": 4096, "attention_factor": 1.0})
    assert b == 1.0


def test_turns_are_the_frequencies_in_fixed_point():
    r = rotary.RotaryEmbedding(128, 500000.0, device="cpu")
    f, _ = rotary.frequencies(128, 500000.0)
    for t, x in zip(r.turns.tolist(), f):
        assert (t % (1 << 64)) / 2.0 ** 64 == pytest.approx(x / (2 * math.pi), rel=1e-15)


@pytest.mark.parametrize("bad", [dict(head_dim=64, rotary_dim=63), dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=0),
                                 dict(head_dim=64, layout="both"), dict(head_dim=64, theta=1.0), dict(head_dim=64, theta=math.inf),
                                 dict(head_dim=64, scaling={"type": "dynamic", "factor": 2.0}),
                                 dict(head_dim=64, scaling={"type": "linear"}),
                                 dict(head_dim=64, scaling={"type": "linear", "factor": 0.0}),
                                 dict(head_dim=64, scaling={"type": "linear", "factor": 2.0, "extra": 1.0}),
                                 dict(head_dim=64, scaling={"type": "llama3", "factor": 8.0, "low_freq_factor": 4.0,
                                                            "high_freq_factor": 4.0, "original_max_position": 8192})])
def test_bad_rotations_are_refused(bad):
    with pytest.raises(RuntimeError):
        rotary.RotaryEmbedding(device="cpu", **bad)


def test_cpu_tensors_are_refused(lib):
    r = rotary.RotaryEmbedding(64, device="cpu")
    with pytest.raises(RuntimeError):
        r.apply(torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, 64))


def test_entry_point_argument_errors(lib):
    """Refusals that come before anything touches a device."""
    z = (0,) * 8
    assert lib.skv_rotary(None, None, None, None, 0, None, 0, None, 4, 2, 0, 64, 64, 0, 1.0, 0, *z, 0, None) == -1
    assert "null" in _lib.last_error()
    assert lib.skv_rotary(16, None, 16, None, 0, 16, 0, 16, 4, 2, 0, 64, 63, 0, 1.0, 0, *z, 0, None) == -1
    assert lib.skv_rotary(16, None, 16, None, 7, 16, 0, 16, 4, 2, 0, 64, 64, 0, 1.0, 0, *z, 0, None) == -2
    assert lib.skv_rotary(16, None, 16, None, 0, 16, 0, 16, -1, 2, 0, 64, 64, 0, 1.0, 0, *z, 0, None) == -1
    assert lib.skv_rotary(None, None, None, None, 0, None, 0, None, 0, 2, 0, 64, 64, 0, 1.0, 0, *z, 0, None) == 0    # no rows
    assert hasattr(skv, "rotary")


@pytest.mark.parametrize("q, k", [((0, 64), None), ((128, 0), None), ((32, 256), None), ((64, 64), None), ((128, 64), (0, 64)),
                                  ((128, 64), (128, 32)), ((128, 64), "same")])
def test_outputs_that_overlap_are_refused(lib, q, k):
    """Expanded or shortened strides, or one destination for both, of four tokens and two heads: before any launch."""
    kp, Hk, ks = (None, 0, (0, 0)) if k is None else (4096, 2, (128, 64)) if k == "same" else (1 << 20, 2, k)
    assert lib.skv_rotary(4096, kp, 4096, kp, 0, 16, 0, 16, 4, 2, Hk, 64, 64, 0, 1.0, 0, *q, *ks, *q, *ks, 0, None) == -1
    assert "overlap" in _lib.last_error()
