"""Scaling options of rotary_frequencies that are missing or out of range."""
import pytest

from quartet_b200.rotary import rotary_frequencies


@pytest.mark.parametrize("scaling", [{"kind": "bands", "factor": 2.0}, {"kind": "yarn", "factor": 2.0}, {"kind": "bands", "factor": 2.0, "original_length": 0},
                                     {"kind": "yarn", "factor": 2.0, "original_length": -1}, {"kind": "yarn", "factor": 2.0, "original_length": 4096, "beta_fast": 0.0},
                                     {"kind": "yarn", "factor": 2.0, "original_length": 4096, "beta_slow": 40.0}, {"kind": "linear", "factor": float("nan")},
                                     {"kind": "linear", "factor": float("inf")}])
def test_scaling_is_refused_by_name(scaling):
    with pytest.raises(ValueError, match="original_length|beta|factor"):
        rotary_frequencies(64, scaling=scaling)


def test_a_base_of_one_turns_all_pairs_alike_and_has_no_ramp():
    assert bool((rotary_frequencies(64, 1.0)[0] == 1.0).all())
    with pytest.raises(ValueError, match="base"):
        rotary_frequencies(64, 1.0, {"kind": "yarn", "factor": 2.0, "original_length": 4096})
