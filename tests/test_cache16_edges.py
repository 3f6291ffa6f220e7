"""Rotary positions, the 16-bit cache and attention over shared prefixes at the edges of their arguments: what is refused and what it means.  No GPU needed, nothing is launched."""
import math

import numpy as np
import pytest

from calm_b200 import seqops


@pytest.mark.parametrize("factor,gain", [(4.0, 0.1 * math.log(4.0) + 1.0), (1.0, 1.0), (0.5, 1.0), (1e-6, 1.0)])
def test_the_ramps_gain(factor, gain):
    """Contexts that are stretched raise cosines and sines; contexts that are not leave them as they are."""
    scaling = {"kind": "ramp", "factor": factor, "length": 4096, "fast": 32.0, "slow": 1.0}
    assert math.isclose(seqops.rotation_frequencies(64, 1e4, scaling)[1], gain, rel_tol=1e-15)
    assert seqops.rotation_frequencies(64, 1e4, dict(scaling, gain=0.25))[1] == 0.25


RAMP = {"kind": "ramp", "factor": 2.0, "length": 64, "fast": 32.0, "slow": 1.0}


@pytest.mark.parametrize("base,scaling", [
    ("x", None), (None, None), (10 ** 400, None), (math.nan, None), (1e4, 5), (1e4, "none"), (1e4, {"kind": "linear", "factor": "4"}), (1e4, {"kind": ["linear"], "factor": 4.0}),
    (1e4, {"kind": "linear", "factor": 10 ** 400}), (1e4, {"kind": "linear", "factor": 1e-320}), (1e4, {"kind": "base", "factor": 1e300}), (5e-324, {"kind": "linear", "factor": 1e-200}),
    (1e4, {"kind": "linear", "factor": 2.0, "gain": math.inf}), (1e4, {"kind": "linear", "factor": 2.0, "gain": "q"}), (1e4, dict(RAMP, fast=1.0, slow=32.0)), (1e4, dict(RAMP, length=1e308, fast=1e-308)),
    (1e4, dict(RAMP, gain=math.nan))])
def test_rotations_that_no_number_holds_are_refused(base, scaling):
    with pytest.raises(ValueError):
        seqops.rotation_frequencies(8, base, scaling)
    with pytest.raises(ValueError, match="base|scaling|gain|factor|length|low|fast"):
        seqops.Rotation(8, base, scaling=scaling, device="cpu")


@pytest.mark.parametrize("frequencies", [[1j] * 4, "abcd", [None] * 4, [[1.0], [2.0, 3.0]], [10 ** 400] * 4])
def test_frequencies_that_are_no_numbers_are_refused(frequencies):
    with pytest.raises(ValueError, match="4 finite numbers"):
        seqops.Rotation(8, frequencies=frequencies, device="cpu")


def test_a_gain_past_float32_is_refused():
    with pytest.raises(ValueError, match="gain"):
        seqops.Rotation(8, scaling=dict(RAMP, gain=1e39), device="cpu")


def test_numbers_of_other_kinds_are_taken():
    want = seqops.rotation_frequencies(8, 1e4, RAMP)
    got = seqops.rotation_frequencies(8, np.float32(1e4), {k: v if k == "kind" else np.float64(v) for k, v in RAMP.items()})
    assert np.array_equal(got[0], want[0]) and got[1] == want[1] and np.array_equal(seqops.rotation_frequencies(8, 10000, {})[0], seqops.rotation_frequencies(8)[0])
