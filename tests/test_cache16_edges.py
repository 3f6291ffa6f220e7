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
