"""The layers' contracts that need no GPU: YaRN's ramp at lengths where its upper end lies past
the last pair."""
from __future__ import annotations

import numpy as np
import pytest


@pytest.mark.parametrize("r, length, base, pairs, tail", [
    # rotary_dim, original length, base, the ramp's ends, the frequencies of the last pairs at factor 8
    (64, 131072.0, 1e4, (22, 35), [0.00012540918635710677, 8.207443430948874e-05, 5.257151799874643e-05]),
    (64, 4096.0, 100.0, (20, 46), [0.010735064724933957, 0.008847401809545132, 0.007272905768957644]),
    (4, 4096.0, 1e4, (0, 2), [1.0, 0.005625]),
])
def test_yarn_ramp_past_the_last_pair(pkg, r, length, base, pairs, tail):
    """The ramp's upper end is bounded by rotary_dim - 1, not by the last pair: slow pairs that still
    turn within the original length are divided in part only."""
    f, _ = pkg.rotary_frequencies(r, base=base, scaling="yarn", factor=8.0, original_length=length)
    np.testing.assert_allclose(f[-len(tail):], tail, rtol=1e-12)
    share = np.clip((np.arange(r // 2) - pairs[0]) / (pairs[1] - pairs[0]), 0, 1)
    np.testing.assert_allclose(f, base ** (-2 * np.arange(r // 2) / r) * (1 - share * 7 / 8), rtol=1e-12)
