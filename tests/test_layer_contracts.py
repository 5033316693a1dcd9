"""The layers' contracts that need no GPU: YaRN's ramp at lengths where its upper end lies past
the last pair, sizes that the gated projection's kernels cannot reach, tensors that require gradients."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch


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


@pytest.mark.parametrize("sizes, code", [
    (dict(features=2 ** 31 - 2 ** 16), 0), (dict(features=2 ** 31 - 2 ** 16 + 1), 2), (dict(features=2 ** 31 - 1), 2),
    (dict(width=2 ** 31 - 2 ** 16), 0), (dict(width=2 ** 31 - 1), 2), (dict(rows=2 ** 31 - 1, features=8, width=8), 0),
    # a broadcast dy, x or weight makes these calls possible; their scratch would not fit 64 bits
    (dict(rows=2 ** 31 - 1, width=2 ** 30), 2), (dict(rows=2 ** 31 - 1, features=2 ** 30), 2), (dict(width=2 ** 30, features=2 ** 30), 2),
    (dict(rows=2 ** 24, width=2 ** 26, features=2 ** 24), 0)])
def test_gated_sizes_past_the_kernels_reach_are_refused(pkg, sizes, code):
    """Positions along the features and the outputs are 32 bits wide in the kernels and run up to a
    tile past the end; the scratch's bytes are 64 bits wide."""
    for dtype in (0, 1, 2):
        c = dict(dict(rows=10, features=64, width=96), **sizes)
        k, n = c["features"], c["width"]
        cfg = pkg.GatedConfig(C.sizeof(pkg.GatedConfig), dtype, 2, k, n, c["rows"], 0, 0, 0, 0, k, k, k)
        need = C.c_size_t(12345)
        assert pkg.lib().stg_gated_workspace(C.byref(cfg), 1, C.byref(need)) == code
        # dg and du alone are rows x width each
        assert need.value >= 2 * c["rows"] * n * (2 if dtype else 4) if code == 0 else need.value == 12345


def test_tensors_that_require_gradients_are_refused_while_they_are_recorded(pkg):
    """The layers record no graph; without the refusal their results would be cut off from it silently."""
    e = pkg.Engine.__new__(pkg.Engine)
    e._h, e.device, e._raw_stream, e._scratch = C.c_void_p(), -1, lambda device: 0, {}      # of CPU tensors' device
    e.last_error = lambda: "no engine"
    x, w, v = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8)
    stats = torch.zeros(4, 2)
    xg = x.clone().requires_grad_()
    for call, args in ((e.gated, (x, w, w, v, v)), (e.gated_backward, (x, x, w, w, v, v)), (e.group_norm, (x, 2, v, v)),
                       (e.group_norm_backward, (x, x, 2, v, v, stats, stats)), (e.rotary, (x.view(1, 2, 2, 8), x.view(1, 2, 2, 8)))):
        for i, a in enumerate(args):
            if a is stats or not torch.is_tensor(a):
                continue
            some = [b if j != i else b.clone().requires_grad_() for j, b in enumerate(args)]
            with pytest.raises(pkg.StemsError, match="requires a gradient"):
                call(*some)
            with torch.no_grad(), pytest.raises(pkg.StemsError, match="no engine"):   # this one reached the library
                call(*some)
    with pytest.raises(pkg.StemsError, match="requires a gradient"):
        e.group_norm(x, 2, out=xg * 1)
