"""The network's layers without a GPU: refusals of their entry points, workspace sizes, the
rotary frequencies, struct layouts, and the 64-bit forms the GPU tests compare with."""
from __future__ import annotations

import ctypes as C
import math
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import layers_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def norm_cfg(pkg, **kw):
    c = pkg.GroupNormConfig(C.sizeof(pkg.GroupNormConfig), 0, 0, 0, 2, 100, 48, 4, 4800, 48, 4800, 48, 4800, 48, 1e-5)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def gated_cfg(pkg, **kw):
    c = pkg.GatedConfig(C.sizeof(pkg.GatedConfig), 2, 2, 64, 96, 10, 64, 64, 64, 96, 64, 64, 64)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def rotary_cfg(pkg, **kw):
    c = pkg.RotaryConfig(C.sizeof(pkg.RotaryConfig), 0, 0, 0, 1, 8, 64, 64, 0, 0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_structs_match_the_header(pkg, tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("needs gcc")
    names = {"stg_rotary_config": pkg.RotaryConfig, "stg_rotary_tensor": pkg.RotaryTensor,
             "stg_group_norm_config": pkg.GroupNormConfig, "stg_gated_config": pkg.GatedConfig,
             "stg_mask_head_config": pkg.MaskHeadConfig}
    src = "#include <stdio.h>\n#include \"stems_gpu_v1.h\"\nint main(void) {\n"
    for n, s in names.items():
        src += f'printf("{n} %zu", sizeof({n}));\n'
        for f, _ in s._fields_:
            src += f'printf(" %zu", offsetof({n}, {f}));\n'
        src += 'printf("\\n");\n'
    (tmp_path / "s.c").write_text(src + "return 0; }\n")
    subprocess.run(["gcc", f"-I{ROOT}/include", str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    for line in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.splitlines():
        n, size, *offs = line.split()
        assert int(size) == C.sizeof(names[n]), n
        assert [int(o) for o in offs] == [getattr(names[n], f).offset for f, _ in names[n]._fields_], n


def test_packed_configurations_are_the_structs(pkg):
    for packed, struct in ((pkg._ROTARY, pkg.RotaryConfig), (pkg._ROTARY_TENSOR, pkg.RotaryTensor), (pkg._GROUP_NORM, pkg.GroupNormConfig),
                           (pkg._GATED, pkg.GatedConfig)):
        values = list(range(1, len(struct._fields_) + 1))
        assert packed.pack(*values) == bytes(struct(*values))


def test_null_engines_and_plans_are_rejected(pkg):
    L, n = pkg.lib(), C.c_size_t()
    assert L.stg_rotary(None, C.byref(rotary_cfg(pkg)), None, 1, None, 0, None) == 1
    assert L.stg_group_norm(None, C.byref(norm_cfg(pkg)), *[None] * 7, 0, None) == 1
    assert L.stg_group_norm_backward(None, C.byref(norm_cfg(pkg)), *[None] * 10, 0, None) == 1
    assert L.stg_gated(None, C.byref(gated_cfg(pkg)), *[None] * 7, 0, None) == 1
    assert L.stg_gated_backward(None, C.byref(gated_cfg(pkg)), *[None] * 12, 0, None) == 1
    head = pkg.MaskHeadConfig(C.sizeof(pkg.MaskHeadConfig), 2, 64, 1)
    assert L.stg_mask_head(None, C.byref(head), *[None] * 5, 0, None) == 1
    assert L.stg_mask_head_workspace(None, C.byref(head), C.byref(n)) == 1
    assert L.stg_mask_head_sizes(None, None, None, None, None) == 1
    assert L.stg_engine_status(None) == 1


@pytest.mark.parametrize("bad, code", [
    (dict(size=8), 1), (dict(dtype=3), 1), (dict(dtype=-1), 1), (dict(param_dtype=1), 1), (dict(activation=5), 1),
    (dict(activation=-1), 1), (dict(batch=-1), 1), (dict(positions=-1), 1), (dict(groups=0), 1), (dict(groups=5), 1),
    (dict(channels=0), 1), (dict(eps=-1e-6), 1), (dict(eps=math.nan), 1), (dict(x_batch=-1), 1), (dict(y_position=-48), 1),
    (dict(dx_batch=-1), 1), (dict(channels=8196), 2), (dict(batch=65536), 2), (dict(positions=1 << 36), 2)])
def test_group_norm_refusals(pkg, bad, code):
    n = C.c_size_t()
    for backward in (0, 1):
        assert pkg.lib().stg_group_norm_workspace(C.byref(norm_cfg(pkg)), backward, C.byref(n)) == 0
        assert pkg.lib().stg_group_norm_workspace(C.byref(norm_cfg(pkg, **bad)), backward, C.byref(n)) == code
    assert pkg.lib().stg_group_norm_workspace(None, 0, C.byref(n)) == 1
    assert pkg.lib().stg_group_norm_workspace(C.byref(norm_cfg(pkg)), 0, None) == 1
    assert pkg.lib().stg_group_norm_workspace(C.byref(norm_cfg(pkg)), 2, C.byref(n)) == 1


@pytest.mark.parametrize("bad, code", [
    (dict(size=4), 1), (dict(dtype=7), 1), (dict(activation=9), 1), (dict(features=0), 1), (dict(width=0), 1),
    (dict(rows=-1), 1), (dict(x_row=-1), 1), (dict(rows=1 << 31), 2)])
def test_gated_refusals(pkg, bad, code):
    n = C.c_size_t()
    for backward in (0, 1):
        assert pkg.lib().stg_gated_workspace(C.byref(gated_cfg(pkg)), backward, C.byref(n)) == 0
        assert pkg.lib().stg_gated_workspace(C.byref(gated_cfg(pkg, **bad)), backward, C.byref(n)) == code
    assert pkg.lib().stg_gated_workspace(C.byref(gated_cfg(pkg, y_row=95)), 0, C.byref(n)) == 1   # rows of y overlap
    assert pkg.lib().stg_gated_workspace(C.byref(gated_cfg(pkg, y_row=0)), 1, C.byref(n)) == 0    # a broadcast dy is fine
    assert pkg.lib().stg_gated_workspace(C.byref(gated_cfg(pkg, rows=0)), 1, C.byref(n)) == 0 and n.value == 0


@pytest.mark.parametrize("bad, code", [
    (dict(size=16), 1), (dict(dtype=4), 1), (dict(layout=2), 1), (dict(inverse=2), 1), (dict(batch=-1), 1), (dict(tokens=-1), 1),
    (dict(head_dim=0), 1), (dict(head_dim=65537), 1), (dict(rotary_dim=63), 1), (dict(rotary_dim=66), 1), (dict(rotary_dim=-2), 1),
    (dict(head_dim=63, rotary_dim=0), 1), (dict(head_dim=514, rotary_dim=514), 2), (dict(scaling=4), 1), (dict(base=-1.0), 1),
    (dict(base=1.0), 1), (dict(base=math.inf), 1), (dict(magnitude=math.nan), 1), (dict(scaling=1, factor=0.5), 1),
    (dict(scaling=1, factor=math.nan), 1), (dict(scaling=2, factor=2.0, rotary_dim=2), 1), (dict(scaling=3, factor=2.0), 1),
    (dict(scaling=3, factor=2.0, original_length=4096.0, beta_fast=1.0, beta_slow=2.0), 1),
    (dict(scaling=3, factor=2.0, original_length=4096.0, beta_fast=1.0), 1), (dict(batch=1 << 40, tokens=1 << 40), 2)])
def test_rotary_refusals(pkg, bad, code):
    f, m = (C.c_double * 512)(), C.c_double()
    assert pkg.lib().stg_rotary_frequencies(C.byref(rotary_cfg(pkg)), f, C.byref(m)) == 0
    assert pkg.lib().stg_rotary_frequencies(C.byref(rotary_cfg(pkg, **bad)), f, C.byref(m)) == code
    assert pkg.lib().stg_rotary_frequencies(C.byref(rotary_cfg(pkg)), None, C.byref(m)) == 1
    assert pkg.lib().stg_rotary_frequencies(None, f, C.byref(m)) == 1


def test_python_refusals_need_no_device_call(pkg):
    e = pkg.Engine.__new__(pkg.Engine)
    e._h, e.device = C.c_void_p(), 0
    x = torch.zeros(2, 4, 8)
    for call in (lambda: e.group_norm(x, 2), lambda: e.gated(x, torch.zeros(4, 8), torch.zeros(4, 8)), lambda: e.group_norm("x", 2),
                 lambda: e.rotary(torch.zeros(1, 2, 3, 8)), lambda: e.gated(x.to(torch.int32), None, None)):
        with pytest.raises(pkg.StemsError) as err:
            call()
        assert err.value.code == 1
    with pytest.raises(pkg.StemsError):
        pkg.rotary_frequencies(8, scaling="other")
    with pytest.raises(pkg.StemsError):
        pkg.rotary_frequencies(7)


def test_runs_of_rows(pkg):
    t = torch.zeros(5, 7, 6, 8)
    assert pkg._run(t.shape[:-1], t.stride()[:-1], 8) == (210, 8)
    s = t[:, :1]
    assert pkg._run(s.shape[:-1], s.stride()[:-1], 8)[1] is None
    s = t[:, :1, :1]
    assert pkg._run(s.shape[:-1], s.stride()[:-1], 8) == (5, 7 * 6 * 8)
    s = t[:, :, ::2]
    assert pkg._run(s.shape[:-1], s.stride()[:-1], 8) == (105, 16)
    assert pkg._run((1, 1), (3, 9), 8) == (1, 8)
    assert pkg._run((4, 0, 3), (0, 3, 1), 8)[0] == 0


@pytest.mark.parametrize("r", [2, 4, 32, 64, 80, 512])
def test_rotary_frequencies(pkg, r):
    i = np.arange(r // 2)
    f, m = pkg.rotary_frequencies(r)
    np.testing.assert_allclose(f, 10000.0 ** (-2 * i / r), rtol=1e-14)
    assert m == 1.0
    f, m = pkg.rotary_frequencies(r, base=500000.0, scaling="linear", factor=4.0, magnitude=0.5)
    np.testing.assert_allclose(f, 500000.0 ** (-2 * i / r) / 4, rtol=1e-14)
    assert m == 0.5
    if r > 2:
        f, m = pkg.rotary_frequencies(r, scaling="ntk", factor=8.0)
        np.testing.assert_allclose(f, (10000.0 * 8.0 ** (r / (r - 2))) ** (-2 * i / r), rtol=1e-13)
        assert f[0] == 1.0 and math.isclose(f[-1], 10000.0 ** (-2 * i[-1] / r) / 8, rel_tol=1e-12)   # the slowest by s exactly
    f, m = pkg.rotary_frequencies(r, scaling="yarn", factor=8.0, original_length=4096)
    plain = 10000.0 ** (-2 * i / r)
    turns = 4096 * plain / (2 * math.pi)     # a pair's turns within the original length
    assert math.isclose(m, 0.1 * math.log(8.0) + 1)
    assert np.all(f <= plain * (1 + 1e-14)) and np.all(f >= plain / 8 * (1 - 1e-14))
    # pairs that turn more than 32 times keep their frequency, those below once are divided
    # (the ramp's ends are whole pairs, so one pair either way may differ)
    np.testing.assert_allclose(f[:max(0, int((turns > 32).sum()) - 1)], plain[:max(0, int((turns > 32).sum()) - 1)], rtol=1e-14)
    below = int((turns < 1).sum()) - 1
    if below > 0:
        np.testing.assert_allclose(f[-below:], plain[-below:] / 8, rtol=1e-14)
    same, _ = pkg.rotary_frequencies(r, scaling="yarn", factor=1.0, original_length=4096)
    np.testing.assert_allclose(same, plain, rtol=1e-14)


@pytest.mark.parametrize("kind", ["none", "silu", "gelu", "sigmoid", "relu"])
def test_the_references_gradients_are_the_formulas(kind):
    """autograd of the 64-bit forward forms, and central differences, against the backward forms."""
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, ga, be, dy = r(2, 5, 6).requires_grad_(), r(6).requires_grad_(), r(6).requires_grad_(), r(2, 5, 6)

    def norm(x, ga, be):
        h = x.reshape(2, 5, 3, 2)
        mean, var = h.mean((1, 3), keepdim=True), h.var((1, 3), correction=0, keepdim=True)
        return ref.act(kind, ((h - mean) / torch.sqrt(var + 1e-5)).reshape(2, 5, 6) * ga + be), mean, var

    y, mean, var = norm(x, ga, be)
    want = torch.autograd.grad((y * dy).sum(), (x, ga, be))
    xs = x.detach()
    stats = mean.flatten(1).detach(), (1 / torch.sqrt(var + 1e-5)).flatten(1).detach()
    old, ref.FAST = ref.FAST, {torch.float64: 0.0}
    try:
        got, _ = ref.group_norm_backward(dy, xs, 3, ga.detach(), be.detach(), *stats, kind)
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b, rtol=1e-10, atol=1e-10)
        step, v = 1e-6, r(2, 5, 6)
        diff = ((norm(xs + step * v, ga, be)[0] - norm(xs - step * v, ga, be)[0]) * dy).sum() / (2 * step)
        assert math.isclose(float(diff.detach()), float((got[0] * v).sum()), rel_tol=1e-6, abs_tol=1e-7)
        x, wg, wu, bg, bu, dy = (t.requires_grad_() for t in (r(7, 4), r(5, 4), r(5, 4), r(5), r(5), r(7, 5)))
        y = ref.act(kind, x @ wg.t() + bg) * (x @ wu.t() + bu)
        want = torch.autograd.grad((y * dy).sum(), (x, wg, wu, bg, bu))
        got, _ = ref.gated_backward(*(t.detach() for t in (dy, x, wg, wu, bg, bu)), kind)
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b, rtol=1e-10, atol=1e-10)
    finally:
        ref.FAST = old


def test_the_rotary_reference_is_a_rotation():
    x = torch.randn(2, 3, 4, 8, dtype=torch.float64)
    pos = torch.tensor([0, 5, 1000])
    f = 10000.0 ** (-torch.arange(3, dtype=torch.float64) / 3)
    for layout in ("interleaved", "half"):
        y, _ = ref.rotary(x, pos, f, 1.0, 6, layout)
        torch.testing.assert_close(y.norm(dim=-1), x.norm(dim=-1))
        torch.testing.assert_close(y[:, 0], x[:, 0])
        back, _ = ref.rotary(y, pos, f, 1.0, 6, layout, inverse=True)
        torch.testing.assert_close(back, x)
        z = torch.view_as_complex(torch.stack((x[0, 1, 2, 2], x[0, 1, 2, 3] if layout == "interleaved" else x[0, 1, 2, 5])))
        w = z * torch.polar(torch.ones((), dtype=torch.float64), 5 * f[1 if layout == "interleaved" else 2])
        got = (y[0, 1, 2, 2], y[0, 1, 2, 3 if layout == "interleaved" else 5])
        torch.testing.assert_close(torch.stack(got), torch.view_as_real(w))
