"""The network's layers on the GPU against their 64-bit forms (layers_ref.py), within bounds that
count the roundings of each output's own terms: worst() is |got - want| over the bound, so 1 is
the limit everywhere."""
from __future__ import annotations

import math

import pytest
import torch

import layers_ref as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
KINDS = ["none", "relu", "silu", "gelu", "sigmoid"]


def rnd(seed, *shape, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def ok(got, want_bound):
    assert ref.worst(got, *want_bound) <= 1.0


# ---- rotary ---------------------------------------------------------------------------------
ROTARY = [
    # batch, tokens, heads, kv heads, head_dim, rotary_dim
    (1, 1, 1, 1, 2, 2), (1, 1, 1, 1, 1, 0), (2, 7, 3, 1, 64, 64), (3, 65, 8, 8, 64, 32), (1, 130, 5, 2, 58, 58), (2, 9, 2, 2, 33, 20),
    (1, 1, 32, 8, 128, 128), (4, 1, 16, 4, 80, 32), (1, 2, 700, 3, 6, 4), (1, 3, 1, 1, 600, 512), (60, 33, 8, 8, 48, 48), (1, 1025, 2, 1, 10, 2),
]


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ROTARY)
def test_rotary(pkg, engine, shape, dtype, layout):
    b, t, h, hk, d, r = shape
    if r == 0:
        with pytest.raises(pkg.StemsError):
            engine.rotary(rnd(1, b, t, h, d, dtype=dtype))
        return
    f, m = pkg.rotary_frequencies(r)
    q, k = rnd(1, b, t, h, d, dtype=dtype), rnd(2, b, t, hk, d, dtype=dtype)
    pos = torch.arange(17, 17 + t, device="cuda", dtype=torch.int32)
    y, z = engine.rotary(q, k, offset=17, rotary_dim=r, layout=layout)
    ok(y, ref.rotary(q, pos, f, m, r, layout))
    ok(z, ref.rotary(k, pos, f, m, r, layout))
    assert torch.equal(y[..., r:], q[..., r:])
    rows = torch.randint(-1000, 1000, (b, t), device="cuda", dtype=torch.int32)   # negative positions turn back
    ok(engine.rotary(q, positions=rows, rotary_dim=r, layout=layout, inverse=True), ref.rotary(q, rows, f, m, r, layout, True))


@pytest.mark.parametrize("scaling", [dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
                                     dict(scaling="yarn", factor=16.0, original_length=4096.0),
                                     dict(scaling="yarn", factor=2.0, original_length=100.0, beta_fast=8.0, beta_slow=0.5, magnitude=0.7)])
def test_rotary_scaled_and_far(pkg, engine, scaling):
    q = rnd(3, 1, 37, 3, 64)
    f, m = pkg.rotary_frequencies(64, **scaling)
    for offset in (0, 1000003, 2 ** 31 - 37, -2 ** 31):
        pos = torch.arange(offset, offset + 37, device="cuda", dtype=torch.int64)
        ok(engine.rotary(q, offset=offset, **scaling), ref.rotary(q, pos, f, m, 64, "interleaved"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary_strides_and_in_place(pkg, engine, dtype, layout):
    f, m = pkg.rotary_frequencies(32)
    qkv = rnd(4, 2, 19, 3, 5, 40, dtype=dtype)            # [b][t][q, k, v][h][d]
    before = qkv.clone()
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    pos = torch.arange(19, device="cuda", dtype=torch.int32)
    want = [ref.rotary(x, pos, f, m, 32, layout) for x in (q, k)]
    for got, w in zip(engine.rotary(q, k, rotary_dim=32, layout=layout), want):
        ok(got, w)
    engine.rotary(q, k, rotary_dim=32, layout=layout, out=q, out_k=k)
    ok(q, want[0]), ok(k, want[1])
    assert torch.equal(qkv[:, :, 2], before[:, :, 2])
    # heads before tokens, and addresses that are not whole vectors
    x = rnd(5, 2, 5, 19, 41, dtype=dtype)[..., 1:].transpose(1, 2)
    ok(engine.rotary(x, rotary_dim=32, layout=layout), ref.rotary(x, pos, f, m, 32, layout))
    shared = rnd(6, 1, 19, 5, 40, dtype=dtype).expand(3, -1, -1, -1)   # one input for the whole batch
    ok(engine.rotary(shared, rotary_dim=32, layout=layout), ref.rotary(shared, pos, f, m, 32, layout))


def test_rotary_long_and_narrow(pkg, engine):
    """Many tokens of one narrow head: the largest blocks of tokens."""
    x = rnd(11, 1, 1300001, 1, 2)
    f, m = pkg.rotary_frequencies(2)
    ok(engine.rotary(x), ref.rotary(x, torch.arange(1300001, device="cuda"), f, m, 2, "interleaved"))


def test_rotary_empty_special_and_gradient(pkg, engine):
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        assert engine.rotary(torch.empty(shape, device="cuda")).shape == shape
    x = rnd(7, 1, 2, 1, 8)
    x[0, 1, 0, 2], x[0, 0, 0, 7] = math.inf, math.nan
    y = engine.rotary(x, layout="half")
    assert torch.isnan(y[0, 0, 0, [3, 7]]).all() and torch.isfinite(y[0, 0, 0, :3]).all()
    assert not torch.isfinite(y[0, 1, 0, [2, 6]]).any() and torch.isfinite(y[0, 1, 0, [0, 1, 3, 4, 5, 7]]).all()
    # the gradient by differences: the map is linear, so <R v, w> = <v, R^T w>
    v, w = rnd(8, 2, 50, 3, 64), rnd(9, 2, 50, 3, 64)
    kw = dict(scaling="yarn", factor=4.0, original_length=32.0, rotary_dim=48)
    a = (engine.rotary(v, **kw).double() * w.double()).sum()
    b = (v.double() * engine.rotary(w, inverse=True, **kw).double()).sum()
    assert abs(float(a - b)) <= 16 * ref.F32 * 2 * float((v.double().abs() * w.double().abs()).sum() + 9600)


def test_rotary_refusals(pkg, engine):
    x = torch.zeros(1, 4, 2, 8, device="cuda")
    for kw in (dict(rotary_dim=7), dict(rotary_dim=10), dict(layout="x"), dict(scaling="ntk", factor=0.0), dict(offset=2 ** 31 - 3),
               dict(positions=torch.zeros(4, device="cuda")), dict(positions=torch.zeros(5, dtype=torch.int32, device="cuda")),
               dict(positions=torch.zeros(4, dtype=torch.int32)), dict(k=torch.zeros(1, 5, 2, 8, device="cuda")),
               dict(k=x.half()), dict(out=torch.zeros(1, 4, 2, 9, device="cuda")), dict(out=torch.zeros(1, 4, 1, 8, device="cuda").expand(-1, -1, 2, -1))):
        with pytest.raises(pkg.StemsError) as err:
            engine.rotary(x, **kw)
        assert err.value.code in (1, 2)
    with pytest.raises(pkg.StemsError):
        engine.rotary(x.transpose(2, 3))
    engine.rotary(x)      # and it still works


# ---- group norm ------------------------------------------------------------------------------
NORM = [
    # batch, positions, channels, groups
    (1, 1, 1, 1), (1, 1, 8, 1), (2, 1, 6, 3), (1, 2, 8, 8), (3, 17, 48, 4), (2, 336, 48, 1), (1, 1000, 75, 5), (2, 129, 96, 96),
    (1, 5000, 64, 2), (4, 3, 2056, 8), (1, 40, 2051, 7), (2, 3, 8192, 1), (1, 50, 8192, 8192), (5, 700, 24, 3), (1, 30011, 16, 4), (2, 9000, 192, 4),
    (65, 9, 32, 8), (1, 33, 36, 1), (7, 9, 16, 2),
    (5, 30000, 24, 2), (1, 400000, 40, 5), (3, 70001, 33, 3), (2, 20000, 520, 520),
    (3, 100, 1000, 1000), (2, 50, 384, 128), (1, 257, 1030, 103), (2, 16, 4096, 4096), (2, 20, 4104, 1026),      # more groups than warps
    (700, 5, 24, 3), (600, 16, 16, 1), (1200, 3, 75, 25), (300, 7, 96, 96), (20, 12, 4104, 8),     # many small items
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORM)
def test_group_norm_and_backward(engine, shape, dtype):
    b, n, c, g = shape
    kind = KINDS[(n + c) % 5]
    pt = dtype if n % 2 else F32
    x, ga, be = rnd(1, b, n, c, dtype=dtype, scale=2.0, shift=0.5), rnd(2, c, dtype=pt, shift=1.0), rnd(3, c, dtype=pt)
    y, mean, rstd = engine.group_norm(x, g, ga, be, activation=kind, return_stats=True)
    want, bound, m64, r64 = ref.group_norm(x, g, ga, be, 1e-5, kind)
    ok(y, (want, bound))
    assert torch.equal(engine.group_norm(x, g, ga, be, activation=kind), y)
    spread = (x.double().reshape(b, n, g, -1) - m64[:, None, :, None]).abs().amax((1, 3))
    ok(mean, (m64, 32 * ref.F32 * 2 * spread + 2 * ref.F32 * m64.abs() + 1e-30))
    ok(rstd, (r64, (64 + 64 * spread * r64) * ref.F32 * r64))
    dy = rnd(4, b, n, c, dtype=dtype)
    got = engine.group_norm_backward(dy, x, g, ga, be, mean, rstd, activation=kind)
    wants, bounds = ref.group_norm_backward(dy, x, g, ga, be, mean, rstd, kind)
    for a, w, e in zip(got, wants, bounds):
        ok(a, (w, e + 1e-30))
    again = engine.group_norm_backward(dy, x, g, ga, be, mean, rstd, activation=kind)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    none = engine.group_norm_backward(dy, x, g, ga, be, mean, rstd, activation=kind, need_dx=False)
    assert none[0] is None and torch.equal(none[1], got[1]) and torch.equal(none[2], got[2])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_activations_strides_and_no_affine(engine, kind, dtype):
    base = rnd(5, 3, 40, 2, 24, dtype=dtype)
    x = base[:, :, 1]                                       # positions 48 apart
    ok(engine.group_norm(x, 3, activation=kind), ref.group_norm(x, 3, None, None, 1e-5, kind)[:2])
    out = torch.full((3, 41, 24), 7.0, device="cuda", dtype=dtype)
    engine.group_norm(x, 3, activation=kind, out=out[:, :40])
    ok(out[:, :40], ref.group_norm(x, 3, None, None, 1e-5, kind)[:2])
    assert (out[:, 40] == 7.0).all()                        # the row behind each item is left as it was
    odd = rnd(6, 3, 40, 25, dtype=dtype)[..., 1:]           # addresses that are not whole vectors
    ga = rnd(7, 24, dtype=dtype)
    want = ref.group_norm(odd, 4, ga, None, 1e-3, kind)[:2]
    ok(engine.group_norm(odd, 4, ga, eps=1e-3, activation=kind), want)
    image = rnd(8, 2, 5, 8, 24, dtype=dtype)                # [batch][height][width][channels]
    got = engine.group_norm(image, 6, ga, activation=kind)
    w, e = ref.group_norm(image.flatten(1, 2), 6, ga, None, 1e-5, kind)[:2]
    ok(got.flatten(1, 2), (w, e))
    y, mean, rstd = engine.group_norm(image, 6, None, ga, activation=kind, return_stats=True)
    dy = rnd(9, 1, 1, 1, 24, dtype=dtype).expand(2, 5, 8, 24)   # a broadcast gradient
    dx, dg, db = engine.group_norm_backward(dy, image, 6, None, ga, mean, rstd, activation=kind)
    wants, bounds = ref.group_norm_backward(dy.reshape(2, 40, 24), image.flatten(1, 2), 6, None, ga, mean, rstd, kind)
    assert dg is None
    ok(dx.flatten(1, 2), (wants[0], bounds[0]))
    ok(db, (wants[2], bounds[2] + ref.half_ulp(dtype) * wants[2].abs()))
    z = image.clone()
    assert torch.equal(engine.group_norm(z, 6, ga, activation=kind, out=z), got) and torch.equal(z, got)


def test_group_norm_far_mean_empty_and_special(pkg, engine):
    x = rnd(10, 2, 3000, 16, scale=0.01, shift=300.0)       # the mean is 30 000 deviations away
    ok(engine.group_norm(x, 2), ref.group_norm(x, 2, None, None, 1e-5, "none")[:2])
    for dtype, value in ((F32, 3.0), (F16, 60000.0), (BF16, 300.0)):        # a constant group is its beta, whatever its mean
        for n in (77, 70000):
            const = torch.full((1, n, 16), value, device="cuda", dtype=dtype)
            be = rnd(3, 16, dtype=dtype)
            assert torch.equal(engine.group_norm(const, 2, None, be), be.expand(1, n, 16))
    for shape in ((0, 5, 8), (2, 0, 8)):
        e = torch.empty(shape, device="cuda")
        ga = torch.ones(8, device="cuda")
        y, mean, rstd = engine.group_norm(e, 2, ga, ga, return_stats=True)
        assert y.shape == shape
        dx, dg, db = engine.group_norm_backward(e, e, 2, ga, ga, mean, rstd)
        assert dx.shape == shape and (dg == 0).all() and (db == 0).all()
    x = rnd(11, 2, 50, 8)
    x[0, 7, 1], x[1, 3, 6] = math.nan, math.inf
    y = engine.group_norm(x, 2, activation="silu")
    assert torch.isnan(y[0, :, :4]).all() and torch.isnan(y[1, :, 4:]).all()
    ok(y[0, :, 4:][None], ref.group_norm(x[:1, :, 4:], 1, None, None, 1e-5, "silu")[:2])
    ok(y[1, :, :4][None], ref.group_norm(x[1:, :, :4], 1, None, None, 1e-5, "silu")[:2])


def test_group_norm_gradient_by_differences(engine):
    """In float the difference quotient of a sum of 2000 outputs is good to a few 1e-3 of its size."""
    x, v, dy = rnd(12, 2, 100, 12), rnd(13, 2, 100, 12), rnd(14, 2, 100, 12)
    ga, be = rnd(15, 12, shift=1.0), rnd(16, 12)
    y, mean, rstd = engine.group_norm(x, 3, ga, be, activation="gelu", return_stats=True)
    dx, dg, db = engine.group_norm_backward(dy, x, 3, ga, be, mean, rstd, activation="gelu")
    h = 2.0 ** -6     # second-order error h^2 times third derivatives; rounding 2^-24 / h per output
    up, dn = (engine.group_norm(x + s * h * v, 3, ga, be, activation="gelu").double() for s in (1, -1))
    diff, want = float(((up - dn) * dy.double()).sum() / (2 * h)), float((dx.double() * v.double()).sum())
    size = float((dx.double() * v.double()).abs().sum())
    assert abs(diff - want) <= 4e-3 * size


def test_group_norm_refusals(pkg, engine):
    x = torch.zeros(2, 6, 8, device="cuda")
    ga = torch.ones(8, device="cuda")
    for call in (lambda: engine.group_norm(x, 3), lambda: engine.group_norm(x, 0), lambda: engine.group_norm(x, 2, eps=-1.0),
                 lambda: engine.group_norm(x, 2, activation="tanh"), lambda: engine.group_norm(x, 2, torch.ones(7, device="cuda")),
                 lambda: engine.group_norm(x, 2, ga.half()), lambda: engine.group_norm(x, 2, ga, ga.half()),
                 lambda: engine.group_norm(x.transpose(1, 2), 2), lambda: engine.group_norm(x, 2, out=torch.zeros(2, 6, 8)),
                 lambda: engine.group_norm(x, 2, out=torch.zeros(1, 6, 8, device="cuda").expand(2, 6, 8)),
                 lambda: engine.group_norm(x.view(2, 2, 3, 8).transpose(1, 2), 2), lambda: engine.group_norm(x.double(), 2)):
        with pytest.raises(pkg.StemsError) as err:
            call()
        assert err.value.code in (1, 2)
    import ctypes as C
    with pytest.raises(pkg.StemsError, match="8192 channels"):      # the reason comes along
        engine.group_norm(torch.zeros(1, 2, 8200, device="cuda"), 1)
    n = C.c_size_t()
    for positions, channels, groups in ((5, 4096, 4096), (60000, 16, 4)):     # three launches; all SMs at once
        cfg = pkg.GroupNormConfig(C.sizeof(pkg.GroupNormConfig), 0, 0, 0, 1, positions, channels, groups, 0, channels, 0, channels, 0,
                                  channels, 1e-5)
        cfg.x_batch = cfg.y_batch = cfg.dx_batch = positions * channels
        x = torch.zeros(1, positions, channels, device="cuda")
        y = torch.zeros_like(x)
        args = (engine._h, C.byref(cfg), x.data_ptr(), None, None, y.data_ptr(), None, None)
        assert pkg.lib().stg_group_norm_workspace(C.byref(cfg), 0, C.byref(n)) == 0 and n.value > 0
        ws = torch.empty(n.value + 256, dtype=torch.uint8, device="cuda")
        assert pkg.lib().stg_group_norm(*args, ws.data_ptr(), n.value, None) == 0
        assert pkg.lib().stg_group_norm(*args, None, 0, None) == 1
        assert pkg.lib().stg_group_norm(*args, ws.data_ptr(), 0, None) == 1
        assert pkg.lib().stg_group_norm(*args, ws.data_ptr() + 8, n.value, None) == 1
    assert "workspace" in engine.last_error()


# ---- gated projection ---------------------------------------------------------------------------
GATED = [
    # rows, features, width
    (1, 1, 1), (1, 64, 64), (1, 2048, 333), (3, 40, 8), (7, 129, 65), (16, 384, 1408), (17, 256, 130), (128, 64, 64), (129, 200, 200),
    (300, 72, 1000), (1000, 384, 136), (257, 515, 301), (33, 16, 2050), (640, 1024, 64), (2000, 8, 24),
    (40, 1, 1), (20, 3, 2), (9, 72, 16), (8, 72, 17), (2, 1000, 5), (5, 40, 3000), (300, 2200, 40),
    (32, 1030, 600), (33, 260, 2400), (128, 1100, 1000), (4000, 33, 30),   # in groups of eight rows, and tiles
]


def _gated_inputs(rows, k, n, dtype, bias=True, seed=0):
    s = 100 * seed
    return (rnd(s + 1, rows, k, dtype=dtype), rnd(s + 2, n, k, dtype=dtype, scale=k ** -0.5), rnd(s + 3, n, k, dtype=dtype, scale=k ** -0.5),
            *((rnd(s + 4, n, dtype=dtype), rnd(s + 5, n, dtype=dtype)) if bias else (None, None)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", GATED)
def test_gated_and_backward(engine, shape, dtype):
    kind = KINDS[sum(shape) % 5]
    bias = shape[0] % 2 == 1
    x, wg, wu, bg, bu = _gated_inputs(*shape, dtype, bias)
    ok(engine.gated(x, wg, wu, bg, bu, activation=kind), ref.gated(x, wg, wu, bg, bu, kind))
    dy = rnd(9, shape[0], shape[2], dtype=dtype)
    got = engine.gated_backward(dy, x, wg, wu, bg, bu, activation=kind)
    want, bound = ref.gated_backward(dy, x, wg, wu, bg, bu, kind)
    assert len(got) == (5 if bias else 3)
    for a, w, e in zip(got, want, bound):
        ok(a, (w, e))
    again = engine.gated_backward(dy, x, wg, wu, bg, bu, activation=kind)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    part = engine.gated_backward(dy, x, wg, wu, bg, bu, activation=kind, need_dx=False)
    assert part[0] is None and all(torch.equal(a, b) for a, b in zip(got[1:], part[1:]))
    part = engine.gated_backward(dy, x, wg, wu, activation=kind, need_dw=False) if not bias else None
    assert part is None or (torch.equal(part[0], got[0]) and part[1] is None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_gated_activations_strides_and_one_bias(engine, dtype, kind):
    x = rnd(1, 5, 60, 2, 72, dtype=dtype)[:, :, 1]           # rows 144 apart
    w = rnd(2, 2, 48, 80, dtype=dtype, scale=0.12)
    wg, wu = w[0, :, :72], w[1, :, 8:]                       # rows 80 apart
    bu = rnd(3, 48, dtype=dtype)
    flat = x.reshape(-1, 72)
    out = torch.full((5, 60, 56), 7.0, device="cuda", dtype=dtype)
    engine.gated(x, wg, wu, None, bu, activation=kind, out=out[..., :48])
    ok(out[..., :48].reshape(-1, 48), ref.gated(flat, wg, wu, None, bu, kind))
    assert (out[..., 48:] == 7.0).all()
    dy = rnd(4, 48, dtype=dtype).expand(5, 60, 48)           # one gradient for every row
    got = engine.gated_backward(dy, x, wg, wu, None, bu, activation=kind)
    want, bound = ref.gated_backward(dy.reshape(-1, 48), flat, wg, wu, None, bu, kind)
    assert got[0].shape == x.shape and len(got) == 4
    for a, i in zip(got, (0, 1, 2, 4)):
        ok(a.reshape(want[i].shape), (want[i], bound[i]))
    odd = rnd(5, 70, 73, dtype=dtype)[:, 1:]                 # addresses that are not whole vectors
    ok(engine.gated(odd, wg, wu, activation=kind), ref.gated(odd, wg, wu, None, None, kind))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 200])
def test_gated_broadcast_and_overlapping_operands(engine, dtype, rows):
    x, wg, wu, _, _ = _gated_inputs(rows, 64, 72, dtype, False)
    one, base, dy = x[:1].expand(rows, 64), rnd(7, rows + 64, dtype=dtype), rnd(8, rows, 72, dtype=dtype)
    windows, same = base.as_strided((rows, 64), (1, 1)), wu[:1].expand(72, 64)
    for a, w in ((one, wu), (windows, wu), (x, same)):
        ok(engine.gated(a, wg, w), ref.gated(a, wg, w, None, None, "silu"))
        want, bound = ref.gated_backward(dy, a, wg, w, None, None, "silu")
        for got, i in zip(engine.gated_backward(dy, a, wg, w), range(3)):
            ok(got, (want[i], bound[i]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [40, 1200])          # one range of rows; parts that are joined
def test_gated_weight_gradients_in_padded_rows_and_alone(pkg, engine, dtype, rows):
    import ctypes as C
    k, n = 72, 200
    x, wg, wu, bg, bu = _gated_inputs(rows, k, n, dtype)
    dy = rnd(9, rows, n, dtype=dtype)
    want = engine.gated_backward(dy, x, wg, wu, bg, bu)
    bits = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    need = C.c_size_t()
    for row, off, asked in ((72, 0, (1, 1)), (80, 0, (1, 1)), (80, 1, (1, 1)), (77, 0, (1, 1)), (80, 0, (1, 0)), (80, 8, (0, 1)), (72, 0, (0, 0))):
        cfg = pkg.GatedConfig(C.sizeof(pkg.GatedConfig), bits, pkg.ACTIVATIONS["silu"], k, n, rows, k, k, k, n, k, row, row)
        assert pkg.lib().stg_gated_workspace(C.byref(cfg), 1, C.byref(need)) == 0
        ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
        dw = [torch.full((off + n * row,), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        db = [torch.empty(n, dtype=dtype, device="cuda") for _ in range(2)]
        ptr = [t[off:].data_ptr() if a else None for t, a in zip(dw, asked)]
        args = [t.data_ptr() for t in (dy, x, wg, wu, bg, bu)] + [None, *ptr, *(t.data_ptr() for t in db)]
        assert pkg.lib().stg_gated_backward(engine._h, C.byref(cfg), *args, ws.data_ptr(), need.value,
                                            torch.cuda.current_stream().cuda_stream) == 0
        for t, a, w, b, v in zip(dw, asked, want[1:3], db, want[3:]):
            got = t[off:].view(n, row)
            assert torch.equal(got[:, :k], w) if a else (t == 7).all()
            assert (got[:, k:] == 7).all() and (t[:off] == 7).all() and torch.equal(b, v)


def test_gated_empty_special_and_refusals(pkg, engine):
    wg, wu = rnd(1, 24, 16), rnd(2, 24, 16)
    e = torch.empty(0, 16, device="cuda")
    assert engine.gated(e, wg, wu).shape == (0, 24)
    dx, dg, du, db = engine.gated_backward(torch.empty(0, 24, device="cuda"), e, wg, wu, torch.ones(24, device="cuda"))
    assert dx.shape == (0, 16) and (dg == 0).all() and (du == 0).all() and (db == 0).all()
    for dtype in TYPES:
        # a NaN or infinity stays in its own row, and in its own column where a weight has it
        x, wg, wu, _, _ = _gated_inputs(200, 64, 72, dtype, False)
        clean = engine.gated(x, wg, wu)
        x[5, 3], x[150, 60] = math.nan, math.inf
        wu[70, 1] = math.nan
        y = engine.gated(x, wg, wu)
        assert torch.isnan(y[5]).all() and torch.isnan(y[:, 70]).all() and not torch.isfinite(y[150]).any()
        keep = [i for i in range(200) if i not in (5, 150)]
        cols = [i for i in range(72) if i != 70]
        assert torch.equal(y[keep][:, cols], clean[keep][:, cols])
    x = torch.zeros(4, 16, device="cuda")
    wg, wu = torch.zeros(24, 16, device="cuda"), torch.zeros(24, 16, device="cuda")
    for call in (lambda: engine.gated(x, wg, wu[:, :8]), lambda: engine.gated(x, wg, wu[:8]), lambda: engine.gated(x, wg, wu.half()),
                 lambda: engine.gated(x, wg, wu, torch.zeros(23, device="cuda")), lambda: engine.gated(x, wg, wu, activation="tanh"),
                 lambda: engine.gated(x, wg.t().contiguous().t(), wu), lambda: engine.gated(x[0], wg, wu),
                 lambda: engine.gated(x, wg, wu, out=torch.zeros(4, 25, device="cuda")),
                 lambda: engine.gated(x, wg, wu, out=torch.zeros(1, 24, device="cuda").expand(4, 24)),
                 lambda: engine.gated_backward(torch.zeros(4, 23, device="cuda"), x, wg, wu),
                 lambda: engine.gated(torch.zeros(4, 0, device="cuda"), torch.zeros(24, 0, device="cuda"), torch.zeros(24, 0, device="cuda"))):
        with pytest.raises(pkg.StemsError) as err:
            call()
        assert err.value.code in (1, 2)


def test_gated_gradient_by_differences(engine):
    x, wg, wu, bg, bu = _gated_inputs(40, 24, 30, F32)
    dy = rnd(9, 40, 30)
    got = engine.gated_backward(dy, x, wg, wu, bg, bu, activation="silu")
    h = 2.0 ** -6
    for i, t in enumerate((x, wg, wu, bg, bu)):
        v = rnd(20 + i, *t.shape)
        args = [x, wg, wu, bg, bu]
        ends = []
        for s in (h, -h):
            args[i] = t + s * v
            ends.append(engine.gated(*args, activation="silu").double())
        diff, terms = ((ends[0] - ends[1]) * dy.double()).sum() / (2 * h), got[i].double() * v.double()
        assert abs(float(diff - terms.sum())) <= 4e-3 * float(terms.abs().sum())


# ---- the mask head ------------------------------------------------------------------------------
def _plan(pkg, engine, bands, frames, stems=1, channels=2):
    sizes, freqs = pkg.bands.mel_bands() if bands == "mel" else pkg.bands.bs_bands()
    chunk = 441 * (frames - 1)
    return engine.plan_roformer(chunk, sizes, freqs, n_stems=stems, n_channels=channels, chunk=chunk, num_overlap=1), [int(s) * 2 * channels for s in sizes]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [("mel", 10, 1, 2, 1, 64, True), ("bs", 40, 2, 2, 2, 72, False), ("mel", 131, 1, 1, 1, 33, True), ("bs", 8, 1, 1, 3, 250, True)])
def test_mask_head(pkg, engine, case, dtype):
    bands, frames, stems, channels, chunks, k, bias = case
    plan, din = _plan(pkg, engine, bands, frames, stems, channels)
    assert plan.mask_head_sizes() == (stems, len(din), frames, sum(din))
    h = torch.tanh(rnd(1, chunks, stems, len(din), frames, k)).to(dtype)
    w, b = rnd(2, stems, 2 * sum(din), k, dtype=dtype, scale=k ** -0.5), rnd(3, stems, 2 * sum(din), dtype=dtype) if bias else None
    out = torch.full((chunks * plan.mask_floats_per_chunk + 5,), 7.0, device="cuda")
    plan.mask_head(h, w, b, out=out[:-5].view(chunks, -1))
    ok(out[:-5].view(chunks, -1), ref.mask_head(h, w, b, din))
    assert (out[-5:] == 7.0).all()
    assert torch.equal(plan.mask_head(h, w, b).flatten(), out[:-5])
    for band in (0, len(din) - 1):        # a NaN in a band's hidden rows stays in that frame and band
        g = h.clone()
        g[0, 0, band, 1, 0] = math.nan
        y = plan.mask_head(g, w, b).flatten()
        at = sum(din[:band]) * frames + din[band]
        assert torch.isnan(y[at:at + din[band]]).all() and int(torch.isnan(y).sum()) == din[band]


def test_mask_head_refusals(pkg, engine):
    plan, din = _plan(pkg, engine, "mel", 10)
    h, w = torch.zeros(1, 1, 60, 10, 16, device="cuda"), torch.zeros(1, 2 * sum(din), 16, device="cuda")
    plan.mask_head(h, w)
    assert plan.mask_head(h[:0], w).shape == (0, plan.mask_floats_per_chunk)
    for call in (lambda: plan.mask_head(h[:, :, :59], w), lambda: plan.mask_head(h, w[:, 1:]), lambda: plan.mask_head(h, w.half()),
                 lambda: plan.mask_head(h, w, torch.zeros(1, 3, device="cuda")), lambda: plan.mask_head(h.transpose(2, 3).contiguous().transpose(2, 3), w),
                 lambda: plan.mask_head(h, w, out=torch.zeros(3, device="cuda")),
                 lambda: engine.plan_tfc(441 * 400, dim_t=256).mask_head(h, w)):
        with pytest.raises(pkg.StemsError) as err:
            call()
        assert err.value.code == 1


# ---- as they are used ---------------------------------------------------------------------------
def test_a_network_of_the_layers_between_the_halves(pkg, engine):
    """A one-layer RoFormer built of the layers, run as separate_network's callback: the masks
    it writes, given to separate(), give the same separation."""
    sizes, freqs = pkg.bands.mel_bands()
    chunk, T, nb, K, H = 441 * 20, 21, 60, 64, 4
    n = chunk * 2 + 777
    plan = engine.plan_roformer(n, sizes, freqs, chunk=chunk, num_overlap=2)
    din = [int(s) * 4 for s in sizes]
    w_in = [rnd(10 + b, d, K, scale=d ** -0.5) for b, d in enumerate(din)]
    w_qkv, w_out = rnd(1, 3 * K, K, scale=K ** -0.5), rnd(2, K, K, scale=K ** -0.5)
    wg, wu, wd = rnd(3, 96, K, scale=K ** -0.5), rnd(4, 96, K, scale=K ** -0.5), rnd(5, K, 96, scale=0.1)
    w_head, b_head = rnd(6, 1, 2 * sum(din), K, scale=K ** -0.5), rnd(7, 1, 2 * sum(din))
    n_in, n_out = plan.network_info()
    masks = torch.zeros(plan.n_chunks, n_out, device="cuda")

    class Floats:
        def __init__(self, ptr, count):
            self.__cuda_array_interface__ = dict(shape=(count,), typestr="<f4", data=(ptr, False), version=3)

    def layer(feat):                       # [c][n_in] -> hidden [c][1][bands][T][K]
        c = feat.shape[0]
        parts, at = [], 0
        for b, d in enumerate(din):
            parts.append(feat[:, at:at + d * T].view(c, T, d) @ w_in[b])
            at += d * T
        x = torch.stack(parts, 1).view(c * nb, T, K)
        x = engine.group_norm(x, 1, activation="none")
        qkv = (x @ w_qkv.t()).view(c * nb, T, 3, H, K // H)
        q, k = engine.rotary(qkv[:, :, 0], qkv[:, :, 1])
        p = torch.softmax(torch.einsum("bthd,bshd->bhts", q, k) * (K // H) ** -0.5, -1)
        x = x + torch.einsum("bhts,bshd->bthd", p, qkv[:, :, 2]).reshape(c * nb, T, K) @ w_out.t()
        x = x + engine.gated(x, wg, wu, activation="silu") @ wd.t()
        return x.view(c, 1, nb, T, K)

    def network(first, count, p_in, p_out, stream):
        feat = torch.as_tensor(Floats(p_in, count * n_in), device="cuda").view(count, n_in)
        plan.mask_head(layer(feat), w_head, b_head, out=p_out)
        masks[first:first + count] = torch.as_tensor(Floats(p_out, count * n_out), device="cuda").view(count, n_out)

    mix = rnd(8, 2, n, scale=0.1)
    out, again = (torch.empty(plan.out_shape, device="cuda") for _ in range(2))
    plan.separate_network(mix, out, network, chunks_per_batch=2)
    assert torch.isfinite(out).all() and float(masks.abs().amax()) > 0.1
    plan.separate(mix, masks, again)
    # the same masks through the fused path: the kernels' own parity bar, 1e-5 of the largest sample
    assert float((out - again).abs().max()) <= 1e-5 * float(again.abs().max())


def _calls(engine, pkg):
    """One call of each layer, with what it returned before."""
    x, wg, wu, bg, bu = _gated_inputs(130, 64, 72, BF16)
    dy = rnd(9, 130, 72, dtype=BF16)
    q = rnd(1, 2, 30, 4, 32, dtype=BF16)
    h = rnd(2, 3, 200, 48, dtype=BF16)
    dh = rnd(3, 3, 200, 48, dtype=BF16)
    ga, be = rnd(4, 48), rnd(5, 48)
    _, mean, rstd = engine.group_norm(h, 4, ga, be, return_stats=True)
    plan, din = _plan(pkg, engine, "bs", 12)
    hidden, w = rnd(6, 1, 1, 62, 12, 40, dtype=BF16), rnd(7, 1, 2 * sum(din), 40, dtype=BF16, scale=0.15)
    return {
        "rotary": (lambda s: [engine.rotary(q, stream=s)], [q]),
        "norm": (lambda s: [engine.group_norm(h, 4, ga, be, activation="gelu", stream=s)], [h]),
        "norm_back": (lambda s: list(engine.group_norm_backward(dh, h, 4, ga, be, mean, rstd, activation="gelu", stream=s)), [h, dh]),
        "gated": (lambda s: [engine.gated(x, wg, wu, bg, bu, stream=s)], [x]),
        "gated_back": (lambda s: list(engine.gated_backward(dy, x, wg, wu, bg, bu, stream=s)), [x, dy]),
        "head": (lambda s: [plan.mask_head(hidden, w, stream=s)], [hidden]),
    }


@pytest.mark.parametrize("name", ["rotary", "norm", "norm_back", "gated", "gated_back", "head"])
def test_layers_in_graphs_and_on_streams(pkg, engine, name):
    call, inputs = _calls(engine, pkg)[name]
    before = [t.clone() for t in inputs]
    want = call(None)
    torch.cuda.synchronize()
    # two graphs of the same call, replayed on two streams at once, with new inputs in place
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(None)
        graphs.append((g, out))
    for t in inputs:
        t.neg_()
    fresh = call(None)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, fresh))
    for t, b in zip(inputs, before):
        t.copy_(b)
    torch.cuda.synchronize()
    # a stream of its own, as an object and as a handle; calls overlap there
    both = [call(streams[0]), call(streams[1].cuda_stream)]
    torch.cuda.synchronize()
    for out in both:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert all(torch.equal(a, b) for a, b in zip(inputs, before))


def test_no_kernel_gave_up(engine):
    engine.status()
