"""The gated projection at sizes where a pair of SMs (tensor cores) or the GPU's blocks (CUDA cores)
take more than one tile: the accumulator sets in turn, the epilogue's two halves, operands ahead
for the next tile, the wide tiles, the splits by 4096 rows, and 16-bit operands at addresses that
the tensor cores do not take. Each case's dispatch is computed here again from the rules on sizes and
asserted, so that a later change of a rule cannot leave these paths unrun."""
from __future__ import annotations

import pytest
import torch

import layers_ref as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIRS = 74


def up(a, b):
    return -(-a // b)


def column_tile(k, rest, sums):
    most, best, width = 224 if sums else 256, None, 0
    few = up(k, most)
    for t in range(few, min(up(k, 64), few + 16) + 1):
        cols = up(up(k, t), 32) * 32
        cost = up(rest * up(k, cols), PAIRS) * (cols + 32)
        if best is None or cost < best:
            best, width = cost, cols
    return width


def mma_tiles(m, k, n, sums):
    """(outputs of a forward tile, forward tiles, dx tiles, dW tiles, dW splits)."""
    mt, tiles = up(m, 256), 2 * up(n, 256) * up(k, 224)
    out = 64 if mt * up(n, 128) < PAIRS else 128
    splits = max(1, min(max(1, PAIRS // tiles), m // 256, 64))
    splits = max(1, up(m, max(64, up(up(m, splits), 64) * 64)))
    rest = 2 * splits * up(n, 256)
    return out, mt * up(n, out), mt * up(k, column_tile(k, mt, False)), rest * up(k, column_tile(k, rest, sums)), splits


def simt_tiles(m, k, n, f32):
    """Tile sides of forward, dx and dW, and their splits (dx, dW)."""
    def side(rows, cols, out, y=1):
        return 128 if up(rows, 128) * up(cols, out) * y >= 222 else 64

    a, b = (128, 128) if f32 else (256, 224)
    tiles = 2 * up(n, a) * up(k, b)
    splits = max(1, min(up(296, tiles) if f32 else max(1, PAIRS // tiles), m // 256, 64))
    if f32:
        splits = max(splits, min(64, up(m, 4096)))
    splits = max(1, up(m, max(64, up(up(m, splits), 64) * 64)))
    dx = 1
    if f32:
        t128, t64 = up(m, 128) * up(k, 128), up(m, 64) * up(k, 64)
        dx = min(32, max(1, 1 if t128 >= 222 else min(up(296, t64), 2 * n // 256), up(2 * n, 4096)))
    return side(m, n, 64), side(m, k, 128, dx), side(n, k, 128, 2 * splits), dx, splits


def rnd(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def both_ways(engine, x, n, kind, bias):
    m, k, dtype = *x.shape, x.dtype
    wg, wu = (rnd(s, n, k, dtype=dtype, scale=k ** -0.5) for s in (2, 3))
    bg, bu = (rnd(s, n, dtype=dtype) for s in (4, 5)) if bias else (None, None)
    y = engine.gated(x, wg, wu, bg, bu, activation=kind)
    want, bound = ref.gated(x, wg, wu, bg, bu, kind)
    assert ref.worst(y, want, bound) <= 1.0
    del want, bound
    dy = rnd(9, m, n, dtype=dtype)
    got = engine.gated_backward(dy, x, wg, wu, bg, bu, activation=kind)
    wants, bounds = ref.gated_backward(dy, x, wg, wu, bg, bu, kind)
    for a, w, e in zip(got, wants, bounds):
        assert ref.worst(a, w, e) <= 1.0
    assert len(got) == (5 if bias else 3)
    again = engine.gated_backward(dy, x, wg, wu, bg, bu, activation=kind)
    assert all(torch.equal(a, b) for a, b in zip(got, again)) and torch.equal(y, engine.gated(x, wg, wu, bg, bu, activation=kind))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m, k, n, kind, bias, least", [
    # rows, features, width; then at least so many tiles to a pair: forward, dx, dW
    (6000, 72, 520, "silu", True, (2, 1, 1)),          # ragged rows and columns; an odd and an even tile to a pair
    (12001, 200, 650, "gelu", True, (4, 1, 1)),
    (20000, 600, 264, "sigmoid", False, (3, 4, 1)),
    (300, 1000, 4001, "relu", True, (1, 1, 3)),        # dW in one part, three and more tiles to a pair
    (5000, 712, 2600, "none", True, (6, 1, 2)),        # and over twenty slices of rows
])
def test_pairs_take_several_tiles(engine, m, k, n, kind, bias, least, dtype):
    out, fwd, dx, dw, splits = mma_tiles(m, k, n, bias)
    assert all(tiles > (l - 1) * PAIRS for tiles, l in zip((fwd, dx, dw), least)), (fwd, dx, dw)
    assert out == (128 if least[0] > 1 else 64)
    both_ways(engine, rnd(1, m, k, dtype=dtype), n, kind, bias)


@pytest.mark.parametrize("m, k, n, kind, sides, splits", [
    (5000, 700, 700, "silu", (128, 128, 128), (1, 5)),
    (9000, 1200, 2000, "gelu", (128, 128, 128), (1, 3)),         # rows in parts of at most 4096
    (2100, 260, 2100, "sigmoid", (128, 64, 128), (2, 3)),        # dx's terms in parts
    (16390, 40, 130, "none", (128, 64, 64), (1, 52)),
])
def test_float_tiles(engine, m, k, n, kind, sides, splits):
    got = simt_tiles(m, k, n, True)
    assert got[:3] == sides and got[3:] == splits, got
    both_ways(engine, rnd(1, m, k), n, kind, m % 2 == 0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m, k, n, sides", [(300, 72, 1000, (64, 64, 64)), (4000, 136, 1000, (128, 64, 128)), (2049, 1800, 1450, (128, 128, 128))])
def test_16_bit_operands_off_16_bytes(engine, m, k, n, sides, dtype):
    """An address off 16 bytes with rows a multiple of 16 bytes apart needs no copy by its strides, and
    takes the CUDA cores."""
    assert simt_tiles(m, k, n, False)[:3] == sides, simt_tiles(m, k, n, False)
    pitch = up(k, 8) * 8 + 8
    x = rnd(1, m * pitch + 8, dtype=dtype)[1:].as_strided((m, k), (pitch, 1), 1)
    assert x.data_ptr() % 16 == 2 and x.stride(0) % 8 == 0
    both_ways(engine, x, n, "silu", m % 2 == 1)
