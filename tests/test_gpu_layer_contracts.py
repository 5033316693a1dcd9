"""The layers' contracts on the GPU, beyond their results: what one call may do to another."""
from __future__ import annotations

import ctypes as C
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def rnd(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# positions x channels x groups, large and small calls of one kernel: clusters; the three launches, whose
# shared memory goes with the groups
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("large, small", [((180, 2048, 1), (100, 2048, 1)), ((40, 8192, 8192), (40, 7000, 7000))])
def test_two_engines_in_two_threads(pkg, large, small, backward):
    """Engines of one device, one to a host thread: neither's calls are refused for the other's sizes."""
    start, faults, L = threading.Barrier(2), [], pkg.lib()
    torch.cuda.synchronize()

    def work(seed, n, ch, groups):
        try:
            engine, stream = pkg.Engine(0), torch.cuda.Stream()
            with torch.cuda.stream(stream):
                x, dy, ga = rnd(seed, 1, n, ch), rnd(seed + 1, 1, n, ch), rnd(seed + 2, ch)
                y, mean, rstd = engine.group_norm(x, groups, ga, ga, return_stats=True)
                want = engine.group_norm_backward(dy, x, groups, ga, ga, mean, rstd) if backward else (y,)
            got = [torch.empty_like(t) for t in want]
            cfg = pkg.GroupNormConfig(C.sizeof(pkg.GroupNormConfig), 0, 0, 0, 1, n, ch, groups, n * ch, ch, n * ch, ch, n * ch, ch, 1e-5)
            need = C.c_size_t()
            assert L.stg_group_norm_workspace(C.byref(cfg), int(backward), C.byref(need)) == 0
            ws = torch.empty(max(need.value, 256), dtype=torch.uint8, device="cuda")
            ptr = lambda *ts: [t.data_ptr() for t in ts]  # noqa: E731
            args = (engine._h, C.byref(cfg), *(ptr(dy, x, ga, ga, mean, rstd, *got) if backward else [*ptr(x, ga, ga), *ptr(*got), None, None]),
                    ws.data_ptr(), need.value, stream.cuda_stream)
            stream.synchronize()
            call = L.stg_group_norm_backward if backward else L.stg_group_norm
            start.wait(30)
            for i in range(3000):
                if call(*args) != 0:
                    faults.append(engine.last_error())
                if i % 200 == 0:
                    stream.synchronize()
            stream.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                faults.append("other results than alone")
            engine.close()
        except Exception as e:   # a thread's failure is the test's
            faults.append(repr(e))
            start.abort()

    threads = [threading.Thread(target=work, args=(10 * i, *shape)) for i, shape in enumerate((large, small))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not faults, (len(faults), faults[0])


@pytest.mark.parametrize("shape", [(2, 40, 24, 3), (3, 5, 4104, 1026), (2, 30000, 24, 2)])      # a cluster; three launches; the same, large
def test_group_norm_parameter_gradients_alone(pkg, engine, shape):
    """Without dx its strides say nothing: a broadcast dy is fine, and so are strides of 0."""
    b, n, ch, groups = shape
    x, dy, ga = rnd(1, b, n, ch), rnd(2, ch).expand(b, n, ch), rnd(3, ch)
    _, mean, rstd = engine.group_norm(x, groups, ga, ga, activation="silu", return_stats=True)
    want = engine.group_norm_backward(dy, x, groups, ga, ga, mean, rstd, activation="silu")
    got = engine.group_norm_backward(dy, x, groups, ga, ga, mean, rstd, activation="silu", need_dx=False)
    assert got[0] is None and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    need, L = C.c_size_t(), pkg.lib()
    for dx_strides in ((0, 0), (1, 1)):      # of which the second would allow scalar accesses only
        cfg = pkg.GroupNormConfig(C.sizeof(pkg.GroupNormConfig), 0, 0, pkg.ACTIVATIONS["silu"], b, n, ch, groups, n * ch, ch, 0, 0, *dx_strides, 1e-5)
        assert L.stg_group_norm_workspace(C.byref(cfg), 1, C.byref(need)) == 0
        ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
        grads = [torch.full((ch,), 7.0, device="cuda") for _ in range(2)]
        ins = [t.data_ptr() for t in (dy, x, ga, ga, mean, rstd)]
        stream = torch.cuda.current_stream().cuda_stream
        for asked in ((1, 1), (1, 0), (0, 1)):
            for g in grads:
                g.fill_(7.0)
            outs = [g.data_ptr() if a else None for g, a in zip(grads, asked)]
            assert L.stg_group_norm_backward(engine._h, C.byref(cfg), *ins, None, *outs, ws.data_ptr(), need.value, stream) == 0, engine.last_error()
            for g, a, w in zip(grads, asked, want[1:]):
                assert torch.equal(g, w) if a else (g == 7).all()
        dx = torch.empty_like(x)             # with dx they count
        assert L.stg_group_norm_backward(engine._h, C.byref(cfg), *ins, dx.data_ptr(), None, None, ws.data_ptr(), need.value, stream) == 1


def test_status_waits_for_every_stream(engine):
    """torch's streams do not block the default one, on which the flag is read."""
    engine.status()
    stream, done = torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(200_000_000)
        done.record()
    engine.status()
    assert done.query()


def _segment_stream(t):
    at = t.data_ptr()
    return next(s["stream"] for s in torch.cuda.memory_snapshot() if s["address"] <= at < s["address"] + s["total_size"])


def test_results_come_from_the_streams_own_pool(engine):
    """Memory of another stream's pool could still be in use there: handle 0 is the default stream."""
    x, w = rnd(1, 1, 30000, 64), rnd(2, 64, 64)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for stream, pool in ((0, 0), (torch.cuda.default_stream(), 0), (None, side.cuda_stream), (side, side.cuda_stream), (side.cuda_stream, side.cuda_stream)):
            for y in (engine.group_norm(x, 4, stream=stream), engine.gated(x, w, w, stream=stream), engine.rotary(x[None], stream=stream)):
                assert _segment_stream(y) == pool
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_mask_heads_sigmoid_is_a_floats(pkg, engine, dtype):
    """The masks are float whatever the inputs' type: sigmoid to 16 half units of the last place over
    [-60, 60], with projections that are exact (one feature of 1, the others 0). The parts, in
    2^-24: power of two and reciprocal 2^-22 each (4 + 4), what the exponent's correction leaves 1,
    the sum 1, the value's product 1."""
    sizes, freqs = pkg.bands.bs_bands()
    plan = engine.plan_roformer(441 * 11, sizes, freqs, chunk=441 * 11, num_overlap=1)
    din = [int(s) * 4 for s in sizes]
    _, bands, frames, cols = plan.mask_head_sizes()
    hidden, weight = torch.zeros(1, 1, bands, frames, 8, device="cuda", dtype=dtype), torch.zeros(1, 2 * cols, 8, device="cuda", dtype=dtype)
    hidden[..., 0] = 1
    want, at = [], 0
    for d in din:
        weight[0, at:at + d, 0] = 1
        z = ((torch.arange(d, device="cuda") % 121 - 60) * 0.99609375).to(dtype)
        weight[0, at + d:at + 2 * d, 0] = z
        want.append(torch.sigmoid(z.double()).expand(frames, d).reshape(-1))
        at += 2 * d
    want = torch.cat(want)
    got = plan.mask_head(hidden, weight).double().flatten()
    assert float(((got - want).abs() / want).max()) <= 16 * 2.0 ** -24


@pytest.mark.parametrize("k", [30.0, 1000.0, 100000.0])
@pytest.mark.parametrize("shape", [(296, 1 << 20, 1, 1), (300, 40000, 64, 2), (4, 172032, 24, 8), (3, 5000, 48, 4)])
def test_group_norm_statistics_behind_an_outlier(engine, shape, k):
    """The first position k deviations from the rest costs the statistics no digits. A thread adds up n
    squares in order, n roundings of their sum; the pivot's turns and the joining of the parts
    count 128 more: the variance is good to (n + 128) 2^-24, rstd to half of that and its own 8
    roundings, the mean to as much of the deviation it is off by at most."""
    b, n, ch, groups = shape
    x = torch.randn(shape[:3], generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    x[:, 0] = k
    _, mean, rstd = engine.group_norm(x, groups, return_stats=True)
    chunks = max(1, -(-296 // b))
    wide = 4 if ch % 4 == 0 else 1
    terms = -(-n // chunks) // (256 // (ch // wide)) + 1            # of a thread
    for i in (0, b // 2, b - 1):
        d = x[i].double().reshape(n, groups, -1)
        mu = d.mean((0, 2))
        var = (d - mu[:, None]).square().mean((0, 2))
        want = 1 / torch.sqrt(var + 1e-5)
        assert float(((rstd[i] - want).abs() / want).max()) <= ((terms * wide + 128) / 2 + 8) * 2.0 ** -24
        assert float(((mean[i] - mu).abs() * want).max()) <= (terms * wide + 128) * 2.0 ** -24


def _large_calls(engine):
    bf = torch.bfloat16
    x, dx, many, dmany = rnd(1, 2, 30000, 24), rnd(2, 2, 30000, 24), rnd(3, 20, 3000, 96, dtype=bf), rnd(4, 20, 3000, 96, dtype=bf)
    ga, gb = rnd(5, 24), rnd(6, 96)
    stats, more = engine.group_norm(x, 3, ga, ga, return_stats=True)[1:], engine.group_norm(many, 8, gb, gb, return_stats=True)[1:]
    h, dh, w, v = rnd(7, 3000, 200, dtype=bf), rnd(8, 3000, 300, dtype=bf), rnd(9, 300, 200, dtype=bf, scale=0.07), rnd(10, 300, 200, dtype=bf, scale=0.07)
    odd = rnd(11, 3000, 203, dtype=bf)[:, 2:202]                  # rows that are copied first
    return {
        "norm": lambda: [engine.group_norm(x, 3, ga, ga, activation="gelu")],
        "norm_back": lambda: list(engine.group_norm_backward(dx, x, 3, ga, ga, *stats, activation="silu")),
        "norm_back_many": lambda: list(engine.group_norm_backward(dmany, many, 8, gb, gb, *more, activation="silu")),
        "gated": lambda: [engine.gated(odd, w, v, gb.new_ones(300).to(bf))],
        "gated_back": lambda: list(engine.gated_backward(dh, h, w, v, gb.new_ones(300).to(bf))),
    }


@pytest.mark.parametrize("name", ["norm", "norm_back", "norm_back_many", "gated", "gated_back"])
def test_calls_of_several_launches_in_graphs_and_overlapping(engine, name):
    """Launches that begin before the one before them has ended, and scratch between them: captured
    twice in a row, replayed on two streams at once, and eager calls side by side."""
    call = _large_calls(engine)[name]
    want = call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = [call(), call()]
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    outs = [o for _, both in graphs for o in both]
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(call())
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
