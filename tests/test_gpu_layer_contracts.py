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
