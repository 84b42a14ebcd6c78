"""Calls of different sizes from several threads at once: each succeeds."""

import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


def _together(calls, times):
    """Each call `times` times in a thread of its own, all at once; what they raised."""
    errors = []
    start = threading.Barrier(len(calls))

    def loop(call):
        start.wait()
        try:
            for _ in range(times):
                call()
        except Exception as e:  # the thread's error is the test's
            errors.append(e)

    threads = [threading.Thread(target=loop, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return errors


def test_gathers_of_different_model_counts(gpu, torch):
    """Feature-major gathers of many rows keep counts of each model in shared memory."""
    from test_mixture_gpu import sort_on_gpu
    core = gpu
    rows = 65_536
    calls, checks = [], []
    for experts in (1, 1_024) * 2:
        ids = np.random.default_rng(experts).integers(0, experts, (rows, 1))
        offsets, counts, order, slots = sort_on_gpu(core, torch, ids, experts, 1)
        x = torch.randn((1, rows), device="cuda")
        out = torch.empty((1, rows), device="cuda")
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()

        def call(e=experts, p=(offsets, order, slots), x=x, out=out, s=stream):
            core.gather_rows_device(0, core.F32, x.data_ptr(), rows, 1, rows, 0, 1, e, p[0].data_ptr(),
                                    p[1].data_ptr(), p[2].data_ptr(), rows, out.data_ptr(), rows, 0,
                                    stream=s.cuda_stream)

        calls.append(call)
        checks.append((out, x[:, order.long()]))
    assert _together(calls, 3_000) == []
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in checks)


def test_heads_of_different_widths(gpu, torch):
    """Heads of few rows keep the rows in shared memory."""
    core = gpu
    calls, checks = [], []
    for cols in (64, 20_000) * 2:
        h = torch.randn((1, cols), device="cuda")
        w = torch.randn((40, cols), device="cuda")
        y = torch.zeros(1, dtype=torch.int32, device="cuda")
        loss, lse = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
        need = core.head_workspace(core.F32, 1, cols, 40)
        room = torch.empty(need, dtype=torch.uint8, device="cuda")
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()

        def call(d=cols, a=(h, w, y, loss, lse, room), need=need, s=stream):
            core.head_loss_device(0, core.F32, a[0].data_ptr(), 1, d, d, a[1].data_ptr(), 40, d,
                                  a[2].data_ptr(), a[3].data_ptr(), a[4].data_ptr(), a[5].data_ptr(),
                                  need, stream=s.cuda_stream)

        calls.append(call)
        checks.append((lse, torch.logsumexp(h.double() @ w.double().t(), 1)))
    assert _together(calls, 3_000) == []
    torch.cuda.synchronize()
    # sums of at most 20,000 float32 products of size one: 1e-3 of values above 100
    assert all(torch.allclose(a.double(), b, rtol=1e-3) for a, b in checks)
