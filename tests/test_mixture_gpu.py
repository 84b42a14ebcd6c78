"""Rows routed among several models: choice, sort, gather, combination and their
gradients on the GPU against plain numpy in 64 bits.

Tolerances.  A weight is exp(l - m) / S: the difference is rounded once (relative
error |l - m| u in the exponential, u = 2^-24), expf is within 2 units in the last
place, S sums E such values (at most E u more) and the division rounds once, so its
relative error is at most (|l - m| + E + 8) 2u.  A sum of products of k (or C) terms
in 32 bits is within (k + 2) u (or (C + 2) u) of the sum of the products' magnitudes.
A result of fewer bits adds half a unit in its last place: with p bits of significand at
most 2^-p of the value (bfloat16 p = 8, float16 p = 11) and the smallest subnormal's half.
A product that is rounded to 32 bits and then to its type is the same in numpy and on the
GPU, bit for bit."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


def _up(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _stream(torch):
    return torch.cuda.current_stream().cuda_stream


# ---- references ----------------------------------------------------------------

def ref_route(logits, k, norm):
    x = logits.astype(np.float64).copy()
    x[np.isnan(x)] = -np.inf
    order = np.argsort(-x, axis=1, kind="stable")[:, :k]
    top = np.take_along_axis(x, order, 1)
    found = top > -np.inf
    m = np.where(found[:, :1], top[:, :1], 0.0)
    e = np.exp(top - m)
    full = np.exp(x - m)
    total = full.sum(1, keepdims=True) if norm else e.sum(1, keepdims=True)
    total = np.where(total > 0, total, 1.0)
    return np.where(found, order, -1), e / total, full / total


def ref_route_grad(logits, ids, w, p, dw, norm):
    there = ids >= 0
    dw = np.where(there, dw, 0.0).astype(np.float64)
    mean = (w * dw).sum(1, keepdims=True)
    d = -p * mean if norm else np.zeros(logits.shape)
    for j in range(ids.shape[1]):
        r = np.nonzero(there[:, j])[0]
        d[r, ids[r, j]] = w[r, j] * (dw[r, j] - mean[r, 0])
    return d


def ref_sort(ids, experts, align):
    flat = ids.reshape(-1)
    offsets, counts = [0], []
    order = np.full(flat.size + experts * (align - 1), -1, np.int64)
    slots = np.full(flat.size, -1, np.int64)
    for e in range(experts):
        mine = np.nonzero(flat == e)[0]
        at = offsets[-1] + np.arange(mine.size)
        order[at] = mine
        slots[mine] = at
        counts.append(mine.size)
        offsets.append(offsets[-1] + -(-mine.size // align) * align)
    return np.array(offsets), np.array(counts), order, slots.reshape(ids.shape)


def sort_on_gpu(core, torch, ids, experts, align):
    n, k = ids.shape
    cap = core.sort_rows_capacity(n, k, experts, align)
    d = _up(torch, ids.astype(np.int32)) if ids.size else torch.empty(1, dtype=torch.int32).cuda()
    offsets = torch.full((experts + 1,), -7, dtype=torch.int64, device="cuda")
    counts = torch.full((experts,), -7, dtype=torch.int32, device="cuda")
    order = torch.full((max(cap, 1),), -7, dtype=torch.int32, device="cuda")
    slots = torch.full((max(n * k, 1),), -7, dtype=torch.int32, device="cuda")
    need = core.sort_rows_workspace(n, k, experts)
    room = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    core.sort_rows_device(0, d.data_ptr(), n, k, experts, align, offsets.data_ptr(),
                          counts.data_ptr(), order.data_ptr(), slots.data_ptr(), room.data_ptr(),
                          need, stream=_stream(torch))
    return offsets, counts, order[:cap], slots[:n * k].view(n, k)


# ---- route ---------------------------------------------------------------------

def _logits(rows, experts, kind, seed):
    r = np.random.default_rng(seed)
    x = (r.standard_normal((rows, experts)) * 3).astype(np.float32)
    if kind == "ties":
        x = np.round(x)
    elif kind == "masked":
        x[r.random(x.shape) < 0.6] = -np.inf
        x[::5] = -np.inf
        x[1::7, 0] = np.nan
        x[2::9] = np.nan
    elif kind == "lowest":
        x[r.random(x.shape) < 0.7] = np.finfo(np.float32).min
        x[::4] = np.finfo(np.float32).min
    return x


SIZES = [(1, 1, 1), (33, 2, 1), (1, 3, 3), (70, 4, 2), (129, 7, 7), (300, 8, 2), (257, 10, 3),
         (40, 16, 16), (65, 17, 4), (31, 32, 32), (100, 33, 8), (19, 64, 32), (77, 65, 8),
         (5, 128, 2), (67, 256, 8), (9, 300, 32), (3, 513, 6), (11, 1000, 8), (2, 1024, 32)]


@pytest.mark.parametrize("kind", ["plain", "ties", "masked", "lowest"])
@pytest.mark.parametrize("rows,experts,k", SIZES)
@pytest.mark.parametrize("norm", [0, 1])
def test_route_and_gradient(gpu, torch, rows, experts, k, norm, kind):
    core = gpu
    x = _logits(rows, experts, kind, rows * 1000 + experts)
    pad = 3 if experts % 2 else 0          # strided rows, and rows of exactly E
    ld = experts + pad
    dx = torch.full((rows, ld), np.nan, device="cuda")
    dx[:, :experts] = _up(torch, x)
    ids = torch.empty((rows, k), dtype=torch.int32, device="cuda")
    w = torch.empty((rows, k), device="cuda")
    core.route_device(0, dx.data_ptr(), rows, experts, ld, k, norm, ids.data_ptr(), w.data_ptr(),
                      stream=_stream(torch))
    rid, rw, rp = ref_route(x, k, norm)
    assert np.array_equal(ids.cpu().numpy(), rid)
    with np.errstate(invalid="ignore", over="ignore"):
        finite = x[np.isfinite(x) & (x > -1e30)]
    spread = float(finite.max() - finite.min()) if finite.size else 0.0
    tol = (spread + experts + 8) * 2 * U
    got = w.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - rw) <= tol * rw + 1e-38)

    dw = np.random.default_rng(1).standard_normal((rows, k)).astype(np.float32)
    dw[rid < 0] = np.nan                   # beside an id of -1: never read
    ddw = _up(torch, dw)
    d = torch.full((rows, ld), 7.0, device="cuda")
    core.route_grad_device(0, dx.data_ptr(), rows, experts, ld, k, norm, ids.data_ptr(),
                           w.data_ptr(), ddw.data_ptr(), d.data_ptr(), ld, stream=_stream(torch))
    ref = ref_route_grad(x, rid, rw, rp, dw, norm)
    got = d.cpu().numpy().astype(np.float64)
    assert np.all(got[:, experts:] == 7.0)
    # every factor (a weight, the mean over k terms) carries a weight's relative error
    big = np.nanmax(np.abs(dw)) if np.any(rid >= 0) else 0.0
    size = rp * big if norm else np.zeros_like(ref)
    for j in range(k):
        r = np.nonzero(rid[:, j] >= 0)[0]
        size[r, rid[r, j]] = 2 * rw[r, j] * big
    assert np.all(np.abs(got[:, :experts] - ref) <= (3 * tol + (k + 8) * 2 * U) * size + 1e-37)


@pytest.mark.parametrize("norm", [0, 1])
def test_route_gradient_against_differences(gpu, torch, norm):
    """d(sum dw . w) along each logit, by central differences of the 64-bit form."""
    core = gpu
    x = _logits(6, 9, "plain", 3)
    k, h = 3, 1e-6
    dw = np.random.default_rng(2).standard_normal((6, k))
    ids, w, _ = ref_route(x, k, norm)

    def f(z):
        m = z.max(1, keepdims=True)
        e = np.exp(z - m)
        s = e.sum(1, keepdims=True) if norm else np.take_along_axis(e, ids, 1).sum(1, keepdims=True)
        return ((np.take_along_axis(e, ids, 1) / s) * dw).sum(1)

    num = np.zeros(x.shape)
    for e in range(9):
        z = np.zeros(x.shape)
        z[:, e] = h
        num[:, e] = (f(x.astype(np.float64) + z) - f(x.astype(np.float64) - z)) / (2 * h)
    dx, di = _up(torch, x), _up(torch, ids.astype(np.int32))
    dwt, ddw = _up(torch, w.astype(np.float32)), _up(torch, dw.astype(np.float32))
    d = torch.empty((6, 9), device="cuda")
    core.route_grad_device(0, dx.data_ptr(), 6, 9, 9, k, norm, di.data_ptr(), dwt.data_ptr(),
                           ddw.data_ptr(), d.data_ptr(), 9, stream=_stream(torch))
    # differences: h^2 / 6 of a third derivative below 10, 2^-52 / h of rounding
    assert np.allclose(d.cpu().numpy(), num, rtol=0, atol=2e-6)


# ---- sort and gather -----------------------------------------------------------

@pytest.mark.parametrize("rows,k,experts,align", [
    (0, 1, 3, 4), (1, 1, 1, 1), (1, 2, 5, 4), (31, 1, 2, 1), (500, 1, 4, 4), (2048, 2, 1024, 4),
    (4096, 1, 7, 1), (4097, 1, 7, 16), (1365, 3, 9, 1), (30_011, 3, 64, 4), (100_003, 1, 8, 4),
    (9_001, 8, 256, 1), (1_100_000, 1, 5, 4), (70_000, 2, 1000, 3)])
@pytest.mark.parametrize("kind", ["even", "one", "bad"])
def test_sort(gpu, torch, rows, k, experts, align, kind):
    r = np.random.default_rng(rows + k)
    ids = r.integers(0, experts, (rows, k))
    if kind == "one":
        ids[:] = experts - 1
    if kind == "bad":
        ids[r.random(ids.shape) < 0.3] = -1
        ids[r.random(ids.shape) < 0.1] = experts
        ids[r.random(ids.shape) < 0.1] = -2 ** 31
    got = sort_on_gpu(gpu, torch, ids, experts, align)
    for a, b, what in zip(got, ref_sort(ids, experts, align), ("offsets", "counts", "order", "slots")):
        assert np.array_equal(a.cpu().numpy(), b), what


TYPES = ["float32", "bfloat16", "float16"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("source,target", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("rows,cols,k,experts,align,pad", [
    (1, 1, 1, 1, 1, 0), (37, 3, 2, 4, 4, 1), (500, 100, 1, 4, 4, 0), (130, 28, 3, 9, 4, 4),
    (65, 257, 2, 70, 1, 8), (2_000, 8, 1, 8, 4, 0), (5_000, 17, 2, 64, 4, 0), (10, 1_030, 8, 9, 1, 2)])
def test_gather(gpu, torch, rows, cols, k, experts, align, pad, source, target, dtype):
    core = gpu
    t = getattr(torch, dtype)
    r = np.random.default_rng(cols)
    ids = r.integers(-1, experts, (rows, k))
    offsets, counts, order, slots = sort_on_gpu(core, torch, ids, experts, align)
    cap = order.numel()
    x = torch.randn((rows, cols), device="cuda").to(t)
    x[0, 0] = float("nan")
    full = torch.zeros((rows, cols + pad) if source else (cols, rows + pad), dtype=t, device="cuda")
    (full if source else full.t())[:rows, :cols] = x
    out = torch.full((cap, cols + pad) if target else (cols, cap + pad), 7.0, dtype=t, device="cuda")
    core.gather_rows_device(0, TYPES.index(dtype), full.data_ptr(), rows, cols, full.shape[1],
                            source, k, experts, offsets.data_ptr(), order.data_ptr(),
                            slots.data_ptr(), cap, out.data_ptr(), out.shape[1], target,
                            stream=_stream(torch))
    rows_of = torch.clamp(order.long(), min=0) // k
    want = torch.where((order >= 0)[:, None], x[rows_of], torch.zeros((), dtype=t, device="cuda"))
    got = (out if target else out.t())[:cap, :cols]
    wide = torch.int32 if t == torch.float32 else torch.int16
    assert torch.equal(got.contiguous().view(wide), want.view(wide))
    assert torch.all((out[:, cols:] if target else out[:, cap:]) == 7.0)


@pytest.mark.parametrize("rows,cols,k,experts,align,kind", [
    (200_001, 96, 2, 64, 4, "even"), (180_000, 100, 3, 7, 1, "uneven"), (17_000, 1_000, 2, 255, 4, "uneven"),
    (17_000, 1_000, 2, 256, 1, "uneven"), (170_000, 100, 2, 40, 4, "one"), (170_000, 100, 8, 200, 4, "bad")])
def test_gather_of_more_than_the_cache(gpu, torch, rows, cols, k, experts, align, kind):
    """Large row-major inputs with several choices, laid out feature-major: tiles run in
    the order of their place in the segments."""
    core = gpu
    r = np.random.default_rng(rows + experts)
    u = r.random((rows, k))
    ids = (u ** (3 if kind == "uneven" else 1) * experts).astype(np.int64)
    if kind == "one":
        ids[:] = 3
        ids[::1000, 0] = 39
    if kind == "bad":
        ids[r.random(ids.shape) < 0.4] = -1
    offsets, counts, order, slots = sort_on_gpu(core, torch, ids, experts, align)
    cap = order.numel()
    x = torch.randn((rows, cols), device="cuda")
    out = torch.full((cols, cap), 7.0, device="cuda")
    core.gather_rows_device(0, core.F32, x.data_ptr(), rows, cols, cols, 1, k, experts,
                            offsets.data_ptr(), order.data_ptr(), slots.data_ptr(), cap,
                            out.data_ptr(), cap, 0, stream=_stream(torch))
    want = torch.where((order >= 0)[:, None], x[torch.clamp(order.long(), min=0) // k], 0.0)
    assert torch.equal(out, want.t())


# ---- combine -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,k,experts,align,pad,kind", [
    (1, 1, 1, 1, 1, 0, "plain"), (37, 3, 2, 4, 4, 1, "bad"), (501, 10, 2, 64, 4, 0, "plain"),
    (130, 28, 8, 9, 4, 4, "bad"), (66, 257, 3, 70, 1, 7, "bad"), (40, 1_032, 8, 9, 1, 0, "plain"),
    (3_001, 1, 1, 8, 4, 0, "ones"), (900, 16, 32, 40, 1, 0, "ones"), (64, 40, 2, 5, 1, 8, "none")])
def test_combine_and_gradient(gpu, torch, rows, cols, k, experts, align, pad, kind, dtype):
    core = gpu
    t = getattr(torch, dtype)
    half = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]
    r = np.random.default_rng(rows + cols)
    ids = r.integers(0, experts, (rows, k))
    if kind == "bad":
        ids[r.random(ids.shape) < 0.4] = -1
        ids[:3] = -1
    if kind == "none":
        ids[:] = -1
    offsets, counts, order, slots = sort_on_gpu(core, torch, ids, experts, align)
    cap, ld = order.numel(), cols + pad
    y = torch.randn((cap, ld), device="cuda").to(t)
    y[order < 0] = float("nan")            # rows of no entry are never read
    w = torch.randn((rows, k), device="cuda")
    w[slots < 0] = float("nan")            # nor is the weight of an entry left out
    out = torch.full((rows, ld), 7.0, dtype=t, device="cuda")
    wp = 0 if kind == "ones" else w.data_ptr()
    code = TYPES.index(dtype)
    core.combine_rows_device(0, code, y.data_ptr(), cap, cols, ld, slots.data_ptr(), wp, rows, k,
                             out.data_ptr(), ld, stream=_stream(torch))
    there = (slots >= 0).cpu().numpy()
    at = slots.clamp(min=0).long().cpu().numpy()
    yf = y.double().cpu().numpy()[:, :cols]
    picked = np.where(there[:, :, None], yf[at], 0.0)
    wf = np.where(there, 1.0 if kind == "ones" else w.double().cpu().numpy(), 0.0)
    terms = picked * wf[:, :, None]
    err = np.abs(out[:, :cols].double().cpu().numpy() - terms.sum(1))
    assert np.all(err <= (k + 2) * U * np.abs(terms).sum(1) + half * np.abs(terms.sum(1)) + 3e-8)
    assert torch.all(out[:, cols:] == 7.0)

    dout = torch.randn((rows, ld), device="cuda").to(t)
    dy = torch.full((cap, ld), 7.0, dtype=t, device="cuda")
    dw = torch.full((rows, k), 7.0, device="cuda")
    core.combine_rows_grad_device(0, code, y.data_ptr(), cap, cols, ld, order.data_ptr(),
                                  slots.data_ptr(), wp, rows, k, dout.data_ptr(), ld,
                                  dy.data_ptr(), ld, dw.data_ptr(), stream=_stream(torch))
    df = dout.double().cpu().numpy()[:, :cols]
    prod = picked * df[:, None, :]
    err = np.abs(dw.double().cpu().numpy() - prod.sum(2))
    assert np.all(err <= (cols + 2) * U * np.abs(prod).sum(2))
    want = torch.zeros((cap, cols), dtype=t, device="cuda")
    wt = torch.ones_like(w) if kind == "ones" else w
    want[slots[slots >= 0].long()] = (wt[:, :, None] * dout.float()[:, None, :cols]).to(t)[slots >= 0]
    assert torch.equal(dy[:, :cols], want)
    assert torch.all(dy[:, cols:] == 7.0)
    if kind == "plain":                    # without dweights the rest is the same
        again = torch.full((cap, ld), 7.0, dtype=t, device="cuda")
        core.combine_rows_grad_device(0, code, y.data_ptr(), cap, cols, ld, order.data_ptr(),
                                      slots.data_ptr(), wp, rows, k, dout.data_ptr(), ld,
                                      again.data_ptr(), ld, 0, stream=_stream(torch))
        assert torch.equal(again, dy)


def test_rows_beyond_32_bit_offsets(gpu, torch):
    """A gather and a combination whose last rows lie past 2^31 values."""
    core = gpu
    rows, cols = 1_100_000, 2_000
    ids = np.full((rows, 1), -1)
    ids[[0, rows - 1]] = 0
    offsets, counts, order, slots = sort_on_gpu(core, torch, ids, 1, 1)
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[0], x[rows - 1] = 1.0, 2.0
    out = torch.empty((2, cols), dtype=torch.bfloat16, device="cuda")
    order2 = order[:2].flip(0).contiguous()
    slots2 = torch.full((rows, 1), -1, dtype=torch.int32, device="cuda")
    slots2[rows - 1], slots2[0] = 0, 1
    # a plan of the caller's own: as many slots as entries, the first two in use
    full = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    full[:2] = order2
    big = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    core.gather_rows_device(0, core.BF16, x.data_ptr(), rows, cols, cols, 1, 1, 1,
                            offsets.data_ptr(), full.data_ptr(), slots2.data_ptr(), rows,
                            big.data_ptr(), cols, 1, stream=_stream(torch))
    assert torch.all(big[0] == 2.0) and torch.all(big[1] == 1.0) and torch.all(big[2:] == 0)
    big[rows - 1] = 5.0
    slots2[0] = rows - 1
    core.combine_rows_device(0, core.BF16, big.data_ptr(), rows, cols, cols, slots2.data_ptr(), 0,
                             rows, 1, x.data_ptr(), cols, stream=_stream(torch))
    out = x[[0, 1, rows - 1]].float()
    assert torch.all(out[0] == 5.0) and torch.all(out[1] == 0.0) and torch.all(out[2] == 2.0)


def test_calls_follow_their_stream(gpu, torch):
    """Work queued on another stream is seen by a call on that stream, and the calls
    give the same bits every time."""
    core = gpu
    side = torch.cuda.Stream()
    rows, experts, k = 200_000, 64, 2
    host = torch.randn((rows, experts), generator=torch.Generator().manual_seed(7)).pin_memory()
    results = []
    for _ in range(3):
        with torch.cuda.stream(side):
            x = torch.zeros((rows, experts), device="cuda")
            for _ in range(20):
                x += 0.0
            x.copy_(host, non_blocking=True)
            ids = torch.empty((rows, k), dtype=torch.int32, device="cuda")
            w = torch.empty((rows, k), device="cuda")
            before = core.kernel_launches()
            core.route_device(0, x.data_ptr(), rows, experts, experts, k, core.ROUTE_ALL,
                              ids.data_ptr(), w.data_ptr(), stream=side.cuda_stream)
            assert core.kernel_launches() == before + 1
        side.synchronize()
        results.append((ids, w))
    want = host.sort(dim=1, descending=True, stable=True).indices[:, :k].int()
    assert torch.equal(results[0][0].cpu(), want)
    for ids, w in results[1:]:
        assert torch.equal(ids, results[0][0]) and torch.equal(w, results[0][1])
