"""The softmax head on the GPU against the formulas in 64 bits.

Tolerances, elementwise, with u = 2^-23 (one unit of float32: the tensor core's sums
are truncated).  A product of D terms: every term's error (0 for bfloat16; at most 5 x
2^-24 for the three-term split of float32) and one truncation for every 16 terms and
plane product (at most 6 D / 16 of them, and the alignment of 16 terms to their
largest): within (D + 16) u of sum |h||w|; call that e, its row maximum E.
lse: E, its own sums over the classes in parts of 32 and 128 (200 u), the exponentials'
arguments (|l - lse| u) and the result's own rounding (|lse| u).
g = dloss (p - [v = y]): p carries the relative error e + E_lse + (|l - lse| + 8) u, g one
rounding to bfloat16 (2^-8) or three of them (2^-22).  dh, dw: the errors of g times
|w| or |h| summed, (terms + 16) u of the magnitudes, and the result's rounding."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -23


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


def _inputs(torch, rows, cols, classes, dtype, pad, seed, ignored=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = getattr(torch, dtype)
    h = torch.randn((rows, cols + pad), device="cuda", generator=g).to(t)
    w = (torch.randn((classes, cols + pad), device="cuda", generator=g) * 3 / cols ** 0.5).to(t)
    y = torch.randint(0, classes, (rows,), device="cuda", generator=g, dtype=torch.int32)
    if ignored:
        off = torch.rand(rows, device="cuda", generator=g) < ignored
        y[off] = torch.tensor([-1, classes, -2 ** 31], device="cuda", dtype=torch.int32)[
            torch.randint(0, 3, (int(off.sum()),), device="cuda", generator=g)]
    dloss = torch.randn(rows, device="cuda", generator=g)
    return h, w, y, dloss


def _run(core, torch, h, w, y, dloss, cols, want="both", strided=False, offset=0):
    """loss, lse, dh, dw on the GPU; outputs have the inputs' strides."""
    rows, classes = h.shape[0], w.shape[0]
    code = core.F32 if h.dtype == torch.float32 else core.BF16
    loss = torch.full((rows,), 7.0, device="cuda")
    lse = torch.full((rows,), 7.0, device="cuda")
    need = core.head_workspace(code, rows, cols, classes, grad=dloss is not None, strided=strided)
    room = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    at = (room.data_ptr() + 255) // 256 * 256
    stream = torch.cuda.current_stream().cuda_stream
    core.head_loss_device(0, code, h.data_ptr(), rows, cols, h.stride(0), w.data_ptr(), classes,
                          w.stride(0), y.data_ptr(), loss.data_ptr(), lse.data_ptr(), at, need,
                          stream=stream)
    core.head_check_device(0, at)
    if dloss is None:
        return loss, lse
    dh = torch.full((rows, h.shape[1]), 7.0, dtype=h.dtype, device="cuda")
    dw = torch.full((classes, w.shape[1]), 7.0, dtype=w.dtype, device="cuda")
    core.head_grad_device(0, code, h.data_ptr(), rows, cols, h.stride(0), w.data_ptr(), classes,
                          w.stride(0), y.data_ptr(), lse.data_ptr(), dloss.data_ptr(),
                          dh.data_ptr() if want != "dw" else 0, dh.stride(0),
                          dw.data_ptr() if want != "dh" else 0, dw.stride(0), at, need,
                          stream=stream)
    core.head_check_device(0, at)
    return loss, lse, dh, dw


def _reference(torch, h, w, y, dloss, cols):
    """Values and bounds in 64 bits: {name: (value, bound)}."""
    rows, classes = h.shape[0], w.shape[0]
    known = (y >= 0) & (y < classes)
    hd, wd = h[:, :cols].double(), w[:, :cols].double()
    hd = torch.where(known[:, None], hd, torch.nan_to_num(hd))
    l = hd @ wd.t()
    e = (cols + 16) * U * (hd.abs() @ wd.abs().t())
    lse = torch.logsumexp(l, 1)
    E = e.amax(1) + (200 + lse.abs() + (l.amax(1) - lse).abs()) * U
    at = y.long().clamp(0, classes - 1)[:, None]
    loss = torch.where(known, lse - l.gather(1, at)[:, 0], 0.0)
    loss_b = torch.where(known, E + e.gather(1, at)[:, 0] + loss.abs() * U, 0.0)
    out = {"lse": (lse, E), "loss": (loss, loss_b)}
    if dloss is not None:
        half = 2.0 ** -8 if h.dtype == torch.bfloat16 else 2.0 ** -22
        last = 2.0 ** -8 if h.dtype == torch.bfloat16 else U
        p = torch.exp(l - lse[:, None])
        up = torch.where(known, dloss.double(), 0.0)[:, None]
        onehot = torch.zeros_like(p).scatter_(1, at, 1.0)
        g = up * (p - onehot)
        gb = up.abs() * p * (e + E[:, None] + ((l - lse[:, None]).abs() + 8) * U)
        gb += g.abs() * half
        hz = torch.where(known[:, None], hd, 0.0)
        dh, dw = g @ wd, g.t() @ hz
        out["dh"] = (dh, gb @ wd.abs() + (classes + 16) * U * (g.abs() @ wd.abs()) + dh.abs() * last)
        out["dw"] = (dw, gb.t() @ hz.abs() + (rows + 16) * U * (g.abs().t() @ hz.abs()) + dw.abs() * last)
    return out


def _check(torch, got, ref, cols, what):
    for name, x in zip(("loss", "lse", "dh", "dw"), got):
        v, b = ref[name]
        x = x[:, :cols] if x.dim() == 2 else x
        err = (x.double() - v).abs()
        worst = float((err / (b + 1e-37)).max()) if err.numel() else 0.0
        assert torch.all(err <= b + 1e-37), f"{what}: {name} is {worst:.3g} of its bound"
        assert torch.isfinite(x).all()


SIZES = [(1, 8, 10), (1, 1024, 5000), (3, 1, 2), (5, 7, 1), (1, 16, 100_000), (128, 64, 256),
         (129, 65, 257), (257, 100, 1000), (300, 72, 513), (70, 200, 40_000), (2000, 16, 33),
         (4100, 264, 700), (513, 300, 255), (33, 1030, 130), (2, 130, 64)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols,classes", SIZES)
def test_head(gpu, torch, rows, cols, classes, dtype):
    h, w, y, dloss = _inputs(torch, rows, cols, classes, dtype, 0, rows + cols, 0.2)
    got = _run(gpu, torch, h, w, y, dloss, cols)
    ref = _reference(torch, h, w, y, dloss, cols)
    _check(torch, got, ref, cols, "head")
    # the same bits again, and without the gradient's part of the workspace
    again = _run(gpu, torch, h, w, y, dloss, cols)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    alone = _run(gpu, torch, h, w, y, None, cols)
    assert all(torch.equal(a, b) for a, b in zip(got, alone))


# a handful of rows (a kernel of its own up to 8 or 16 of them), one more than that, and
# narrow heads (at most 64 columns and 32 classes)
FEW = [(1, 1024, 3001), (2, 65, 700), (2, 64, 33), (3, 257, 1000), (4, 512, 999), (5, 72, 20_000),
       (7, 1000, 2049), (8, 2048, 130), (8, 9, 4000), (9, 72, 1500), (11, 100, 350), (16, 1030, 640),
       (16, 64, 257), (17, 128, 600), (1, 65, 1), (4, 3000, 50), (1, 20_000, 40)]
NARROW = [(1, 1, 1), (31, 64, 32), (33, 63, 31), (1000, 10, 10), (129, 16, 4), (300, 17, 5),
          (97, 5, 17), (4000, 32, 12), (200_001, 3, 9), (65, 40, 13), (64, 48, 16)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols,classes", FEW + NARROW)
def test_small_heads(gpu, torch, rows, cols, classes, dtype):
    for pad in (0, 8, 3):
        h, w, y, dloss = _inputs(torch, rows, cols, classes, dtype, pad, rows + cols, 0.2)
        off = (y < 0) | (y >= classes)
        h[off] = float("nan")
        dloss[off] = float("nan")
        loss, lse, dh, dw = _run(gpu, torch, h, w, y, dloss, cols, strided=True)
        ref = _reference(torch, h, w, y, dloss, cols)
        assert torch.all(loss[off] == 0) and torch.all(dh[off][:, :cols] == 0)
        keep = ~off
        _check(torch, (loss[keep], lse[keep], dh[keep], dw),
               {k: (v[keep], b[keep]) if k != "dw" else (v, b) for k, (v, b) in ref.items()},
               cols, f"pad {pad}")
        assert torch.all(dh[:, cols:] == 7.0) and torch.all(dw[:, cols:] == 7.0)
        alone = _run(gpu, torch, h, w, y, dloss, cols, want="dh", strided=True)
        assert torch.equal(alone[2], dh) and torch.all(alone[3] == 7.0)
        alone = _run(gpu, torch, h, w, y, dloss, cols, want="dw", strided=True)
        assert torch.equal(alone[3], dw) and torch.all(alone[2] == 7.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("want", ["dh", "dw"])
def test_one_gradient(gpu, torch, dtype, want):
    rows, cols, classes = 200, 136, 3000
    h, w, y, dloss = _inputs(torch, rows, cols, classes, dtype, 0, 3, 0.1)
    got = _run(gpu, torch, h, w, y, dloss, cols, want=want)
    ref = _reference(torch, h, w, y, dloss, cols)
    keep = 2 if want == "dh" else 3
    v, b = ref[want]
    assert torch.all((got[keep].double() - v).abs() <= b + 1e-37)
    assert torch.all(got[5 - keep] == 7.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("pad", [1, 4, 8])
def test_strides(gpu, torch, dtype, pad):
    """Rows off 16-byte boundaries are copied, others read in place; what lies between
    rows is neither read nor written."""
    rows, cols, classes = 150, 72, 600
    h, w, y, dloss = _inputs(torch, rows, cols, classes, dtype, pad, 5, 0.1)
    h[:, cols:] = float("nan")
    w[:, cols:] = float("nan")
    got = _run(gpu, torch, h, w, y, dloss, cols, strided=True)
    _check(torch, got, _reference(torch, h, w, y, dloss, cols), cols, "strided")
    assert torch.all(got[2][:, cols:] == 7.0) and torch.all(got[3][:, cols:] == 7.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rows_without_label_add_nothing(gpu, torch, dtype):
    rows, cols, classes = 140, 64, 300
    h, w, y, dloss = _inputs(torch, rows, cols, classes, dtype, 0, 9, 0.3)
    off = (y < 0) | (y >= classes)
    h[off] = float("nan")
    dloss[off] = float("nan")
    loss, lse, dh, dw = _run(gpu, torch, h, w, y, dloss, cols)
    ref = _reference(torch, h, w, y, dloss, cols)
    assert torch.all(loss[off] == 0) and torch.all(dh[off] == 0) and torch.isnan(lse[off]).all()
    keep = ~off
    _check(torch, (loss[keep], lse[keep], dh[keep], dw),
           {k: (v[keep], b[keep]) if k != "dw" else (v, b) for k, (v, b) in ref.items()}, cols, "masked")
    y[:] = -1                                # no row has a label
    _, _, dh, dw = _run(gpu, torch, h, w, y, dloss, cols)
    assert torch.all(dh == 0) and torch.all(dw == 0)


def test_infinite_logits(gpu, torch):
    """Classes of minus infinity have no probability; a row of nothing else has lse
    -inf; NaN stays NaN."""
    rows, cols, classes = 6, 8, 700
    h = torch.ones((rows, cols), device="cuda", dtype=torch.bfloat16)
    w = torch.zeros((classes, cols), device="cuda", dtype=torch.bfloat16)
    w[5:, 0] = -float("inf")
    y = torch.zeros(rows, dtype=torch.int32, device="cuda")
    loss, lse = _run(gpu, torch, h, w, y, None, cols)
    assert torch.allclose(lse, torch.full_like(lse, np.log(5.0)), atol=1e-6)
    assert torch.allclose(loss, lse)
    w[:, 0] = -float("inf")
    loss, lse = _run(gpu, torch, h, w, y, None, cols)
    assert torch.all(lse == -float("inf"))
    w[:] = 0
    w[400, 0] = float("nan")
    _, lse = _run(gpu, torch, h, w, y, None, cols)
    assert torch.isnan(lse).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_several_pieces(gpu, torch, dtype):
    """More g than one piece of the classes holds: dh is summed over the pieces."""
    rows, cols, classes = 70_001, 24, 4_100
    h, w, y, dloss = _inputs(torch, rows, cols, classes, dtype, 0, 11, 0.1)
    got = _run(gpu, torch, h, w, y, dloss, cols)
    _check(torch, got, _reference(torch, h, w, y, dloss, cols), cols, "pieces")


def test_weights_beyond_32_bit_offsets(gpu, torch):
    rows, cols, classes = 2, 1024, 2_200_000
    h = torch.ones((rows, cols), device="cuda", dtype=torch.bfloat16)
    w = torch.zeros((classes, cols), device="cuda", dtype=torch.bfloat16)
    w[classes - 1, :8] = 1.0
    y = torch.tensor([classes - 1, 0], dtype=torch.int32, device="cuda")
    dloss = torch.ones(rows, device="cuda")
    loss, lse, dh, dw = _run(gpu, torch, h, w, y, dloss, cols)
    want = np.log(classes - 1 + np.exp(8.0))
    assert np.allclose(lse.cpu().numpy(), want, rtol=1e-5)
    assert np.allclose(loss.cpu().numpy(), [want - 8.0, want], rtol=1e-5)
    p = np.exp(8.0 - want)
    assert np.allclose(dw[classes - 1].float().cpu().numpy(), 2 * p - 1, rtol=2.0 ** -7)
    assert np.allclose(dh[0, :8].float().cpu().numpy(), p - 1, rtol=2.0 ** -7)


def test_gradient_against_differences(gpu, torch):
    """The gradient along random directions, against central differences of the 64-bit
    loss; float32 inputs."""
    rows, cols, classes = 9, 12, 40
    h, w, y, dloss = _inputs(torch, rows, cols, classes, "float32", 0, 21)
    _, _, dh, dw = _run(gpu, torch, h, w, y, dloss, cols)

    def f(a, b):
        l = a @ b.t()
        return (dloss.double() * (torch.logsumexp(l, 1) - l.gather(1, y.long()[:, None])[:, 0])).sum()

    step = 1e-5
    g = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(8):
        a = torch.randn(h.shape, device="cuda", generator=g, dtype=torch.float64)
        b = torch.randn(w.shape, device="cuda", generator=g, dtype=torch.float64)
        num = (f(h.double() + step * a, w.double() + step * b)
               - f(h.double() - step * a, w.double() - step * b)) / (2 * step)
        ana = (dh.double() * a).sum() + (dw.double() * b).sum()
        # step^2 / 6 of the third derivative along the direction: (|a||w| + |h||b|)^3
        # stays below 1e5 here; float32 gradients: 1e-6 of the sums' magnitudes
        size = (dh.double() * a).abs().sum() + (dw.double() * b).abs().sum()
        assert abs(num - ana) <= 1e-10 * 1e5 + 1e-6 * size


def test_calls_follow_their_stream(gpu, torch):
    core = gpu
    rows, cols, classes = 64, 128, 5000
    h, w, y, dloss = _inputs(torch, rows, cols, classes, "bfloat16", 0, 31)
    want = _run(core, torch, h, w, y, dloss, cols)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    before = core.kernel_launches()
    with torch.cuda.stream(side):
        h2 = torch.zeros_like(h)
        for _ in range(50):
            h2 += 0
        h2.copy_(h)
        got = _run(core, torch, h2, w, y, dloss, cols)
    assert core.kernel_launches() > before
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_no_rows(gpu, torch):
    core = gpu
    dw = torch.full((5, 9), 7.0, device="cuda")
    core.head_grad_device(0, core.F32, 0, 0, 8, 8, 0, 5, 8, 0, 0, 0, 0, 8, dw.data_ptr(), 9, 0, 0,
                          stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.all(dw[:, :8] == 0) and torch.all(dw[:, 8] == 7.0)


def test_wait_runs_out_and_recovers(gpu, torch, monkeypatch):
    """With the test hook no copy is issued: every wait ends after its limit, the check
    reports it, and the next call is right again."""
    core = gpu
    rows, cols, classes = 300, 64, 2000
    h, w, y, dloss = _inputs(torch, rows, cols, classes, "bfloat16", 0, 41)
    want = _run(core, torch, h, w, y, dloss, cols)
    monkeypatch.setenv("MACBOOST_WAIT_LIMIT_US", "3000")
    monkeypatch.setenv("MACBOOST_TEST_STALL_TILES", "1")
    with pytest.raises(core.MacBoostError, match="gave up waiting"):
        _run(core, torch, h, w, y, dloss, cols)
    monkeypatch.delenv("MACBOOST_TEST_STALL_TILES")
    monkeypatch.delenv("MACBOOST_WAIT_LIMIT_US")
    got = _run(core, torch, h, w, y, dloss, cols)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
