"""Infinities, NaN and the largest floats in the softmax head: every form of it (narrow,
few rows, tensor cores) gives the definition's values.

Tolerances: finite values as in test_head_gpu.py, by its own reference and bounds."""

import pytest

import test_head_gpu as H

pytestmark = pytest.mark.gpu

INF = float("inf")
LOWEST = -3.4028234663852886e38


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


# rows x cols x classes of each form: narrow, few rows, tensor cores (one and several tiles)
FORMS = [(40, 8, 20), (3, 72, 700), (6, 8, 700), (17, 8, 700), (300, 72, 700), (300, 136, 300)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols,classes", FORMS)
def test_classes_switched_off(gpu, torch, dtype, rows, cols, classes):
    """A constant column is a bias; classes whose bias is -inf, or the lowest float32, have
    no probability, and the others' values are as if those did not exist."""
    h, w, y, dloss = H._inputs(torch, rows, cols, classes, dtype, 0, rows + cols, 0.1)
    h[:, 0] = 1.0
    on = torch.ones(classes, dtype=torch.bool, device="cuda")
    on[3::5] = False
    y = torch.where(on[y.long().clamp(0, classes - 1)], y, 0)
    # the same labels among the classes that are on
    number = (on.cumsum(0) - 1).int()
    inside = (y >= 0) & (y < classes)
    y_on = torch.where(inside, number[y.long().clamp(0, classes - 1)], -1)
    ref = H._reference(torch, h, w[on], y_on, dloss, cols)
    for off in (-INF, LOWEST if dtype == "float32" else -3.3895313892515355e38):
        w[~on, 0] = off
        loss, lse, dh, dw = H._run(gpu, torch, h, w, y, dloss, cols)
        H._check(torch, (loss, lse), ref, cols, f"{off}")
        # dh's column 0 holds 0 x off, NaN for -inf
        v, b = ref["dh"]
        assert torch.all((dh[:, 1:].double() - v[:, 1:]).abs() <= b[:, 1:] + 1e-37)
        if off != -INF:
            assert torch.all((dh[:, 0].double() - v[:, 0]).abs() <= b[:, 0] + 1e-37)
        v, b = ref["dw"]
        assert torch.all((dw[on].double() - v).abs() <= b + 1e-37)
        assert torch.all(dw[~on] == 0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols,classes", FORMS)
def test_infinite_and_nan_logits(gpu, torch, dtype, rows, cols, classes):
    """Every class at -inf: lse -inf.  An infinite class: lse inf.  NaN in one class, or in
    one row, stays where the definition has it."""
    t = getattr(torch, dtype)
    h = torch.randn((rows, cols), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(t)
    h[:, 0] = 0.37                          # three terms, of both signs, as a float32
    w = torch.zeros((classes, cols), device="cuda", dtype=t)
    y = torch.zeros(rows, dtype=torch.int32, device="cuda")
    w[:, 0] = -INF
    assert torch.all(H._run(gpu, torch, h, w, y, None, cols)[1] == -INF)
    w[:, 0] = 0
    w[classes - 1, 0] = INF
    assert torch.all(H._run(gpu, torch, h, w, y, None, cols)[1] == INF)
    w[classes - 1, 0] = float("nan")
    assert torch.isnan(H._run(gpu, torch, h, w, y, None, cols)[1]).all()
    w[classes - 1, 0] = 0
    w[:, 1] = -1.0                          # a row of h at +inf beside it: all classes -inf
    h[0, 1] = INF
    h[1, 1] = float("nan")
    loss, lse = H._run(gpu, torch, h, w, y, None, cols)
    assert lse[0] == -INF and torch.isnan(lse[1])
    assert torch.isfinite(lse[2:]).all() and torch.isfinite(loss[2:]).all()


@pytest.mark.parametrize("rows,cols,classes", FORMS)
def test_largest_floats(gpu, torch, rows, cols, classes):
    """float32 values above bfloat16's largest one are finite values like any other.  A
    gradient's sum is compared where its terms stay within float32."""
    h, w, y, dloss = H._inputs(torch, rows, cols, classes, "float32", 0, 3)
    big = 3.4e38
    h[:, 0] = 0
    h[0, 0] = 2.0 ** -126
    w[::7, 0] = big
    h[rows - 1, 2] = -big
    w[:, 2] = 2.0 ** -127
    got = H._run(gpu, torch, h, w, y, dloss, cols)
    ref = H._reference(torch, h, w, y, dloss, cols)
    H._check(torch, got[:2], ref, cols, "largest")
    p = torch.softmax(h.double() @ w.double().t(), 1)
    p.scatter_add_(1, y.long()[:, None], torch.full((rows, 1), -1.0, dtype=p.dtype, device="cuda"))
    g = (dloss.double()[:, None] * p).abs()
    for x, name, size in ((got[2], "dh", g @ w.double().abs()), (got[3], "dw", g.t() @ h.double().abs())):
        v, b = ref[name]
        fits = size < 1e38
        assert fits.any()
        assert torch.all((x.double() - v).abs()[fits] <= b[fits] + 1e-37)


def test_all_nan_takes_no_longer(gpu, torch):
    """float32 values that are not finite are looked at again; with nothing else among many
    rows and classes every wait still ends in time."""
    rows, cols, classes = 2_048, 512, 8_192
    h, w, y, dloss = H._inputs(torch, rows, cols, classes, "float32", 0, 3)
    for value in (float("nan"), INF, LOWEST):
        h[:] = value
        loss, lse, dh, dw = H._run(gpu, torch, h, w, y, dloss, cols)
        assert not torch.isfinite(loss).any()
