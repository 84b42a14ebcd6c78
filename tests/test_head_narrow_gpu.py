"""A narrow softmax head over more rows than its blocks take at once: a row's values stay
its own, whatever the rows before it held."""

import pytest

import test_head_gpu as H

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("cols,classes", [(10, 10), (3, 4), (17, 30), (62, 32)])
@pytest.mark.parametrize("bad", ["h", "dloss", "infinite h"])
def test_a_bad_row_spoils_no_other(gpu, torch, dtype, cols, classes, bad):
    """A labelled row with a value that is not finite, early among more rows than a narrow
    head takes at once: dh of all other rows is as without it."""
    rows = 200_000
    h, w, y, dloss = H._inputs(torch, rows, cols, classes, dtype, 0, 17, 0.1)
    at = torch.tensor([0, 37, 4_000], device="cuda")
    y[at] = 1
    want = H._run(gpu, torch, h, w, y, dloss, cols)
    spoiled, weight = h.clone(), dloss.clone()
    if bad == "dloss":
        weight[at] = float("nan")
    else:
        spoiled[at] = float("nan") if bad == "h" else INF
    got = H._run(gpu, torch, spoiled, w, y, weight, cols)
    others = torch.ones(rows, dtype=torch.bool, device="cuda")
    others[at] = False
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a[others], b[others])
    assert not torch.isfinite(got[2][at]).any()
