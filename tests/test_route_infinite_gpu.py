"""Route with infinite logits, and rows laid out without padding for every small number of
models (their rows pass through shared memory in a form of their own)."""

import numpy as np
import pytest

import test_mixture_gpu as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


def _route(core, torch, x, k, norm):
    rows, experts = x.shape
    ids = torch.full((rows, k), 7, dtype=torch.int32, device="cuda")
    w = torch.full((rows, k), 7.0, device="cuda")
    core.route_device(0, x.data_ptr(), rows, experts, experts, k, norm, ids.data_ptr(), w.data_ptr(),
                      stream=M._stream(torch))
    return ids, w


@pytest.mark.parametrize("experts,k", [(3, 2), (3, 3), (16, 2), (16, 5), (20, 4), (40, 3), (100, 4), (600, 32)])
@pytest.mark.parametrize("norm", [0, 1])
def test_no_choice_has_no_weight(gpu, torch, experts, k, norm):
    """A row with one infinite logit and nothing else to choose: the softmax at the choice
    is inf / inf, but a choice that does not exist has weight 0."""
    x = torch.full((70, experts), -float("inf"), device="cuda")
    x[:, experts // 2] = float("inf")
    ids, w = _route(gpu, torch, x, k, norm)
    assert torch.all(ids[:, 0] == experts // 2) and torch.all(ids[:, 1:] == -1)
    assert torch.isnan(w[:, 0]).all() and torch.all(w[:, 1:] == 0)


@pytest.mark.parametrize("kind", ["plain", "masked"])
@pytest.mark.parametrize("experts", list(range(1, 18)))
@pytest.mark.parametrize("norm", [0, 1])
def test_adjacent_rows(gpu, torch, experts, norm, kind):
    """More than a block's rows of exactly `experts` logits each, and the rest of a tile."""
    core = gpu
    rows = 32 * 4 * 3 + 45
    for k in {1, min(2, experts), min(3, experts), experts}:
        x = M._logits(rows, experts, kind, experts)
        dx = M._up(torch, x)
        ids, w = _route(core, torch, dx, k, norm)
        rid, rw, rp = M.ref_route(x, k, norm)
        assert np.array_equal(ids.cpu().numpy(), rid)
        finite = x[np.isfinite(x)]
        tol = (float(finite.max() - finite.min()) + experts + 8) * 2 * M.U
        assert np.all(np.abs(w.cpu().numpy() - rw) <= tol * rw + 1e-38)
        dw = np.random.default_rng(k).standard_normal((rows, k)).astype(np.float32)
        d = torch.full((rows, experts), 7.0, device="cuda")
        ddw = M._up(torch, dw)
        core.route_grad_device(0, dx.data_ptr(), rows, experts, experts, k, norm, ids.data_ptr(),
                               w.data_ptr(), ddw.data_ptr(), d.data_ptr(), experts,
                               stream=M._stream(torch))
        ref = M.ref_route_grad(x, rid, rw, rp, dw, norm)
        size = rp * np.abs(dw).max() if norm else np.zeros_like(ref)
        for j in range(k):
            r = np.nonzero(rid[:, j] >= 0)[0]
            size[r, rid[r, j]] = 2 * rw[r, j] * np.abs(dw).max()
        err = np.abs(d.cpu().numpy() - ref)
        assert np.all(err <= (3 * tol + (k + 8) * 2 * M.U) * size + 1e-37)
