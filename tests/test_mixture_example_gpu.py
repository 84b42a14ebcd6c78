"""The mixture example: its step on the GPU against the same forests scored one by one
from host memory and the formulas in 64 bits.

Tolerances: the margins are bit-exact, the weights within 1e-6 of themselves (two
exponentials of differences below 8 and a division), so the combination of margins below
1 is within 2e-6, the loss of ten classes within 1e-5, and every gradient (a mean over
rows of values below 1) within 1e-5 of the largest of its kind."""

import sys

import numpy as np
import pytest

from conftest import ROOT
from macboost_b200 import synth

pytestmark = pytest.mark.gpu


def test_mixture_step(gpu):
    core = gpu
    torch = pytest.importorskip("torch")
    sys.path.insert(0, str(ROOT / "examples"))
    try:
        import mixture
    finally:
        sys.path.pop(0)
    rows = 4_099
    gate, experts = mixture.make_forests(trees=30)
    X = np.ascontiguousarray(synth.make_data("cfg4", rows=rows, layout="row", seed=3))
    r = np.random.default_rng(4)
    y = r.integers(-1, 10, rows).astype(np.int32)
    W = (np.eye(10) + 0.3 * r.standard_normal((10, 10))).astype(np.float32)
    out = mixture.step(gate, experts, torch.from_numpy(X).cuda(), torch.from_numpy(y).cuda(),
                       torch.from_numpy(W).cuda())
    got = {k: v.cpu().numpy() for k, v in out.items()}

    logits = core.predict_ex(gate, X, kind=core.KIND_RAW).astype(np.float64)
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :2]
    assert np.array_equal(got["ids"], ids)
    top = np.take_along_axis(logits, ids, 1)
    w = np.exp(top - top[:, :1])
    w /= w.sum(1, keepdims=True)
    assert np.all(np.abs(got["weights"] - w) <= 1e-6 * w)
    every = np.stack([core.predict_ex(h, X, kind=core.KIND_RAW) for h in experts])
    mine = every[ids, np.arange(rows)[:, None]]
    assert np.array_equal(got["margins"][got["slots"]], mine)
    comb = (w[:, :, None] * mine).sum(1)
    assert np.abs(got["combined"] - comb).max() <= 2e-6

    known = y >= 0
    l = comb @ W.astype(np.float64).T
    lse = np.log(np.exp(l - l.max(1, keepdims=True)).sum(1)) + l.max(1)
    loss = (lse - l[np.arange(rows), np.clip(y, 0, 9)])[known].mean()
    assert abs(got["loss"] - loss) <= 1e-5
    g = np.exp(l - lse[:, None])
    g[np.arange(rows), np.clip(y, 0, 9)] -= 1.0
    g *= known[:, None] / known.sum()
    dcomb = g @ W
    dm = np.zeros_like(got["dmargins"], dtype=np.float64)
    dm[got["slots"]] = w[:, :, None] * dcomb[:, None, :]
    dw = (dcomb[:, None, :] * mine).sum(2)
    dl = np.zeros((rows, 10))
    np.put_along_axis(dl, ids, w * (dw - (w * dw).sum(1, keepdims=True)), 1)
    for name, want in (("dhead", g.T @ comb), ("dmargins", dm), ("dlogits", dl)):
        assert np.abs(got[name] - want).max() <= 1e-5 * np.abs(want).max(), name
