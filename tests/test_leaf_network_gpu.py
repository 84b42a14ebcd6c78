"""The example of a network over a forest's leaves: it runs, and its gradients are those of the
formulas in 64 bits (relative to each one's largest value, 7 x 2^-18 as in the test of the
operators together)."""

import sys

import numpy as np
import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


@pytest.fixture(scope="module")
def example(torch):
    sys.path.insert(0, str(ROOT / "examples"))
    import leaf_network
    return leaf_network


def test_step(gpu, torch, example):
    rows = 3001
    forest, trees, nodes = example.make_forest(trees=12)
    x = torch.from_numpy(np.ascontiguousarray(example.synth.make_data("cfg2", rows=rows, layout="row"))).cuda()
    ids = example.leaves_of(forest, trees, x)
    assert int(ids.min()) >= 0 and int(ids.max()) < nodes
    labels = torch.randint(-1, example.CLASSES, (rows,), device="cuda", dtype=torch.int32)
    net = example.LeafNetwork(trees, nodes, rows)
    net.forward_backward(ids, labels, max_norm=float("inf"))
    w = {k: v.double().requires_grad_(True) for k, v in net.weights.items()}
    h = w["table"][(ids + net.starts).long()].sum(1)
    gate, up = (h @ w["w_in"].t()).split(example.WIDTH, 1)
    y = (torch.nn.functional.silu(gate) * up) @ w["w_out"].t()
    loss = torch.nn.functional.cross_entropy(y @ w["head"].t(), labels.long(), ignore_index=-1, reduction="none")
    grads = torch.autograd.grad(loss.sum() / rows, tuple(w.values()))
    for (name, got), want in zip(net.grads.items(), grads):
        assert float((got.double() - want).abs().max()) <= 7 * 2.0 ** -18 * float(want.abs().max()), name
    before = {k: v.clone() for k, v in net.weights.items()}
    net.update(0.25)
    for k, v in net.weights.items():
        assert torch.equal(v, before[k] - 0.25 * net.grads[k]) or torch.allclose(v, before[k] - 0.25 * net.grads[k])


def test_command(gpu, example, capsys):
    example.main(500, 2)
    assert capsys.readouterr().out.count("loss") == 2
