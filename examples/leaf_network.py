"""A network on the leaves of a forest, trained on device memory.

    python examples/leaf_network.py [rows] [steps]

A saved forest sends every row to a leaf of each tree; the leaves' embeddings are added up
(one table for all trees' nodes), go through a gated feed-forward block and into a softmax
head.  One step is the loss, all gradients back to the embeddings, their norm and clipping,
and an update.  The forest itself stays as it is: it finds the features.

The device buffers are PyTorch tensors; any allocation serves, the package itself takes
addresses.
"""

from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from macboost_b200 import _core, synth  # noqa: E402

COLS, WIDTH, CLASSES = 64, 256, 10


def make_forest(trees: int = 40):
    """(handle, trees, nodes of a tree)."""
    model = synth.make_model("cfg2", trees=trees)
    forest = _core.load_json(synth.model_to_json(model))
    _core.prepare(forest, [0])
    return forest, trees, max(len(t["feature"]) for t in model["trees"])


def leaves_of(forest, trees: int, x: torch.Tensor) -> torch.Tensor:
    """The leaf that each row (float32, row-major) reaches in every tree: rows x trees int32."""
    rows, features = x.shape
    ids = torch.empty((rows, trees), dtype=torch.int32, device=x.device)
    _core.predict_device(forest, 0, x.data_ptr(), rows, features, features, ids.data_ptr(),
                         kind=_core.KIND_LEAF, layout=_core.LAYOUT_ROW_MAJOR,
                         stream=torch.cuda.current_stream().cuda_stream)
    _core.check_device(forest, 0)
    return ids


class LeafNetwork:
    """Weights, gradients and buffers of a fixed number of rows, all float32."""

    def __init__(self, trees: int, nodes: int, rows: int, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, scale):
            return torch.randn(shape, device="cuda", generator=g) * scale

        self.rows, self.trees, self.entries = rows, trees, trees * nodes
        self.starts = torch.arange(trees, dtype=torch.int32, device="cuda") * nodes
        self.weights = {"table": normal(self.entries, COLS, scale=trees ** -0.5),
                        "w_in": normal(2 * WIDTH, COLS, scale=COLS ** -0.5),
                        "w_out": normal(COLS, WIDTH, scale=WIDTH ** -0.5),
                        "head": normal(CLASSES, COLS, scale=COLS ** -0.5)}
        self.grads = {k: torch.empty_like(w) for k, w in self.weights.items()}
        self.list = _core.GradientList([_core.F32] * 4, [g.data_ptr() for g in self.grads.values()],
                                       [g.numel() for g in self.grads.values()],
                                       [g.data_ptr() for g in self.grads.values()])  # in place
        self.x, self.y, self.dy, self.dx = (torch.empty((rows, COLS), device="cuda") for _ in range(4))
        self.hidden = torch.empty((rows, WIDTH), device="cuda")
        self.pre = torch.empty((rows, 2 * WIDTH), device="cuda")
        self.loss, self.lse = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        self.dloss = torch.full((rows,), 1.0 / rows, device="cuda")
        self.norm = torch.empty((), device="cuda")
        # one workspace for calls that follow each other on one stream
        self.room = max(_core.embed_workspace(self.entries, COLS, rows, trees),
                        _core.ffn_workspace(_core.F32, rows, COLS, WIDTH, COLS, grad=True),
                        _core.head_workspace(_core.F32, rows, COLS, CLASSES, grad=True),
                        _core.clip_workspace(self.list))
        self.space = torch.empty(self.room, dtype=torch.uint8, device="cuda")

    def forward_backward(self, ids: torch.Tensor, labels: torch.Tensor, max_norm: float = 1.0) -> None:
        """loss, lse, norm and the clipped gradients (labels int32; one outside the classes leaves
        its row out).  Raises where a kernel gave up waiting."""
        w, d, rows = self.weights, self.grads, self.rows
        stream = torch.cuda.current_stream().cuda_stream
        space = (self.space.data_ptr(), self.room)

        def address(t):
            return t.data_ptr()

        _core.embed_device(0, _core.F32, address(w["table"]), self.entries, COLS, COLS, address(ids), rows,
                           self.trees, address(self.starts), 1.0, address(self.x), COLS, stream=stream)
        block = (address(self.x), rows, COLS, COLS, address(w["w_in"]), WIDTH, COLS, address(w["w_out"]), COLS,
                 WIDTH, address(self.hidden), WIDTH, address(self.pre), 2 * WIDTH)
        _core.ffn_device(0, _core.F32, _core.ACT_SILU, *block, address(self.y), COLS, *space, stream=stream)
        _core.ffn_check_device(0, space[0])  # the head's loss begins a status of its own
        head = (address(self.y), rows, COLS, COLS, address(w["head"]), CLASSES, COLS, address(labels))
        _core.head_loss_device(0, _core.F32, *head, address(self.loss), address(self.lse), *space, stream=stream)
        _core.head_grad_device(0, _core.F32, *head, address(self.lse), address(self.dloss), address(self.dy), COLS,
                               address(d["head"]), COLS, *space, stream=stream)
        _core.ffn_grad_device(0, _core.F32, _core.ACT_SILU, *block, address(self.dy), COLS, address(self.dx), COLS,
                              address(d["w_in"]), COLS, address(d["w_out"]), WIDTH, *space, stream=stream)
        _core.embed_grad_device(0, _core.F32, address(self.dx), rows, COLS, COLS, address(ids), self.trees,
                                address(self.starts), 1.0, address(d["table"]), self.entries, COLS, *space,
                                stream=stream)
        _core.clip_device(0, self.list, max_norm, address(self.norm), *space, stream=stream)
        # the head's calls and the block's gradient, whose status the calls since left alone
        _core.ffn_check_device(0, space[0])

    def update(self, rate: float) -> None:
        for k, w in self.weights.items():
            w.sub_(self.grads[k], alpha=rate)


def main(rows: int = 50_000, steps: int = 5) -> None:
    forest, trees, nodes = make_forest()
    x = torch.from_numpy(np.ascontiguousarray(synth.make_data("cfg2", rows=rows, layout="row"))).cuda()
    ids = leaves_of(forest, trees, x)
    labels = torch.randint(0, CLASSES, (rows,), device="cuda", dtype=torch.int32)
    net = LeafNetwork(trees, nodes, rows)
    for i in range(steps):
        net.forward_backward(ids, labels)
        net.update(0.5)
        print(f"step {i}: loss {float(net.loss.mean()):.6f}, gradients' norm {float(net.norm):.6f}")


if __name__ == "__main__":
    main(*(int(a) for a in sys.argv[1:3]))
