"""A mixture of forests with a softmax head, one training step on device memory.

    python examples/mixture.py [rows]

A ten-class gate forest scores every row; its raw margins choose two of ten expert
forests.  The rows are sorted by expert and laid out for the forests, every expert
scores its segment, and the ten margins of both experts are combined with the gate's
weights.  A softmax head (here a 10 x 10 calibration of the combined margins) gives the
loss; its gradient goes back through the combination to the margins of each expert and
to the gate's margins: what the next trees of each forest would be fitted to.

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

EXPERTS, CHOICES, CLASSES = 10, 2, 10


def make_forests(trees: int = 60):
    """(gate, experts): models of the ten-class configuration, each of its own seed."""
    handles = [_core.load_json(synth.model_to_json(synth.make_model("cfg4", trees=trees, seed=s)))
               for s in range(1, EXPERTS + 2)]
    for h in handles:
        _core.prepare(h, [0])
    return handles[0], handles[1:]


def step(gate, experts, x: torch.Tensor, labels: torch.Tensor, head: torch.Tensor) -> dict:
    """Loss and gradients of one step: x (rows, features) float32 row-major, labels int32
    (a label outside the classes leaves its row out), head (classes, classes) float32."""
    rows, features = x.shape
    dev = x.device
    stream = torch.cuda.current_stream().cuda_stream

    def buffer(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=dev)

    def address(t):
        return t.data_ptr()

    # the gate's margins choose the experts (a row-major predict waits for its work)
    logits = buffer(rows, EXPERTS)
    _core.predict_device(gate, 0, address(x), rows, features, features, address(logits),
                         kind=_core.KIND_RAW, layout=_core.LAYOUT_ROW_MAJOR, stream=stream)
    ids, weights = buffer(rows, CHOICES, dtype=torch.int32), buffer(rows, CHOICES)
    _core.route_device(0, address(logits), rows, EXPERTS, EXPERTS, CHOICES, _core.ROUTE_CHOSEN,
                       address(ids), address(weights), stream=stream)

    # rows sorted by expert; segments start at multiples of 4, so that every segment of the
    # feature-major matrix is 16-byte aligned as the forests' bulk copies want it
    slots_all = _core.sort_rows_capacity(rows, CHOICES, EXPERTS, align=4)
    ld = (slots_all + 3) // 4 * 4
    offsets = buffer(EXPERTS + 1, dtype=torch.int64)
    counts = buffer(EXPERTS, dtype=torch.int32)
    order = buffer(slots_all, dtype=torch.int32)
    slots = buffer(rows, CHOICES, dtype=torch.int32)
    room = _core.sort_rows_workspace(rows, CHOICES, EXPERTS)
    space = buffer(max(room, 1), dtype=torch.uint8)
    _core.sort_rows_device(0, address(ids), rows, CHOICES, EXPERTS, 4, address(offsets),
                           address(counts), address(order), address(slots), address(space), room,
                           stream=stream)
    gathered = buffer(features, ld)
    _core.gather_rows_device(0, _core.F32, address(x), rows, features, features,
                             _core.LAYOUT_ROW_MAJOR, CHOICES, EXPERTS, address(offsets),
                             address(order), address(slots), slots_all, address(gathered), ld,
                             _core.LAYOUT_FEATURE_MAJOR, stream=stream)

    # every expert scores its segment
    margins = torch.zeros((slots_all, CLASSES), device=dev)
    starts, sizes = offsets.tolist(), counts.tolist()  # the one copy to the host
    for e, forest in enumerate(experts):
        if sizes[e]:
            _core.predict_device(forest, 0, address(gathered) + 4 * starts[e], sizes[e], features, ld,
                                 address(margins) + 4 * CLASSES * starts[e], kind=_core.KIND_RAW,
                                 stream=stream)
    combined = buffer(rows, CLASSES)
    _core.combine_rows_device(0, _core.F32, address(margins), slots_all, CLASSES, CLASSES,
                              address(slots), address(weights), rows, CHOICES, address(combined),
                              CLASSES, stream=stream)

    # the head's loss, averaged over the labelled rows, and its gradient
    loss, lse = buffer(rows), buffer(rows)
    room = _core.head_workspace(_core.F32, rows, CLASSES, CLASSES, grad=True)
    space2 = buffer(room, dtype=torch.uint8)
    known = (labels >= 0) & (labels < CLASSES)
    dloss = torch.full((rows,), 1.0, device=dev) / known.sum().clamp(min=1)
    common = (address(combined), rows, CLASSES, CLASSES, address(head), CLASSES, CLASSES,
              address(labels))
    _core.head_loss_device(0, _core.F32, *common, address(loss), address(lse), address(space2),
                           room, stream=stream)
    dcombined, dhead = buffer(rows, CLASSES), buffer(CLASSES, CLASSES)
    _core.head_grad_device(0, _core.F32, *common, address(lse), address(dloss),
                           address(dcombined), CLASSES, address(dhead), CLASSES, address(space2),
                           room, stream=stream)

    # back to the experts' margins (by slot) and to the gate's
    dmargins, dweights = buffer(slots_all, CLASSES), buffer(rows, CHOICES)
    _core.combine_rows_grad_device(0, _core.F32, address(margins), slots_all, CLASSES, CLASSES,
                                   address(order), address(slots), address(weights), rows, CHOICES,
                                   address(dcombined), CLASSES, address(dmargins), CLASSES,
                                   address(dweights), stream=stream)
    dlogits = buffer(rows, EXPERTS)
    _core.route_grad_device(0, address(logits), rows, EXPERTS, EXPERTS, CHOICES, _core.ROUTE_CHOSEN,
                            address(ids), address(weights), address(dweights), address(dlogits),
                            EXPERTS, stream=stream)
    for h in (gate, *experts):
        _core.check_device(h, 0)
    _core.head_check_device(0, address(space2))
    return {"loss": loss.sum() / known.sum().clamp(min=1), "combined": combined, "ids": ids,
            "weights": weights, "slots": slots, "counts": counts, "margins": margins,
            "dhead": dhead, "dmargins": dmargins, "dlogits": dlogits}


def main(rows: int = 200_000) -> None:
    gate, experts = make_forests()
    x = torch.from_numpy(np.ascontiguousarray(synth.make_data("cfg4", rows=rows, layout="row"))).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    labels = torch.randint(0, CLASSES, (rows,), device="cuda", generator=g, dtype=torch.int32)
    head = torch.eye(CLASSES, device="cuda")
    for i in range(5):
        out = step(gate, experts, x, labels, head)
        print(f"step {i}: loss {float(out['loss']):.6f}, rows by expert {out['counts'].tolist()}")
        head -= 2.0 * out["dhead"]


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 200_000)
