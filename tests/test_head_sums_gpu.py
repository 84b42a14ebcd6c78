"""Long sums of the softmax head's gradients that do not cancel: dw over many rows, dh over
many classes.

Logits are zero here and the classes a power of two, so p = 1 / classes; dloss is held in
8 bits, so g = dloss p is exact in bfloat16 and the terms are what the formula says.  The
tensor core truncates its sum at each step of 16 terms: up to 2 units of 2^-23 (the sum,
and the terms' alignment to it).  Over a sum that grows evenly from zero that is half of
steps x 2^-22 at most; a part of a sum has at most 2,048 steps, so 2^-12, however many
there are.  The result's own rounding to bfloat16, at most 2^-8 of it, is as often up as
down: in the mean over n columns of their own scales 6 x 2^-8 / sqrt(3 n) at most."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


def _positive(torch, rows, cols, g):
    """Values in [1, 4): [1, 2) times the column's scale."""
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    scale = 2.0 ** torch.rand(cols, device="cuda", generator=g)
    for part in x.split(65536):
        part.copy_((1 + torch.rand(part.shape, device="cuda", generator=g)) * scale)
    return x


def _step(core, torch, h, w, y, dloss):
    (rows, cols), classes = h.shape, w.shape[0]
    need = core.head_workspace(core.BF16, rows, cols, classes, grad=True)
    room = torch.empty(need, dtype=torch.uint8, device="cuda")
    loss, lse = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    args = (0, core.BF16, h.data_ptr(), rows, cols, cols, w.data_ptr(), classes, cols, y.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    core.head_loss_device(*args, loss.data_ptr(), lse.data_ptr(), room.data_ptr(), need, stream=stream)
    core.head_grad_device(*args, lse.data_ptr(), dloss.data_ptr(), dh.data_ptr(), cols, dw.data_ptr(),
                          cols, room.data_ptr(), need, stream=stream)
    core.head_check_device(0, room.data_ptr())
    return dh, dw


def _bound(cols):
    return 2.0 ** -12 + 6 * 2.0 ** -8 / (3 * cols) ** 0.5


def test_dw_over_many_rows(gpu, torch):
    rows, cols, classes = 300_000, 8_192, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    h = _positive(torch, rows, cols, g)
    w = torch.zeros((classes, cols), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(rows, dtype=torch.int32, device="cuda")
    dloss = (1 + torch.rand(rows, device="cuda", generator=g)).bfloat16().float()
    _, dw = _step(gpu, torch, h, w, y, dloss)
    want = sum((d.double() / classes) @ x.double() for d, x in zip(dloss.split(65536), h.split(65536)))
    off = (dw[1:].double() / want - 1).mean(1)       # class 0 is every row's label
    assert off.abs().max() <= _bound(cols)


def test_dh_over_many_classes(gpu, torch):
    rows, cols, classes = 17, 2_048, 1 << 20
    g = torch.Generator(device="cuda").manual_seed(2)
    w = _positive(torch, classes, cols, g)
    w[0] = 0
    h = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(rows, dtype=torch.int32, device="cuda")
    dloss = (1 + torch.rand(rows, device="cuda", generator=g)).bfloat16().float()
    dh, _ = _step(gpu, torch, h, w, y, dloss)
    mean = sum(x.double().sum(0) for x in w.split(65536)) / classes
    off = (dh.double() / (dloss.double()[:, None] * mean) - 1).mean(1)
    assert off.abs().max() <= _bound(cols)
