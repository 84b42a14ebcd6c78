"""Which calls clear the head's status word: a wait of the loss call that ran out is still
reported after the gradient call that follows it in the same workspace."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


class Step:
    def __init__(self, core, torch, rows=300, cols=64, classes=2000, fill=255):
        self.core, self.torch = core, torch
        self.shape = rows, cols, classes
        g = torch.Generator(device="cuda").manual_seed(41)
        self.h = torch.randn((rows, cols), device="cuda", generator=g).bfloat16()
        self.w = torch.randn((classes, cols), device="cuda", generator=g).bfloat16()
        self.y = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.loss_out, self.lse = torch.empty(rows, device="cuda"), torch.zeros(rows, device="cuda")
        self.dloss = torch.ones(rows, device="cuda")
        self.dh, self.dw = torch.empty_like(self.h), torch.empty_like(self.w)
        self.need = core.head_workspace(core.BF16, rows, cols, classes, grad=True)
        self.room = torch.full((self.need,), fill, dtype=torch.uint8, device="cuda")
        self.args = (0, core.BF16, self.h.data_ptr(), rows, cols, cols, self.w.data_ptr(), classes, cols,
                     self.y.data_ptr())

    def loss(self):
        self.core.head_loss_device(*self.args, self.loss_out.data_ptr(), self.lse.data_ptr(),
                                   self.room.data_ptr(), self.need,
                                   stream=self.torch.cuda.current_stream().cuda_stream)

    def grad(self):
        cols = self.shape[1]
        self.core.head_grad_device(*self.args, self.lse.data_ptr(), self.dloss.data_ptr(),
                                   self.dh.data_ptr(), cols, self.dw.data_ptr(), cols,
                                   self.room.data_ptr(), self.need,
                                   stream=self.torch.cuda.current_stream().cuda_stream)

    def check(self):
        self.core.head_check_device(0, self.room.data_ptr())


@pytest.mark.parametrize("last", ["loss", "grad"])
def test_a_wait_that_ran_out_is_reported(gpu, torch, monkeypatch, last):
    core = gpu
    s = Step(core, torch)
    monkeypatch.setenv("MACBOOST_WAIT_LIMIT_US", "3000")
    monkeypatch.setenv("MACBOOST_TEST_STALL_TILES", "1")
    s.loss()
    monkeypatch.delenv("MACBOOST_TEST_STALL_TILES")
    monkeypatch.delenv("MACBOOST_WAIT_LIMIT_US")
    if last == "grad":
        s.grad()
    for _ in range(2):                     # looking does not clear it
        with pytest.raises(core.MacBoostError, match="gave up waiting"):
            s.check()
    s.loss()                               # the next loss call does
    s.grad()
    s.check()


@pytest.mark.parametrize("fill", [0, 1, 255])
def test_a_gradient_alone_reports_nothing(gpu, torch, fill):
    """A workspace that no loss call has seen, whatever it holds."""
    s = Step(gpu, torch, fill=fill)
    s.grad()
    s.check()
