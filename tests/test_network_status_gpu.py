"""A workspace that calls of a network share: a wait that ran out in a gradient's tiles is
still reported after the embeddings' gradient and the clipping that follow it there."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


def _stalled(monkeypatch, call):
    """The call with its copies left out, so that its (bounded) waits run out."""
    monkeypatch.setenv("MACBOOST_WAIT_LIMIT_US", "3000")
    monkeypatch.setenv("MACBOOST_TEST_STALL_TILES", "1")
    call()
    monkeypatch.delenv("MACBOOST_TEST_STALL_TILES")
    monkeypatch.delenv("MACBOOST_WAIT_LIMIT_US")


class Chain:
    """Inputs of the calls behind a block's gradient, all in the block's workspace."""

    def __init__(self, core, torch, block, rows, entries, ids_per_row, tensors):
        self.core, self.torch, self.block = core, torch, block
        cols = block.shape[1]
        g = torch.Generator(device="cuda").manual_seed(5)
        self.embed = rows, entries, cols, ids_per_row
        self.ids = torch.randint(0, entries, (rows, ids_per_row), device="cuda", generator=g, dtype=torch.int32)
        self.dout = torch.randn((rows, cols), device="cuda", generator=g)
        self.dtable = torch.empty((entries, cols), device="cuda")
        self.grads = [torch.randn(n, device="cuda", generator=g) for n in tensors]
        self.list = core.GradientList([core.F32] * len(tensors), [t.data_ptr() for t in self.grads], tensors,
                                      [t.data_ptr() for t in self.grads])
        self.norm = torch.empty((), device="cuda")
        self.need = max(core.embed_workspace(entries, cols, rows, ids_per_row), core.clip_workspace(self.list),
                        block.need)
        self.room = torch.full((self.need + 256,), 255, dtype=torch.uint8, device="cuda")
        self.at = (self.room.data_ptr() + 255) // 256 * 256
        block.at, block.need = self.at, self.need

    def run(self):
        core, s = self.core, self.torch.cuda.current_stream().cuda_stream
        rows, entries, cols, k = self.embed
        core.embed_grad_device(0, core.F32, self.dout.data_ptr(), rows, cols, cols, self.ids.data_ptr(), k, 0, 1.0,
                               self.dtable.data_ptr(), entries, cols, self.at, self.need, stream=s)
        core.clip_device(0, self.list, 1.0, self.norm.data_ptr(), self.at, self.need, stream=s)


# a sort of one block and of tiles; clipping in one launch and in two
@pytest.mark.parametrize("rows,entries,ids,tensors", [(300, 50, 1, [1000]), (9000, 700, 2, [1000, 3_000_000])])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_status_survives(gpu, torch, monkeypatch, dtype, rows, entries, ids, tensors):
    from test_ffn_gpu import Block
    b = Block(gpu, torch, 300, 64, 128, 48, dtype, "silu", seed=11)
    chain = Chain(gpu, torch, b, rows, entries, ids, tensors)
    b.forward()
    b.grad()
    chain.run()
    b.check()
    b.forward()
    _stalled(monkeypatch, b.grad)
    chain.run()
    for _ in range(2):
        with pytest.raises(gpu.MacBoostError, match="gave up waiting"):
            b.check()
    b.forward()
    b.grad()
    chain.run()
    b.check()
    b.compare()
    # the calls' own results are right there
    want = torch.zeros((entries, 64), dtype=torch.float64, device="cuda")
    for j in range(ids):
        want.index_add_(0, chain.ids[:, j].long(), chain.dout.double())
    most = float(torch.zeros((entries, 64), dtype=torch.float64, device="cuda").index_add_(
        0, chain.ids.long().flatten(), chain.dout.double().abs().repeat_interleave(ids, 0)).max())
    assert float((chain.dtable.double() - want).abs().max()) <= rows * ids * 2.0 ** -24 * most
    assert abs(float(sum((t.double() ** 2).sum() for t in chain.grads)) ** 0.5 - 1.0) <= 2.0 ** -20
