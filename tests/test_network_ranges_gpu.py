"""The network's operators where the other tests do not go: rows of hundreds and thousands of ids, a wide
block with one output and few rows, and a whole step in bfloat16."""

import pytest

from test_embed_gpu import _forward, _grad, _lookups

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,k,entries,cols", [(1, 129, 5000, 64), (1, 1000, 40_000, 64), (2, 4097, 300, 1),
                                                 (3, 20_000, 70_000, 200), (40, 501, 9000, 8), (1, 257, 3, 2050)])
def test_rows_of_many_ids(gpu, torch, rows, k, entries, cols, dtype):
    """A prediction from a large forest.  k float32 terms in the order of their columns: k roundings of 2^-24 of
    the magnitudes; the gradient adds at most rows x k in groups of 64 on three levels; a product, and the
    rounding to the type."""
    g = torch.Generator(device="cuda").manual_seed(k)
    t = getattr(torch, dtype)
    half = 2.0 ** -24 if dtype == "float32" else 2.0 ** -8
    table = torch.randn((entries, cols), device="cuda", generator=g).to(t)
    dout = torch.randn((rows, cols), device="cuda", generator=g).to(t)
    ids = torch.randint(-1, entries, (rows, k), device="cuda", generator=g, dtype=torch.int32)
    starts = torch.randint(-3, 4, (k,), device="cuda", generator=g, dtype=torch.int32)
    out = _forward(gpu, torch, table, entries, cols, ids, starts, 0.75)
    d = _grad(gpu, torch, dout, entries, cols, ids, starts, 0.75)
    at = _lookups(torch, ids, starts, entries)
    there = at >= 0
    for n in range(rows):
        found = table[at[n][there[n]]].double()
        value, size = 0.75 * found.sum(0), 0.75 * found.abs().sum(0)
        assert torch.all((out[n].double() - value).abs() <= (k + 2) * 2.0 ** -24 * size + value.abs() * half + 2.0 ** -133)
    times = torch.zeros((rows, entries), dtype=torch.float64, device="cuda")
    for n in range(rows):
        times[n].index_add_(0, at[n][there[n]], torch.ones(int(there[n].sum()), dtype=torch.float64, device="cuda"))
    value, size = 0.75 * times.t() @ dout.double(), 0.75 * times.t() @ dout.double().abs()
    terms = times.sum(0)[:, None].clamp(max=300)
    assert torch.all((d.double() - value).abs() <= (terms + 2) * 2.0 ** -24 * size + value.abs() * half + 2.0 ** -133)


@pytest.mark.parametrize("rows", [17, 33, 100, 1000])
@pytest.mark.parametrize("width,outs", [(16_384, 1), (16_385, 1), (8192, 2), (4096, 4), (1023, 16)])
def test_wide_with_few_outputs(gpu, torch, rows, width, outs):
    """Both sides of what the kernels for few outputs take."""
    from test_ffn_gpu import ACTS, Block
    b = Block(gpu, torch, rows, 12, width, outs, "float32", ACTS[rows % 3], seed=rows)
    b.forward()
    b.grad()
    b.check()
    b.compare()
    b.intact()


class Step:
    """A step in bfloat16: embeddings, block, head, their gradients, clipping.  `shared`: all of it in one
    workspace; else each call has its own, filled with ones first."""

    def __init__(self, core, torch, rows, trees, nodes, cols, width, classes, seed):
        from test_ffn_gpu import Block
        self.core, self.torch = core, torch
        self.shape = rows, trees, nodes, cols, width, classes
        g = torch.Generator(device="cuda").manual_seed(seed)
        bf16 = torch.bfloat16
        self.block = Block(core, torch, rows, cols, width, cols, "bfloat16", "silu", seed=seed)
        self.ids = torch.randint(-1, nodes, (rows, trees), device="cuda", generator=g, dtype=torch.int32)
        self.starts = torch.arange(trees, device="cuda", dtype=torch.int32) * nodes
        self.table = (torch.randn((trees * nodes, cols), device="cuda", generator=g) * trees ** -0.5).to(bf16)
        self.head = (torch.randn((classes, cols), device="cuda", generator=g) * cols ** -0.5).to(bf16)
        self.labels = torch.randint(-1, classes, (rows,), device="cuda", generator=g, dtype=torch.int32)
        self.dloss = torch.full((rows,), 1.0 / rows, device="cuda")
        self.loss, self.lse = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
        self.dtable, self.dhead = torch.zeros_like(self.table), torch.zeros_like(self.head)
        self.norm = torch.zeros((), device="cuda")
        b = self.block
        self.grads = [self.dtable, b.dw_in, b.dw_out, self.dhead]
        self.clipped = [torch.zeros_like(t) for t in self.grads]
        self.list = core.GradientList([core.BF16] * 4, [t.data_ptr() for t in self.grads],
                                      [t.numel() for t in self.grads], [t.data_ptr() for t in self.clipped])
        self.needs = {"embed": core.embed_workspace(trees * nodes, cols, rows, trees), "ffn": b.need,
                      "head": core.head_workspace(core.BF16, rows, cols, classes, grad=True),
                      "clip": core.clip_workspace(self.list)}

    def run(self, shared):
        core, torch, b = self.core, self.torch, self.block
        rows, trees, nodes, cols, width, classes = self.shape
        s = torch.cuda.current_stream().cuda_stream
        if shared:
            if not hasattr(self, "room"):
                self.room = torch.full((max(self.needs.values()) + 256,), 255, dtype=torch.uint8, device="cuda")
            at = (self.room.data_ptr() + 255) // 256 * 256
            places = {k: at for k in self.needs}
        else:
            self.rooms = {k: torch.full((n + 256,), 1, dtype=torch.uint8, device="cuda") for k, n in self.needs.items()}
            places = {k: (r.data_ptr() + 255) // 256 * 256 for k, r in self.rooms.items()}
        b.at = places["ffn"]

        def space(k):
            return places[k], self.needs[k]

        core.embed_device(0, core.BF16, self.table.data_ptr(), trees * nodes, cols, cols, self.ids.data_ptr(), rows,
                          trees, self.starts.data_ptr(), 1.0, b.x.data_ptr(), cols, stream=s)
        b.forward()
        head = (b.y.data_ptr(), rows, cols, cols, self.head.data_ptr(), classes, cols, self.labels.data_ptr())
        core.head_loss_device(0, core.BF16, *head, self.loss.data_ptr(), self.lse.data_ptr(), *space("head"), stream=s)
        core.head_grad_device(0, core.BF16, *head, self.lse.data_ptr(), self.dloss.data_ptr(), b.dy.data_ptr(), cols,
                              self.dhead.data_ptr(), cols, *space("head"), stream=s)
        b.grad()
        core.embed_grad_device(0, core.BF16, b.dx.data_ptr(), rows, cols, cols, self.ids.data_ptr(), trees,
                               self.starts.data_ptr(), 1.0, self.dtable.data_ptr(), trees * nodes, cols,
                               *space("embed"), stream=s)
        core.clip_device(0, self.list, 1e-3, self.norm.data_ptr(), *space("clip"), stream=s)

    def outputs(self):
        b = self.block
        return {"x": b.x, "hidden": b.hidden, "pre": b.pre, "y": b.y, "loss": self.loss, "lse": self.lse, "dy": b.dy,
                "dx": b.dx, "norm": self.norm, **{f"grad {i}": t for i, t in enumerate(self.grads)},
                **{f"clipped {i}": t for i, t in enumerate(self.clipped)}}


@pytest.mark.parametrize("shape", [(700, 9, 31, 40, 72, 11), (33, 5, 15, 64, 128, 300), (3000, 20, 127, 128, 512, 1000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_step_in_bfloat16(gpu, torch, shape):
    """All calls in one workspace, on a stream, and as a graph's replay: the bits of calls that share
    nothing.  The block's part is compared with 64 bits from the inputs that the chain gave it, the clipped
    gradients from the gradients."""
    s = Step(gpu, torch, *shape, seed=3)
    s.run(shared=False)
    torch.cuda.synchronize()
    apart = {k: v.clone() for k, v in s.outputs().items()}
    assert all(torch.isfinite(v.float()).all() for v in apart.values())
    s.block.compare()
    n = sum(float((t.double() ** 2).sum()) for t in s.grads) ** 0.5
    assert n > 1e-3 and abs(float(s.norm) - n) <= 5 * 2.0 ** -24 * n
    for t, c in zip(s.grads, s.clipped):
        value = t.double() * (1e-3 / n)
        assert torch.all((c.double() - value).abs() <= value.abs() * (2.0 ** -8 + 7 * 2.0 ** -24) + 2.0 ** -133)

    def wipe():
        for k, v in s.outputs().items():
            v.zero_()

    wipe()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.run(shared=True)
    torch.cuda.current_stream().wait_stream(side)
    for k, v in s.outputs().items():
        assert torch.equal(v, apart[k]), k
    gpu.ffn_check_device(0, s.block.at)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        s.run(shared=True)
    for _ in range(2):
        wipe()
        graph.replay()
        for k, v in s.outputs().items():
            assert torch.equal(v, apart[k]), k
