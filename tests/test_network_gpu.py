"""The operators of a network over forests together, as they are used: leaves embedded, a gated
block, the softmax head, all gradients back to the embeddings and clipped; and calls that
share a process.

The float32 step is compared with 64 bits as a whole: relative to the largest value of each
result, every step of the chain adds less than 2^-18 (the bounds of the single operators'
tests, of sums of at most a few thousand terms of similar size), and there are seven."""

import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


class Network:
    def __init__(self, core, torch, rows=700, trees=9, nodes=31, cols=40, width=72, classes=11, seed=1):
        self.core, self.torch = core, torch
        self.shape = rows, trees, nodes, cols, width, classes
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, scale=1.0):
            return torch.randn(shape, device="cuda", generator=g) * scale

        self.ids = torch.randint(-1, nodes, (rows, trees), device="cuda", generator=g, dtype=torch.int32)
        self.starts = torch.arange(trees, device="cuda", dtype=torch.int32) * nodes
        self.table = normal(trees * nodes, cols, scale=0.3)
        self.w_in, self.w_out = normal(2 * width, cols, scale=cols ** -0.5), normal(cols, width, scale=width ** -0.5)
        self.head = normal(classes, cols, scale=2 * cols ** -0.5)
        self.labels = torch.randint(-1, classes, (rows,), device="cuda", generator=g, dtype=torch.int32)
        self.dloss = torch.full((rows,), 1.0 / rows, device="cuda")
        f = torch.empty
        self.x, self.hidden, self.pre = f((rows, cols), device="cuda"), f((rows, width), device="cuda"), f((rows, 2 * width), device="cuda")
        self.y, self.loss, self.lse = f((rows, cols), device="cuda"), f(rows, device="cuda"), f(rows, device="cuda")
        self.dy, self.dx = f((rows, cols), device="cuda"), f((rows, cols), device="cuda")
        self.grads = {k: torch.empty_like(getattr(self, k)) for k in ("table", "w_in", "w_out", "head")}
        self.clipped = {k: torch.empty_like(v) for k, v in self.grads.items()}
        self.norm = f((), device="cuda")
        rooms = {"embed": core.embed_workspace(trees * nodes, cols, rows, trees),
                 "ffn": core.ffn_workspace(core.F32, rows, cols, width, cols, grad=True),
                 "head": core.head_workspace(core.F32, rows, cols, classes, grad=True)}
        self.list = core.GradientList([core.F32] * 4, [g.data_ptr() for g in self.grads.values()],
                                      [g.numel() for g in self.grads.values()],
                                      [c.data_ptr() for c in self.clipped.values()])
        rooms["clip"] = core.clip_workspace(self.list)
        # one workspace: the calls follow each other on one stream
        self.room = max(rooms.values())
        self.space = f(self.room, dtype=torch.uint8, device="cuda")
        self.max_norm = 0.05

    def step(self):
        core, s = self.core, self.torch.cuda.current_stream().cuda_stream
        rows, trees, nodes, cols, width, classes = self.shape
        space = (self.space.data_ptr(), self.room)

        def p(t):
            return t.data_ptr()

        core.embed_device(0, core.F32, p(self.table), trees * nodes, cols, cols, p(self.ids), rows, trees,
                          p(self.starts), 1.0, p(self.x), cols, stream=s)
        block = (p(self.x), rows, cols, cols, p(self.w_in), width, cols, p(self.w_out), cols, width, p(self.hidden),
                 width, p(self.pre), 2 * width)
        core.ffn_device(0, core.F32, core.ACT_GELU, *block, p(self.y), cols, *space, stream=s)
        head = (p(self.y), rows, cols, cols, p(self.head), classes, cols, p(self.labels))
        core.head_loss_device(0, core.F32, *head, p(self.loss), p(self.lse), *space, stream=s)
        core.head_grad_device(0, core.F32, *head, p(self.lse), p(self.dloss), p(self.dy), cols, p(self.grads["head"]),
                              cols, *space, stream=s)
        core.ffn_grad_device(0, core.F32, core.ACT_GELU, *block, p(self.dy), cols, p(self.dx), cols,
                             p(self.grads["w_in"]), cols, p(self.grads["w_out"]), width, *space, stream=s)
        core.embed_grad_device(0, core.F32, p(self.dx), rows, cols, cols, p(self.ids), trees, p(self.starts), 1.0,
                               p(self.grads["table"]), trees * nodes, cols, *space, stream=s)
        core.clip_device(0, self.list, self.max_norm, p(self.norm), *space, stream=s)

    def check(self):
        torch = self.torch
        rows, trees, nodes, cols, width, classes = self.shape
        w = {k: getattr(self, k).double().requires_grad_(True) for k in self.grads}
        at = self.ids.long() + self.starts.long()
        x = (torch.where((self.ids >= 0)[..., None], w["table"][at.clamp(min=0)], 0.0)).sum(1)
        gate, up = (x @ w["w_in"].t()).split(width, 1)
        y = (torch.nn.functional.gelu(gate) * up) @ w["w_out"].t()
        loss = torch.nn.functional.cross_entropy(y @ w["head"].t(), self.labels.long(), ignore_index=-1,
                                                 reduction="none")
        grads = torch.autograd.grad((loss * self.dloss.double()).sum(), tuple(w.values()))
        norm = sum(float((g * g).sum()) for g in grads) ** 0.5
        assert norm > self.max_norm
        tolerance = 7 * 2.0 ** -18

        def close(got, want, what):
            assert float((got.double() - want).abs().max()) <= tolerance * float(want.abs().max()), what

        close(self.loss, loss.detach(), "loss")
        close(self.norm, torch.tensor(norm, dtype=torch.float64, device="cuda"), "norm")
        for (k, got), want in zip(self.grads.items(), grads):
            close(got, want, k)
            close(self.clipped[k], want * (self.max_norm / norm), "clipped " + k)


def test_step(gpu, torch):
    net = Network(gpu, torch)
    net.step()
    net.check()


def test_step_captured(gpu, torch):
    """A whole step as a graph, replayed with other ids, labels and weights."""
    net = Network(gpu, torch, rows=300, seed=2)
    net.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        net.step()
    for seed in (3, 4):
        other = Network(gpu, torch, rows=300, seed=seed)
        for name in ("ids", "labels", "table", "w_in", "w_out", "head"):
            getattr(net, name).copy_(getattr(other, name))
        graph.replay()
        net.check()


def test_two_threads(gpu, torch):
    """Steps of different sizes at once, each thread on its own stream with its own workspace."""
    nets = [Network(gpu, torch, rows=r, width=w, seed=s) for r, w, s in ((400, 72, 5), (3, 200, 6), (1500, 16, 7))]
    errors = []

    def work(net):
        try:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                for _ in range(20):
                    net.step()
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 -- shown by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in nets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for net in nets:
        net.check()


def test_offsets_of_more_than_32_bits(gpu, torch):
    """A table of more than 4 GB, looked up and given gradients at both ends."""
    core, entries, cols, rows = gpu, 2_200_000, 1024, 900
    table = torch.zeros((entries, cols), dtype=torch.bfloat16, device="cuda")
    ids = torch.cat((torch.arange(300), entries - 1 - torch.arange(300), torch.full((300,), entries // 2))).int().cuda()
    table[ids.long()] = torch.randn((rows, cols), device="cuda").bfloat16()
    table[ids[899].long()] = 3.0
    out = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    core.embed_device(0, core.BF16, table.data_ptr(), entries, cols, cols, ids.data_ptr(), rows, 1, 0, 1.0,
                      out.data_ptr(), cols, stream=s)
    assert torch.equal(out, table[ids.long()])
    dout = torch.ones((rows, cols), dtype=torch.bfloat16, device="cuda")
    need = core.embed_workspace(entries, cols, rows, 1)
    room = torch.empty(need, dtype=torch.uint8, device="cuda")
    table.fill_(9.0)
    core.embed_grad_device(0, core.BF16, dout.data_ptr(), rows, cols, cols, ids.data_ptr(), 1, 0, 1.0,
                           table.data_ptr(), entries, cols, room.data_ptr(), need, stream=s)
    want = torch.zeros(entries, device="cuda").index_add_(0, ids.long(), torch.ones(rows, device="cuda"))
    assert torch.equal(table[:, 0].float(), want) and torch.equal(table[:, -1].float(), want)
    assert float(table.float().sum(0)[0]) == rows


def test_block_of_more_than_4_gb(gpu, torch):
    """pre and the gradients of gates and factors past 4 GB: the last rows, and the weights' gradients."""
    from test_ffn_gpu import Block
    rows, cols, width, outs = 70_000, 32, 16_384, 24
    b = Block(gpu, torch, rows, cols, width, outs, "bfloat16", "silu", seed=21)
    b.forward()
    b.grad()
    b.check()
    x, dy = b.x, b.dy
    b.x, b.dy = x[-200:].contiguous(), dy[-200:].contiguous()
    got = {k: v for k, v in b.results().items()}
    ref = b.reference()
    for name in ("hidden", "pre", "y", "dx"):
        value, bound = ref[name]
        assert torch.all((got[name][-200:].double() - value).abs() <= 1.02 * bound + 1e-37), name
    # the weights' gradients: sums of 14 parts of rows
    total = {"dw_in": 0.0, "dw_out": 0.0}
    slack = {"dw_in": 0.0, "dw_out": 0.0}
    for i in range(0, rows, 5000):
        b.x, b.dy = x[i:i + 5000].contiguous(), dy[i:i + 5000].contiguous()
        ref = b.reference()
        for name in total:
            total[name] = total[name] + ref[name][0]
            slack[name] = slack[name] + ref[name][1]
    for name, value in total.items():
        # a part's bound counts (5,000 + 16) steps of its sums, the whole has 14 times as many; what the
        # tensor core truncates is bounded by parts of 32,768 rows
        bound = 8 * slack[name]
        assert torch.all((got[name].double() - value).abs() <= bound + 1e-37), name
