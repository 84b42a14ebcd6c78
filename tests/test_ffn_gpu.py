"""The gated feed-forward block on the GPU against the formulas in 64 bits.

Tolerances, elementwise, with u = 2^-23 (the tensor core's sums are truncated) and `half` a
rounding to the type (2^-24, 2^-8 for bfloat16).  A product of D terms is within (D + 16) u of
the sum of magnitudes, as in the head's test.  The activations' slopes are below 1.13 and
their slopes' slopes below 0.85; an activation's own error is within |a| (|a| + 8) u (its
sigmoid or distribution function a few u, and |a| u of the exponential's argument; the
formula used for bfloat16 is off by 1.5e-7 / 2, less than u), its slope's within (16 + 16 |a|) u.
hidden carries the errors of both halves of pre and one rounding; the gradients of gates and
factors those of the pre that was kept (float32) and a rounding of their own (2^-8; 2^-22 for
three bfloat16 terms).  Each result adds the errors of what it sums, (terms + 16) u of
the magnitudes and its rounding; products of two errors add less than 2%."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
ACTS = ["silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


class Block:
    """Inputs, outputs (filled with 7, `pad` columns wider) and the calls."""

    def __init__(self, core, torch, rows, cols, width, outs, dtype, act, pad=0, seed=1, scale=1.0, workspace=None):
        self.core, self.torch = core, torch
        self.shape = rows, cols, width, outs
        self.dtype, self.act, self.pad = dtype, act, pad
        self.code = core.F32 if dtype == "float32" else core.BF16
        t = getattr(torch, dtype)
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(r, c, s):
            return (torch.randn((r, c + pad), device="cuda", generator=g) * s).to(t)

        def empty(r, c):
            return torch.full((r + 2, c + pad), 7.0, dtype=t, device="cuda")[:r]

        self.x = normal(rows, cols, scale)
        self.w_in = normal(2 * width, cols, 2 / cols ** 0.5)
        self.w_out = normal(outs, width, 1 / width ** 0.5)
        self.dy = normal(rows, outs, 1.0)
        self.hidden, self.y = empty(rows, width), empty(rows, outs)
        self.pre = torch.full((rows + 2, 2 * width + pad), 7.0, device="cuda")[:rows]
        self.dx, self.dw_in, self.dw_out = empty(rows, cols), empty(2 * width, cols), empty(outs, width)
        self.need = core.ffn_workspace(self.code, rows, cols, width, outs, grad=True, strided=pad % 8 != 0)
        self.room = torch.full((self.need + 512,), 255, dtype=torch.uint8, device="cuda")
        self.at = (self.room.data_ptr() + 255) // 256 * 256

    def common(self):
        rows, cols, width, outs = self.shape
        act = ACTS.index(self.act)
        return (0, self.code, act, self.x.data_ptr(), rows, cols, self.x.stride(0), self.w_in.data_ptr(), width,
                self.w_in.stride(0), self.w_out.data_ptr(), outs, self.w_out.stride(0), self.hidden.data_ptr(),
                self.hidden.stride(0))

    def stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    def forward(self, keep=True):
        self.core.ffn_device(*self.common(), self.pre.data_ptr() if keep else 0, self.pre.stride(0),
                             self.y.data_ptr(), self.y.stride(0), self.at, self.need, stream=self.stream())

    def grad(self, want=("dx", "dw_in", "dw_out")):
        out = []
        for name in ("dx", "dw_in", "dw_out"):
            t = getattr(self, name)
            out += [t.data_ptr() if name in want else 0, t.stride(0)]
        self.core.ffn_grad_device(*self.common(), self.pre.data_ptr(), self.pre.stride(0), self.dy.data_ptr(),
                                  self.dy.stride(0), *out, self.at, self.need, stream=self.stream())

    def check(self):
        self.core.ffn_check_device(0, self.at)

    def results(self):
        rows, cols, width, outs = self.shape
        return {"hidden": self.hidden[:, :width], "pre": self.pre[:, :2 * width], "y": self.y[:, :outs],
                "dx": self.dx[:, :cols], "dw_in": self.dw_in[:, :cols], "dw_out": self.dw_out[:, :width]}

    def intact(self):
        """Nothing was written behind the columns, nor behind the last row."""
        rows, cols, width, outs = self.shape
        for t, c in ((self.hidden, width), (self.pre, 2 * width), (self.y, outs), (self.dx, cols),
                     (self.dw_in, cols), (self.dw_out, width)):
            assert self.torch.all(t[:, c:] == 7.0) and self.torch.all(t._base[t.shape[0]:] == 7.0)
        end = self.at + self.need - self.room.data_ptr()
        assert self.torch.all(self.room[end:] == 255)

    def reference(self):
        """{name: (value, bound)} in 64 bits."""
        torch = self.torch
        rows, cols, width, outs = self.shape
        half = 2.0 ** -8 if self.dtype == "bfloat16" else 2.0 ** -24
        half_d = 2.0 ** -8 if self.dtype == "bfloat16" else 2.0 ** -22
        x, w_in, w_out, dy = (t[:, :c].double() for t, c in ((self.x, cols), (self.w_in, cols),
                                                             (self.w_out, width), (self.dy, outs)))
        pre = x @ w_in.t()
        e_pre = (cols + 16) * U * (x.abs() @ w_in.abs().t())
        a, b = pre[:, :width].detach().requires_grad_(True), pre[:, width:]
        fn = torch.nn.functional
        f = fn.silu(a) if self.act == "silu" else fn.gelu(a, approximate="none" if self.act == "gelu" else "tanh")
        slope, = torch.autograd.grad(f.sum(), a)
        a, f = a.detach(), f.detach()
        ea, eb = e_pre[:, :width], e_pre[:, width:]
        own = a.abs() * (a.abs() + 8) * U
        h = f * b
        eh = b.abs() * (1.13 * ea + own) + f.abs() * eb + h.abs() * half
        y = h @ w_out.t()
        ey = eh @ w_out.abs().t() + (width + 16) * U * (h.abs() @ w_out.abs().t()) + y.abs() * half
        kept = e_pre + pre.abs() * 2.0 ** -24
        ka, kb = kept[:, :width], kept[:, width:]
        dh = dy @ w_out
        edh = (outs + 16) * U * (dy.abs() @ w_out.abs())
        da, db = dh * b * slope, dh * f
        eda = ((b * slope).abs() * edh + (dh * slope).abs() * kb +
               (dh * b).abs() * (0.85 * ka + (16 + 16 * a.abs()) * U) + da.abs() * half_d)
        edb = f.abs() * edh + dh.abs() * (1.13 * ka + own) + db.abs() * half_d
        d, ed = torch.cat((da, db), 1), torch.cat((eda, edb), 1)
        dx = d @ w_in
        edx = ed @ w_in.abs() + (2 * width + 16) * U * (d.abs() @ w_in.abs()) + dx.abs() * half
        dw_in = d.t() @ x
        ew_in = ed.t() @ x.abs() + (rows + 16) * U * (d.abs().t() @ x.abs()) + dw_in.abs() * half
        dw_out = dy.t() @ h
        ew_out = dy.abs().t() @ eh + (rows + 16) * U * (dy.abs().t() @ h.abs()) + dw_out.abs() * half
        return {"hidden": (h, eh), "pre": (pre, kept), "y": (y, ey), "dx": (dx, edx), "dw_in": (dw_in, ew_in),
                "dw_out": (dw_out, ew_out)}

    def compare(self, names=("hidden", "pre", "y", "dx", "dw_in", "dw_out")):
        got, ref = self.results(), self.reference()
        for name in names:
            value, bound = ref[name]
            bound = 1.02 * bound + 1e-37
            err = (got[name].double() - value).abs()
            assert self.torch.all(err <= bound), \
                f"{name} is {float((err / bound).max()):.3g} of its bound, {self.shape} {self.dtype} {self.act}"


SIZES = [(5, 8, 10, 1), (6, 16, 8, 8), (128, 64, 128, 256), (129, 65, 257, 7), (257, 100, 403, 10),
         (300, 72, 513, 65), (1000, 264, 96, 300), (33, 1030, 130, 130), (48, 512, 1024, 256),
         (700, 128, 256, 1), (2000, 24, 40, 16), (4100, 32, 64, 129), (17, 4096, 24, 40)]
FEW = [(1, 1, 1, 1), (1, 1024, 3001, 300), (2, 65, 70, 33), (3, 257, 100, 10), (4, 512, 999, 128),
       (1, 72, 16_384, 64), (2, 8, 20_000, 24), (4, 1000, 136, 1), (1, 40_000, 8, 8), (5, 64, 2048, 72),
       (8, 40, 4000, 136), (8, 512, 1000, 64), (11, 264, 72, 1000), (12, 33, 70, 9), (16, 96, 130, 260),
       (16, 2056, 640, 48), (25, 8, 8, 8), (47, 128, 1032, 512), (64, 512, 2000, 264), (65, 512, 2000, 264)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("shape", SIZES + FEW, ids=lambda s: "x".join(map(str, s)))
def test_ffn(gpu, torch, shape, dtype):
    act = ACTS[sum(shape) % 3]
    b = Block(gpu, torch, *shape, dtype, act, seed=sum(shape))
    b.forward()
    b.check()
    b.compare(("hidden", "pre", "y"))
    b.grad()
    b.check()
    b.compare()
    b.intact()
    # the same bits again, and without pre, and each gradient alone
    first = {k: v.clone() for k, v in b.results().items()}
    b.forward(keep=False)
    assert torch.equal(b.results()["y"], first["y"])
    for name in ("dx", "dw_in", "dw_out"):
        getattr(b, name).fill_(7.0)
        b.grad((name,))
        assert torch.equal(b.results()[name], first[name]), name


@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 15, 16, 17, 24, 25, 32, 33, 47, 48, 49])
@pytest.mark.parametrize("sizes", [(8, 8, 1), (136, 1184, 17), (1000, 24, 2400), (520, 4800, 40), (24, 9608, 2369)],
                         ids=lambda s: "x".join(map(str, s)))
def test_warp_products(gpu, torch, sizes, rows):
    """A few rows of bfloat16 on 16 bytes; K below, at and beyond a step of all warps, outputs that
    end inside a block's, and more of them than blocks."""
    for pad in (0, 8):
        b = Block(gpu, torch, rows, *sizes, "bfloat16", ACTS[rows % 3], pad=pad, seed=rows)
        b.forward()
        b.check()
        b.compare(("hidden", "pre", "y"))
        b.intact()
        y = b.results()["y"].clone()
        b.forward(keep=False)
        assert torch.equal(b.results()["y"], y)
        if rows > 1:
            b.x[rows // 2, 3] = float("nan")
            b.w_in[0, 0] = float("inf")  # of a gate that every row's y takes part of
            b.forward()
            keep = b.results()["pre"][[i for i in range(rows) if i != rows // 2]]
            assert torch.isfinite(keep[:, 1:]).all() and not torch.isfinite(keep[:, 0]).any()
            assert torch.isnan(b.results()["y"][rows // 2]).all()


@pytest.mark.parametrize("outs", [1, 4, 5, 8, 11, 12, 13, 16, 17])
@pytest.mark.parametrize("sizes", [(17, 12, 24), (33, 9, 403), (1001, 16, 1000), (20_003, 5, 136)],
                         ids=lambda s: "x".join(map(str, s)))
def test_few_outputs(gpu, torch, sizes, outs):
    """float32 with a few outputs, up to one more than the last that has kernels of its own."""
    for pad in (0, 3, 4):
        b = Block(gpu, torch, *sizes, outs, "float32", ACTS[outs % 3], pad=pad, seed=outs)
        b.forward()
        b.grad()
        b.check()
        b.compare()
        b.intact()
        first = {k: v.clone() for k, v in b.results().items()}
        b.forward(keep=False)
        assert torch.equal(b.results()["y"], first["y"])
        for name in ("dx", "dw_in", "dw_out"):
            getattr(b, name).fill_(7.0)
            b.grad((name,))
            assert torch.equal(b.results()[name], first[name]), name
            b.intact()


def test_few_outputs_rows_apart(gpu, torch):
    b = Block(gpu, torch, 100, 24, 200, 7, "float32", "silu", seed=3)
    b.forward()
    b.grad(("dx",))
    y, dx = b.results()["y"].clone(), b.results()["dx"].clone()
    b.x[10, 3], b.dy[20, 2], b.dy[21, 6] = float("nan"), float("inf"), float("nan")
    b.forward()
    b.grad(("dx",))
    keep = [i for i in range(100) if i not in (10, 20, 21)]
    assert torch.equal(b.results()["y"][keep], y[keep]) and torch.equal(b.results()["dx"][keep], dx[keep])
    assert torch.equal(b.results()["y"][20:22], y[20:22]) and torch.isnan(b.results()["y"][10]).all()
    assert not torch.isfinite(b.results()["dx"][[10, 20, 21]]).any()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_activations(gpu, torch, act, dtype):
    """Pre-activations far from zero too: x twenty times as large."""
    for rows in (3, 300):
        b = Block(gpu, torch, rows, 40, 96, 24, dtype, act, seed=7, scale=20.0)
        b.forward()
        b.grad()
        b.check()
        b.compare()
        for t in b.results().values():
            assert torch.all(torch.isfinite(t))


@pytest.mark.parametrize("pad", [8, 3])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("shape", [(130, 64, 72, 48), (3, 64, 72, 48), (300, 33, 40, 17)],
                         ids=lambda s: "x".join(map(str, s)))
def test_strides(gpu, torch, shape, dtype, pad):
    b = Block(gpu, torch, *shape, dtype, "silu", pad=pad, seed=3)
    b.forward()
    b.grad()
    b.check()
    b.compare()
    b.intact()


def test_far_gates(gpu, torch):
    """Gates whose square or cube overflows: the activation is the gate or 0, its slope 1 or 0."""
    for dtype in ("bfloat16", "float32"):
        for act in ACTS:
            for rows in (2, 200):
                b = Block(gpu, torch, rows, 8, 16, 8, dtype, act, seed=4)
                b.x.fill_(0.0)
                b.x[:, 0] = 1.0
                b.w_in.zero_()
                b.w_in[:16, 0] = torch.linspace(-1, 1, 16, device="cuda").to(b.x.dtype) * 1e30
                b.w_in[16:, 0] = 0.5
                b.forward()
                b.grad()
                b.check()
                gate = b.w_in[:16, 0].double()
                want = torch.where(gate > 0, gate * 0.5, 0.0)
                got = b.results()["hidden"].double()
                assert torch.all((got - want).abs() <= want.abs() * 2.0 ** -7), (dtype, act)
                assert torch.all(torch.isfinite(b.results()["dx"]))


def test_rows_apart(gpu, torch):
    """A row that is not finite leaves the others as they were."""
    for dtype in ("bfloat16", "float32"):
        for rows in (4, 300):
            b = Block(gpu, torch, rows, 40, 96, 24, dtype, "gelu", seed=5)
            b.forward()
            b.grad(("dx",))
            y, dx = b.results()["y"].clone(), b.results()["dx"].clone()
            b.x[1, 3] = float("nan")
            b.x[2] = float("inf")
            b.forward()
            b.grad(("dx",))
            keep = [i for i in range(rows) if i not in (1, 2)]
            assert torch.equal(b.results()["y"][keep], y[keep])
            assert torch.equal(b.results()["dx"][keep], dx[keep])
            assert not torch.isfinite(b.results()["y"][1]).any()


def test_differences(gpu, torch):
    """dx, dw_in and dw_out against differences of y: of f(t) = <dy, y(x + t dir)> over t = -s, s, which are
    off by s^2 / 6 of the third derivative (taken from 64 bits by halving s) -- here all in float32, where
    the differences themselves carry y's rounding, 2 x its bound / 2 s."""
    s = 2.0 ** -6
    for act in ACTS:
        b = Block(gpu, torch, 200, 24, 40, 16, "float32", act, seed=6)
        b.forward()
        b.grad()
        grads = {"x": b.dx.double(), "w_in": b.dw_in.double(), "w_out": b.dw_out.double()}
        bound_y = float((b.dy.double().abs() * (1.02 * b.reference()["y"][1])).sum())
        g = torch.Generator(device="cuda").manual_seed(9)
        for name, grad in grads.items():
            t = getattr(b, name)
            base = t.clone()
            direction = torch.randn(t.shape, device="cuda", generator=g)
            direction /= direction.norm()

            def value(step):
                t.copy_(base + step * direction)
                b.forward(keep=False)
                got = float((b.y.double() * b.dy.double()).sum())
                exact = float((b.reference()["y"][0] * b.dy.double()).sum())
                return got, exact

            (up, up64), (down, down64) = value(s), value(-s)
            (_, up64b), (_, down64b) = value(s / 2), value(-s / 2)
            t.copy_(base)
            curve = abs((up64 - down64) / (2 * s) - (up64b - down64b) / s) * 4 / 3
            want = float((grad * direction.double()).sum())
            # the points themselves are rounded to float32: 2^-24 of each value, times the gradient
            moved = 2 * float((base.double().abs() * 2.0 ** -23 * grad.abs()).sum()) / (2 * s)
            slack = float((1.02 * b.reference()[{"x": "dx"}.get(name, "d" + name)][1] * direction.double().abs()).sum())
            assert abs((up - down) / (2 * s) - want) <= 1.1 * curve + bound_y / s + moved + slack, (act, name)


def test_captured_and_other_stream(gpu, torch):
    """Two captured graphs that share a workspace, replayed in turn on one stream."""
    b = Block(gpu, torch, 300, 64, 128, 48, "bfloat16", "silu", seed=11)
    few = Block(gpu, torch, 2, 64, 128, 48, "bfloat16", "silu", seed=12)
    few.at, few.need = b.at, b.need
    graphs = []
    for block in (b, few):
        block.forward(), block.grad()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            block.forward(), block.grad()
        graphs.append(graph)
    side = torch.cuda.Stream()
    for seed in (13, 14):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for block in (b, few):
            block.x.copy_(torch.randn(block.x.shape, device="cuda", generator=g))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[0].replay()
            graphs[1].replay()
            graphs[0].replay()
        torch.cuda.current_stream().wait_stream(side)
        for block in (b, few):
            block.compare()


def test_no_rows(gpu, torch):
    b = Block(gpu, torch, 4, 16, 24, 8, "bfloat16", "silu")
    b.shape = (0, 16, 24, 8)
    b.forward()
    b.grad()
    assert torch.all(b.y == 7.0) and torch.all(b.dx == 7.0)
    assert torch.all(b.dw_in == 0) and torch.all(b.dw_out == 0)


def test_a_wait_that_ran_out_is_reported(gpu, torch, monkeypatch):
    b = Block(gpu, torch, 300, 64, 128, 48, "bfloat16", "silu", seed=11)
    monkeypatch.setenv("MACBOOST_WAIT_LIMIT_US", "3000")
    monkeypatch.setenv("MACBOOST_TEST_STALL_TILES", "1")
    b.forward()
    monkeypatch.delenv("MACBOOST_TEST_STALL_TILES")
    monkeypatch.delenv("MACBOOST_WAIT_LIMIT_US")
    b.grad()
    for _ in range(2):
        with pytest.raises(gpu.MacBoostError, match="gave up waiting"):
            b.check()
    b.forward()
    b.grad()
    b.check()
    b.compare()
