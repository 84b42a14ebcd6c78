"""Long sums of the gated block: what is lost must not grow with their length.

Tolerances are relative to sums whose terms have one sign.  The tensor core truncates its sums
at each step of 16 terms, by at most 2^-23 of them; a part of a sum there has at most 32,768
terms, 2,048 steps: 2^-12.  Parts, and products of float32 on the CUDA cores, are added up in
float32."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


def _block(*a, **k):
    from test_ffn_gpu import Block
    return Block(*a, **k)


def _positive(torch, t, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for i in range(0, t.shape[0], 64):
        part = t[i:i + 64]
        part.copy_(torch.rand(part.shape, device="cuda", generator=g) + 1.0)


# products of warps, the CUDA cores' few rows (which a row of this length does not fit), tiles
@pytest.mark.parametrize("rows", [1, 3, 16, 40, 64, 300])
@pytest.mark.parametrize("cols", [40_000, 2 ** 20 - 8])
def test_long_rows(gpu, torch, rows, cols):
    """pre = x w_in^T over many columns, bfloat16."""
    width = 40
    b = _block(gpu, torch, rows, cols, width, 8, "bfloat16", "silu", seed=4)
    _positive(torch, b.x, 5)
    _positive(torch, b.w_in, 6)
    b.w_in.mul_(1.0 / cols)
    pre = torch.cat([b.x[i:i + 32].double() @ b.w_in.double().t() for i in range(0, rows, 32)])
    b.forward()
    b.check()
    got = b.results()
    assert float((got["pre"].double() / pre - 1).abs().max()) <= 2.0 ** -12 + 2.0 ** -18
    # the activation of what was kept
    gate, up = got["pre"].double().split(width, 1)
    want = torch.nn.functional.silu(gate) * up
    assert float((got["hidden"].double() / want - 1).abs().max()) <= 2.0 ** -8 + 2.0 ** -18
    y = b.results()["y"].clone()
    hidden = b.results()["hidden"].clone()
    b.hidden.fill_(7.0)
    b.forward(keep=False)
    assert torch.equal(b.results()["y"], y) and torch.equal(b.results()["hidden"], hidden)
    b.intact()


@pytest.mark.parametrize("rows,outs,pad", [(5, 2 ** 20 - 8, 0), (100, 2 ** 20 - 8, 0), (300, 40_000, 0), (70, 40_001, 3)])
def test_long_outputs(gpu, torch, rows, outs, pad):
    """dh = dy w_out over many outputs, bfloat16.  The gradients of gates and factors are rounded to
    bfloat16, by 2^-9 of each on average 0: their mean over `width` x rows values is off by what the
    sums lost, 2^-12, and by eight times 2^-9 / sqrt(rows x width)."""
    width = cols = 64
    b = _block(gpu, torch, rows, cols, width, outs, "bfloat16", "silu", pad=pad, seed=7)
    _positive(torch, b.dy, 8)
    _positive(torch, b.w_out, 9)
    b.w_out.mul_(1.0 / outs)
    b.forward()
    b.x.zero_()
    b.x[:, :cols] = 1.0
    # dw_in of one column is the sum of the rows' gradients; dx of an identity is the gradients themselves
    b.w_in.zero_()
    b.w_in[width:2 * width, :width] = torch.eye(width, device="cuda").bfloat16()
    b.grad()
    b.check()
    dy, w_out = b.dy[:, :outs], b.w_out[:, :width]
    dh = sum(dy[:, i:i + 65_536].double() @ w_out[i:i + 65_536].double() for i in range(0, outs, 65_536))
    gate = b.results()["pre"][:, :width].double()
    db = dh * torch.nn.functional.silu(gate)
    got = b.results()["dx"].double()
    there = db.abs() > 2.0 ** -60
    error = (got - db)[there] / db[there]
    assert float(error.abs().max()) <= 2.0 ** -8 + 2.0 ** -11
    assert abs(float(error.mean())) <= 2.0 ** -12 + 8 * 2.0 ** -9 / error.numel() ** 0.5
    first = {k: v.clone() for k, v in b.results().items()}
    for name in ("dx", "dw_in", "dw_out"):
        getattr(b, name).fill_(7.0)
        b.grad((name,))
        assert torch.equal(b.results()[name], first[name]), name
    dw_in = torch.cat((dh * b.results()["pre"][:, width:].double() * _silu_slope(torch, gate), db), 1).sum(0)
    most = torch.cat(((dh * b.results()["pre"][:, width:].double() * _silu_slope(torch, gate)).abs(), db.abs()), 1).sum(0)
    assert torch.all((first["dw_in"][:, 0].double() - dw_in).abs() <= most * (2.0 ** -8 + 2.0 ** -11) + dw_in.abs() * 2.0 ** -8)
    b.intact()


def _silu_slope(torch, a):
    p = 1.0 / (1.0 + torch.exp(-a))
    return p * (1.0 + a * (1.0 - p))


def test_narrow_gradient_of_many_rows(gpu, torch):
    """float32 with one output: dw_out of 500,000 rows, each of them 1 + 0.9 x 2^-12.  A sum past 4,096 in
    steps of 2^-11 leaves all of the 0.9 x 2^-12 behind, term after term.  A warp has at
    most 256 rows (251 in 27 rounds), and loses at most 2^-24 of what is there with each, half of them on
    average; eight threads share the 1,993 warps' sums and lose the same with each of theirs, and at most 2^-24
    of the whole with each of the eight: (251 / 2 + 250 / 2 + 8) x 2^-24 of it."""
    rows, width = 500_000, 2048
    b = _block(gpu, torch, rows, 4, width, 1, "float32", "silu", seed=3)
    b.hidden.fill_(1.0 + 0.9 * 2.0 ** -12)
    b.dy.fill_(1.0)
    b.grad(("dw_out",))
    want = rows * float(b.hidden[0, 0].double())
    got = b.results()["dw_out"].double()
    assert float((got - want).abs().max()) <= (251 / 2 + 250 / 2 + 8) * 2.0 ** -24 * want
    # with dx and dw_in beside it, the same bits
    first = b.results()["dw_out"].clone()
    b.pre.fill_(0.25)
    b.grad()
    assert torch.equal(b.results()["dw_out"], first)


@pytest.mark.parametrize("rows", [2, 70])
def test_long_rows_apart(gpu, torch, rows):
    """Rows that start off 16 bytes, odd sizes, a width of more than one tile; a row that is not finite leaves
    the others as they were."""
    cols, width = 33_001, 301
    b = _block(gpu, torch, rows, cols, width, 9, "bfloat16", "gelu_tanh", pad=3, seed=12)
    _positive(torch, b.x, 13)
    _positive(torch, b.w_in, 14)
    b.w_in.mul_(1.0 / cols)
    b.forward()
    b.check()
    b.intact()
    pre = b.x[:, :cols].double() @ b.w_in[:, :cols].double().t()
    got = {k: v.clone() for k, v in b.results().items()}
    assert float((got["pre"].double() / pre - 1).abs().max()) <= 2.0 ** -12 + 2.0 ** -18
    b.x[1, 5] = float("nan")
    b.forward()
    keep = [i for i in range(rows) if i != 1]
    assert torch.equal(b.results()["y"][keep], got["y"][keep]) and torch.isnan(b.results()["y"][1]).all()
    b.grad()
    b.check()
    b.intact()
