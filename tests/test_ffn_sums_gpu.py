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
