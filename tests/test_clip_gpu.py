"""The norm of many gradients and their clipping, on the GPU against 64 bits.

Tolerances: the squares of up to 8 values are added up in float32 (8 x 2^-24 of the
sum, halved by the root), the rest in 64 bits, the norm is rounded once: 5 x 2^-24 of itself.
A clipped value carries the factor's error (the same and one rounding), its own product and
rounding: 7 x 2^-24 and `half`, and half a subnormal step."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}
CODES = {"float32": 0, "bfloat16": 1, "float16": 2}


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


def _name(t):
    return str(t.dtype)[6:]


def _clip(core, torch, grads, max_norm, outs="new"):
    if outs == "new":
        outs = [torch.full_like(g, 7.0) for g in grads]
    gl = core.GradientList([CODES[_name(g)] for g in grads], [g.data_ptr() for g in grads],
                           [g.numel() for g in grads], None if outs is None else [o.data_ptr() for o in outs])
    need = core.clip_workspace(gl)
    room = torch.full((need + 8,), 255, dtype=torch.uint8, device="cuda")
    norm = torch.full((), 7.0, device="cuda")
    core.clip_device(0, gl, max_norm, norm.data_ptr(), room.data_ptr(), need,
                     stream=torch.cuda.current_stream().cuda_stream)
    assert torch.all(room[need:] == 255)
    return norm, outs


def _norm(torch, grads):
    return sum(float((g.double() ** 2).sum()) for g in grads) ** 0.5


def _check(torch, grads, norm, outs, max_norm):
    n = _norm(torch, grads)
    assert abs(float(norm) - n) <= 5 * 2.0 ** -24 * n
    factor = max_norm / n if n > max_norm else 1.0
    for g, o in zip(grads, outs):
        value = g.double() * factor
        bound = value.abs() * (7 * 2.0 ** -24 + HALF[_name(g)]) + TINY[_name(g)]
        assert torch.all((o.double() - value).abs() <= (bound if factor != 1.0 else 0.0))


def _grads(torch, sizes, seed, dtypes=("float32", "bfloat16", "float16"), offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        t = torch.randn(n + offset, device="cuda", generator=g).to(getattr(torch, dtypes[i % len(dtypes)]))
        out.append(t[offset:])
    return out


SIZES = [[1], [3], [7, 8, 9], [16_384, 8_192, 8_193, 1, 16_385], [100_003, 5, 0, 70_000], [1_000_003],
         [5, 11, 23] * 400, [33] * 1025, [2_000_000, 3_000_001, 4_000_000]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("ratio", [0.25, 3.0])
def test_clip(gpu, torch, sizes, ratio):
    grads = _grads(torch, sizes, len(sizes))
    limit = ratio * _norm(torch, grads)
    norm, outs = _clip(gpu, torch, grads, limit)
    _check(torch, grads, norm, outs, limit)
    again, outs2 = _clip(gpu, torch, grads, limit)
    assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(outs, outs2))
    # only the norm, and in place
    alone, _ = _clip(gpu, torch, grads, limit, None)
    assert torch.equal(norm, alone)
    same = [g.clone() for g in grads]
    _clip(gpu, torch, same, limit, same)
    assert all(torch.equal(a, b) for a, b in zip(same, outs))


@pytest.mark.parametrize("offset", [1, 3, 4])
def test_alignment(gpu, torch, offset):
    """Sides that reach a 16-byte boundary together, and sides that never do."""
    grads = _grads(torch, [20_000, 9_001, 17_000, 2], 3, offset=offset)
    limit = 0.5 * _norm(torch, grads)
    for shift in (offset, 0, 2):
        whole = [torch.full((g.numel() + shift + 1,), 7.0, dtype=g.dtype, device="cuda") for g in grads]
        outs = [w[shift:-1] for w in whole]
        norm, _ = _clip(gpu, torch, grads, limit, outs)
        _check(torch, grads, norm, outs, limit)
        assert all(torch.all(w[:shift] == 7.0) and float(w[-1]) == 7.0 for w in whole)


def test_extremes(gpu, torch):
    for scale in (1e30, 3e38, 1e-30, 1e-40, 1e-45):
        g = [torch.full((n,), scale, device="cuda") for n in (5, 1000, 40_000)]
        limit = 1e-46 if scale < 1e-35 else scale
        norm, outs = _clip(gpu, torch, g, limit)
        n = _norm(torch, g)
        if n < 3.4e38:
            assert abs(float(norm) - n) <= 5 * 2.0 ** -24 * n + 2.0 ** -149
        else:
            assert float(norm) == float("inf")
        factor = limit / n
        for a, o in zip(g, outs):
            value = a.double() * factor
            # a factor below the smallest normal number is rounded to its last place
            bound = value.abs() * 8 * 2.0 ** -24 + a.double().abs() * 2.0 ** -150 + 2.0 ** -149
            assert torch.all((o.double() - value).abs() <= bound)


def test_not_finite(gpu, torch):
    g = [torch.ones(10, device="cuda"), torch.ones(30_000, dtype=torch.bfloat16, device="cuda")]
    g[1][12_345] = float("inf")
    norm, outs = _clip(gpu, torch, g, 1.0)
    assert float(norm) == float("inf")
    assert torch.all(outs[0] == 0) and torch.isnan(outs[1][12_345])
    assert torch.all(torch.cat((outs[1][:12_345], outs[1][12_346:])) == 0)
    g[0][3] = float("nan")
    norm, outs = _clip(gpu, torch, g, 1.0)
    assert torch.isnan(norm) and all(torch.all(torch.isnan(o)) for o in outs)
    # no limit: copied
    norm, outs = _clip(gpu, torch, [torch.full((9,), float("inf"), device="cuda")], float("inf"))
    assert float(norm) == float("inf") and torch.all(outs[0] == float("inf"))


def test_limits(gpu, torch):
    g = _grads(torch, [1000, 2000], 5)
    norm, outs = _clip(gpu, torch, g, 0.0)
    assert float(norm) > 0 and all(torch.all(o == 0) for o in outs)
    zero = [torch.zeros(100, device="cuda")]
    norm, outs = _clip(gpu, torch, zero, 0.0)
    assert float(norm) == 0 and torch.all(outs[0] == 0)
    for empty in ([], [torch.empty(0, device="cuda")]):
        norm, _ = _clip(gpu, torch, empty, 1.0)
        assert float(norm) == 0
        norm, _ = _clip(gpu, torch, empty, 1.0, None)
        assert float(norm) == 0


def test_captured(gpu, torch):
    """A captured call keeps its list: replayed with other values, in place."""
    core = gpu
    grads = _grads(torch, [70_000, 13, 9_999], 6)
    gl = core.GradientList([CODES[_name(g)] for g in grads], [g.data_ptr() for g in grads],
                           [g.numel() for g in grads], [g.data_ptr() for g in grads])
    need = core.clip_workspace(gl)
    room = torch.empty(need, dtype=torch.uint8, device="cuda")
    norm = torch.empty((), device="cuda")

    def step(what):
        core.clip_device(0, what, 2.0, norm.data_ptr(), room.data_ptr(), need,
                         stream=torch.cuda.current_stream().cuda_stream)

    step(gl)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(gl)
    del gl
    for seed in (7, 8):
        fresh = _grads(torch, [70_000, 13, 9_999], seed)
        for g, f in zip(grads, fresh):
            g.copy_(f)
        graph.replay()
        _check(torch, fresh, norm, grads, 2.0)
