"""Clipping of lists that take more than one launch's table: many tensors, tensors that lie far
apart, tensors of more than 2^31 values, more than the L2 cache keeps, mostly zeros.  Tolerances as
in the test of shorter lists."""

import pytest

from test_clip_gpu import _check, _clip, _grads, _name, _norm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


# a table holds 2,032 tensors; one of up to 64 goes by a smaller table
@pytest.mark.parametrize("count", [64, 65, 2032, 2033, 2100, 4064, 4100, 6200])
@pytest.mark.parametrize("ratio", [0.25, 3.0])
def test_many_tensors(gpu, torch, count, ratio):
    sizes = [(i * 37) % 91 for i in range(count - 1)] + [70_001]  # some of them empty
    grads = _grads(torch, sizes, count)
    limit = ratio * _norm(torch, grads)
    norm, outs = _clip(gpu, torch, grads, limit)
    _check(torch, grads, norm, outs, limit)
    alone, _ = _clip(gpu, torch, grads, limit, None)
    assert torch.equal(norm, alone)
    same = [g.clone() for g in grads]
    again, _ = _clip(gpu, torch, same, limit, same)
    assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(same, outs))


@pytest.mark.parametrize("ratio", [0.25, 3.0])
def test_more_than_the_cache(gpu, torch, ratio):
    """400 MB, of which the last 80 are scaled first."""
    grads = _grads(torch, [30_000_000, 5, 40_000_003, 20_000_001, 35_000_000], 9)
    limit = ratio * _norm(torch, grads)
    norm, outs = _clip(gpu, torch, grads, limit)
    _check(torch, grads, norm, outs, limit)
    same = [g.clone() for g in grads]
    _clip(gpu, torch, same, limit, same)
    assert all(torch.equal(a, b) for a, b in zip(same, outs))


def test_far_apart(gpu, torch):
    """Gradients from both ends of 20 GB in turn, outputs elsewhere: a table's tensors lie within 8 GB, on
    either side."""
    here = torch.empty(20 << 28, dtype=torch.float32, device="cuda")      # 20 GB
    there = torch.empty(11 << 28, dtype=torch.float32, device="cuda")
    n, count = 50_001, 24
    assert here.numel() * 4 > 2 << 33
    g = torch.Generator(device="cuda").manual_seed(4)
    grads, outs = [], []
    for i in range(count):
        third = [0, here.numel() // 2, here.numel() - count * (n + 3)][i % 3]
        grads.append(here[third + i * (n + 3):][:n])
        end = [0, there.numel() - count * (n + 3)][i // 2 % 2]
        outs.append(there[end + i * (n + 3) + 1:][:n])
    for t, o in zip(grads, outs):
        t.copy_(torch.randn(n, device="cuda", generator=g))
        o.fill_(7.0)
    for ratio in (0.25, 3.0):
        limit = ratio * _norm(torch, grads)
        norm, _ = _clip(gpu, torch, grads, limit, outs)
        _check(torch, grads, norm, outs, limit)
        alone, _ = _clip(gpu, torch, grads, limit, None)
        assert torch.equal(norm, alone)
    limit = 0.25 * _norm(torch, grads)
    _clip(gpu, torch, grads, limit, outs)
    want = [o.clone() for o in outs]
    _clip(gpu, torch, grads, limit, grads)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


@pytest.mark.parametrize("dtype,extra", [("bfloat16", 5), ("bfloat16", 2 ** 31 + 3), ("float32", 1)])
def test_a_tensor_of_more_than_32_bits(gpu, torch, dtype, extra):
    n = 2 ** 31 + extra
    t = torch.empty(n, dtype=getattr(torch, dtype), device="cuda")
    g = torch.Generator(device="cuda").manual_seed(6)
    total, step = 0.0, 1 << 27
    for i in range(0, n, step):
        t[i:i + step].copy_(torch.randn(min(step, n - i), device="cuda", generator=g))
        total += float((t[i:i + step].double() ** 2).sum())
    small = torch.ones(3, device="cuda")
    exact = (total + 3.0) ** 0.5
    limit = 0.5 * exact
    ends = [t[:1000].clone(), t[2 ** 31 - 500:2 ** 31 + 500].clone(), t[-1000:].clone()]
    norm, _ = _clip(gpu, torch, [t, small], limit, None)
    assert abs(float(norm) - exact) <= 5 * 2.0 ** -24 * exact
    again, _ = _clip(gpu, torch, [t, small], limit, [t, small])
    assert torch.equal(norm, again)
    factor = limit / exact
    half = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}[dtype]
    for was, now in zip(ends, (t[:1000], t[2 ** 31 - 500:2 ** 31 + 500], t[-1000:])):
        value = was.double() * factor
        assert torch.all((now.double() - value).abs() <= value.abs() * (7 * 2.0 ** -24 + half) + 2.0 ** -133)
    scaled = sum(float((t[i:i + step].double() ** 2).sum()) for i in range(0, n, step)) + float((small ** 2).sum())
    assert abs(scaled ** 0.5 - limit) <= limit * (half + 7 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_mostly_zeros(gpu, torch, dtype):
    """As a table's gradient: whole units of zeros, zeros beside values, values too small for their squares."""
    g = torch.Generator(device="cuda").manual_seed(8)
    t = torch.zeros((40_000, 64), device="cuda")
    t[torch.randint(0, 40_000, (300,), device="cuda", generator=g)] = 0.01
    t[17, 3], t[18, :9] = 3.0, -2.0
    t[100:200] = 1e-30 if dtype != "float16" else 6e-8
    grads = [t.to(getattr(torch, dtype)).flatten(), torch.zeros(9, device="cuda")]
    for ratio in (0.25, 3.0):
        limit = ratio * _norm(torch, grads)
        norm, outs = _clip(gpu, torch, grads, limit)
        _check(torch, grads, norm, outs, limit)
    zero = [torch.zeros_like(x) for x in grads]
    norm, outs = _clip(gpu, torch, zero, 1.0)
    assert float(norm) == 0.0 and all(torch.all(o == 0) for o in outs)


def test_far_below_the_norm(gpu, torch):
    """A largest norm so far below the norm that their quotient is no normal float32, though the clipped
    values are: 5 roundings as ever, and half a subnormal step of the result."""
    for size, limit in ((1e38, 1e-5), (1e30, 1e-12), (3e38, 1e-4), (1e25, 1e-14), (1e38, 1e-8)):
        grads = [torch.full((n,), size, device="cuda") * torch.linspace(0.5, 1.0, n, device="cuda") for n in (7, 30_000)]
        grads.append(torch.full((999,), size, device="cuda").bfloat16())
        norm, outs = _clip(gpu, torch, grads, limit)
        n = _norm(torch, grads)
        for g, o in zip(grads, outs):
            value = g.double() * (limit / n)
            bound = value.abs() * (7 * 2.0 ** -24 + (2.0 ** -8 if _name(g) == "bfloat16" else 2.0 ** -24)) + 2.0 ** -133
            assert torch.all((o.double() - value).abs() <= bound), (size, limit)
        same = [g.clone() for g in grads]
        _clip(gpu, torch, same, limit, same)
        assert all(torch.equal(a, b) for a, b in zip(same, outs))
    # a limit of 0, and infinities, as ever
    norm, outs = _clip(gpu, torch, [torch.full((9,), 1e38, device="cuda")], 0.0)
    assert torch.all(outs[0] == 0)
