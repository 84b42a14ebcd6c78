"""Embeddings and their gradient on the GPU against the formulas in 64 bits.

Tolerances, elementwise: a sum of n float32 terms, added one after the other or in groups of
64 on three levels, is off by at most min(n, 300) roundings of 2^-24 of the sum of
magnitudes, the scale's product by one more, the result's own rounding by `half` of
itself (2^-24, 2^-8 for bfloat16, 2^-11 for float16) and by half a subnormal step."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}
CODES = {"float32": 0, "bfloat16": 1, "float16": 2}


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


def _lookups(torch, ids, starts, entries):
    at = ids.long() + (0 if starts is None else starts.long())
    return torch.where((ids >= 0) & (at >= 0) & (at < entries), at, -1)


def _forward(core, torch, table, entries, cols, ids, starts, scale, pad=0):
    rows, k = ids.shape
    out = torch.full((rows, cols + pad), 7.0, dtype=table.dtype, device="cuda")
    core.embed_device(0, CODES[str(table.dtype)[6:]], table.data_ptr(), entries, cols, table.stride(0),
                      ids.data_ptr(), rows, k, 0 if starts is None else starts.data_ptr(), scale,
                      out.data_ptr(), out.stride(0), stream=torch.cuda.current_stream().cuda_stream)
    assert torch.all(out[:, cols:] == 7.0)
    return out[:, :cols]


def _grad(core, torch, dout, entries, cols, ids, starts, scale, pad=0):
    rows, k = ids.shape
    need = core.embed_workspace(entries, cols, rows, k)
    room = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
    room[need:] = 3
    whole = torch.full((entries + 1, cols + pad), 7.0, dtype=dout.dtype, device="cuda")
    d = whole[:entries]
    core.embed_grad_device(0, CODES[str(dout.dtype)[6:]], dout.data_ptr(), rows, cols, dout.stride(0),
                           ids.data_ptr(), k, 0 if starts is None else starts.data_ptr(), scale,
                           d.data_ptr(), entries, d.stride(0), room.data_ptr(), need,
                           stream=torch.cuda.current_stream().cuda_stream)
    assert torch.all(d[:, cols:] == 7.0) and torch.all(whole[entries] == 7.0) and torch.all(room[need:] == 3)
    return d[:, :cols]


def _within(torch, got, value, magnitude, terms, dtype, what):
    bound = (terms.clamp(max=300) + 2) * 2.0 ** -24 * magnitude + value.abs() * HALF[dtype] + TINY[dtype]
    err = (got.double() - value).abs()
    assert torch.all(err <= bound), f"{what}: {float((err / bound).max()):.3g} of the bound"


def _check(core, torch, ids, starts, entries, cols, dtype, scale, pad, seed):
    rows, k = ids.shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = getattr(torch, dtype)
    table = torch.randn((entries, cols + pad), device="cuda", generator=g).to(t)
    dout = torch.randn((rows, cols + pad), device="cuda", generator=g).to(t)
    at = _lookups(torch, ids, starts, entries)
    got = _forward(core, torch, table, entries, cols, ids, starts, scale, pad)
    d = _grad(core, torch, dout, entries, cols, ids, starts, scale, pad)
    value = torch.zeros((rows, cols), dtype=torch.float64, device="cuda")
    size, terms = value.clone(), torch.zeros((rows, 1), dtype=torch.float64, device="cuda")
    dvalue = torch.zeros((entries, cols), dtype=torch.float64, device="cuda")
    dsize, dterms = dvalue.clone(), torch.zeros((entries, 1), dtype=torch.float64, device="cuda")
    for j in range(k):
        r = (at[:, j] >= 0).nonzero()[:, 0]
        e = at[r, j]
        row, up = scale * table[e, :cols].double(), scale * dout[r, :cols].double()
        value[r] += row
        size[r] += row.abs()
        terms[r] += 1
        dvalue.index_add_(0, e, up)
        dsize.index_add_(0, e, up.abs())
        dterms.index_add_(0, e, torch.ones((len(e), 1), dtype=torch.float64, device="cuda"))
    _within(torch, got, value, size, terms, dtype, "out")
    _within(torch, d, dvalue, dsize, dterms, dtype, "dtable")
    assert torch.all(d[dterms[:, 0] == 0] == 0) and torch.all(got[terms[:, 0] == 0] == 0)
    # the same bits again
    assert torch.equal(d, _grad(core, torch, dout, entries, cols, ids, starts, scale, pad))


def _ids(torch, rows, k, entries, seed, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = (torch.rand((rows, k), device="cuda", generator=g) ** spread * entries).int().clamp_(max=entries - 1)
    off = torch.rand((rows, k), device="cuda", generator=g) < 0.1
    ids[off] = torch.tensor([-1, entries, 2 ** 31 - 1, -2 ** 31], device="cuda", dtype=torch.int32)[
        torch.randint(0, 4, (int(off.sum()),), device="cuda", generator=g)]
    return ids


SIZES = [(1, 1, 1, 1), (1, 1, 100_000, 1024), (3, 2, 5, 3), (33, 7, 40, 33), (4096, 1, 300, 8),
         (4097, 1, 300, 8), (700, 9, 1023, 130), (2049, 2, 1024, 5), (64, 64, 2, 16), (5000, 3, 70_000, 20),
         (300_000, 1, 7, 4), (30, 1, 12, 5000), (20_000, 1, 300, 64), (1000, 100, 12_700, 64)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,k,entries,cols", SIZES)
def test_embed(gpu, torch, rows, k, entries, cols, dtype):
    ids = _ids(torch, rows, k, entries, rows + k)
    _check(gpu, torch, ids, None, entries, cols, dtype, 0.75, 0, rows)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,k,entries,cols", [
    (65_003, 1, 900, 256), (64_900, 1, 30_011, 260),      # chunks of 64 entries, long stretches and short ones
    (60_001, 1, 500, 2048), (26_001, 5, 20_011, 1000),    # of 128
    (5_000, 1, 1 << 20, 64), (16_384, 1, 1 << 19, 129),   # one block's sort while a large table is cleared
    (50_001, 1, 300, 100), (9_999, 1, 777, 520), (12_345, 2, 999, 520), (20_003, 3, 500, 96)])  # several units, rows
def test_plans(gpu, torch, rows, k, entries, cols, dtype):
    _check(gpu, torch, _ids(torch, rows, k, entries, rows), None, entries, cols, dtype, 1.0, 0, rows)


@pytest.mark.parametrize("pad", [1, 2, 8])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides(gpu, torch, pad, dtype):
    for rows, k, entries, cols in [(70, 3, 90, 64), (513, 1, 33, 7), (129, 2, 1000, 4)]:
        _check(gpu, torch, _ids(torch, rows, k, entries, 5), None, entries, cols, dtype, -2.0, pad, 6)


def test_starts(gpu, torch):
    """One table for several columns of ids, as the leaves of trees have it; starts that lead
    outside the table, and sums that 32 bits do not hold."""
    nodes, trees = 31, 20
    entries = nodes * trees
    ids = _ids(torch, 3000, trees, nodes, 8)
    ids[ids >= nodes] = -1
    starts = torch.arange(trees, dtype=torch.int32, device="cuda") * nodes
    _check(gpu, torch, ids, starts, entries, 12, "float32", 1.0, 0, 9)
    starts[3], starts[4], starts[5], starts[6] = -5, entries, 2 ** 31 - 1, -2 ** 31
    ids[:50, 5] = 2 ** 31 - 1
    ids[:50, 6] = 2 ** 31 - 1
    _check(gpu, torch, ids, starts, entries, 12, "float32", 1.0, 0, 9)


def test_one_row_for_all(gpu, torch):
    """A stretch of all levels of sums: 600,000 entries of one row of the table."""
    ids = torch.full((600_000, 1), 3, dtype=torch.int32, device="cuda")
    ids[5] = 4
    _check(gpu, torch, ids, None, 6, 3, "float32", 1.0, 0, 10)


def test_nothing_looked_up(gpu, torch):
    for rows in (1, 5000):
        ids = torch.full((rows, 2), -1, dtype=torch.int32, device="cuda")
        dout = torch.full((rows, 8), float("nan"), device="cuda")
        assert torch.all(_grad(gpu, torch, dout, 9, 8, ids, None, 1.0) == 0)
        table = torch.full((9, 8), float("nan"), device="cuda")
        assert torch.all(_forward(gpu, torch, table, 9, 8, ids, None, 1.0) == 0)
    empty = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    assert torch.all(_grad(gpu, torch, torch.empty((0, 8), device="cuda"), 9, 8, empty, None, 1.0) == 0)


def test_rows_that_add_nothing_stay_out(gpu, torch):
    """NaN in rows of dout, or of the table, that no id leads to."""
    ids = _ids(torch, 6000, 1, 50, 12)
    dout = torch.ones((6000, 4), device="cuda")
    off = (ids[:, 0] < 0) | (ids[:, 0] >= 50)
    dout[off] = float("nan")
    d = _grad(gpu, torch, dout, 50, 4, ids, None, 1.0)
    count = torch.bincount(ids[~off, 0].long(), minlength=50)
    assert torch.equal(d, count.float()[:, None].expand(50, 4))


def test_captured(gpu, torch):
    """A captured pair of calls, replayed with other ids, on another stream."""
    core, rows, entries, cols = gpu, 5000, 400, 24
    ids = _ids(torch, rows, 2, entries, 13)
    table, dout = torch.randn((entries, cols), device="cuda"), torch.randn((rows, cols), device="cuda")
    out, d = torch.empty((rows, cols), device="cuda"), torch.empty((entries, cols), device="cuda")
    need = core.embed_workspace(entries, cols, rows, 2)
    room = torch.empty(need, dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream().cuda_stream
        core.embed_device(0, 0, table.data_ptr(), entries, cols, cols, ids.data_ptr(), rows, 2, 0, 1.0,
                          out.data_ptr(), cols, stream=s)
        core.embed_grad_device(0, 0, dout.data_ptr(), rows, cols, cols, ids.data_ptr(), 2, 0, 1.0,
                               d.data_ptr(), entries, cols, room.data_ptr(), need, stream=s)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (14, 15):
        ids.copy_(_ids(torch, rows, 2, entries, seed))
        graph.replay()
        got = out.clone(), d.clone()
        out.fill_(7.0), d.fill_(7.0)
        step()
        assert torch.equal(got[0], out) and torch.equal(got[1], d)
