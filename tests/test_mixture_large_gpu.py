"""Gathers and combinations of many rows: the forms that only large calls take (columns in
runs of adjacent slots from 65,536 entries on, one warp a wide row from some 2,400 rows on).
Gathers move bits; tolerances of combinations as in test_mixture_gpu.py."""

import numpy as np
import pytest

import test_mixture_gpu as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(gpu):
    return pytest.importorskip("torch")


# tiles of the column form hold 4,096 / k rows: one row more than whole tiles, and less
CASES = [(65_536, 1, 1, 1, 1, 0), (69_633, 1, 28, 8, 4, 0), (22_000, 3, 5, 7, 1, 3),
         (16 * 1_365 + 1, 3, 3, 1_000, 4, 1), (8_193, 8, 17, 64, 16, 0), (70_001, 1, 9, 1_024, 4, 2),
         (40_000, 2, 33, 256, 1, 5), (3_000, 32, 2, 40, 1, 0), (200_000, 1, 3, 2, 1024, 1)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("target", [0, 1])
@pytest.mark.parametrize("kind", ["even", "few", "bad", "ordered"])
@pytest.mark.parametrize("rows,k,cols,experts,align,pad", CASES)
def test_gather_of_columns(gpu, torch, rows, k, cols, experts, align, pad, kind, target, dtype):
    """Feature-major input to both layouts.  few: most models have no row; bad: entries that
    are left out; ordered: every model's rows together."""
    core = gpu
    r = np.random.default_rng(rows + k)
    ids = r.integers(0, experts, (rows, k))
    if kind == "few":
        ids[:] = np.where(r.random(ids.shape) < 0.5, experts - 1, experts // 2)
    if kind == "bad":
        ids[r.random(ids.shape) < 0.4] = -1
        ids[r.random(ids.shape) < 0.1] = experts
    if kind == "ordered":
        ids.sort(axis=0)
    offsets, counts, order, slots = M.sort_on_gpu(core, torch, ids, experts, align)
    cap = order.numel()
    t = getattr(torch, dtype)
    x = torch.full((cols, rows + pad), float("nan"), dtype=t, device="cuda")
    x[:, :rows] = torch.randn((cols, rows), device="cuda").to(t)
    out = torch.full((cap, cols + pad) if target else (cols, cap + pad), 7.0, dtype=t, device="cuda")
    core.gather_rows_device(0, M.TYPES.index(dtype), x.data_ptr(), rows, cols, rows + pad, 0, k,
                            experts, offsets.data_ptr(), order.data_ptr(), slots.data_ptr(), cap,
                            out.data_ptr(), out.shape[1], target, stream=M._stream(torch))
    want = torch.where((order >= 0)[None, :], x[:, torch.clamp(order.long(), min=0) // k],
                       torch.zeros((), dtype=t, device="cuda"))
    got = out[:, :cols].t() if target else out[:, :cap]
    assert torch.equal(got, want)
    assert torch.all((out[:, cols:] if target else out[:, cap:]) == 7.0)


@pytest.mark.parametrize("dtype", M.TYPES)
@pytest.mark.parametrize("rows,cols,k,pad", [(2_368, 264, 2, 0), (5_000, 300, 1, 4), (2_600, 520, 8, 8),
                                             (3_001, 515, 4, 0), (2_500, 2_056, 3, 0)])
def test_combine_gradient_of_many_wide_rows(gpu, torch, rows, cols, k, pad, dtype):
    core = gpu
    t = getattr(torch, dtype)
    experts = 11
    r = np.random.default_rng(cols)
    ids = r.integers(-1, experts, (rows, k))
    offsets, counts, order, slots = M.sort_on_gpu(core, torch, ids, experts, 4)
    cap, ld = order.numel(), cols + pad
    y = torch.randn((cap, ld), device="cuda").to(t)
    y[order < 0] = float("nan")
    w = torch.randn((rows, k), device="cuda")
    w[slots < 0] = float("nan")
    dout = torch.randn((rows, ld), device="cuda").to(t)
    out = torch.full((rows, ld), 7.0, dtype=t, device="cuda")
    dy = torch.full((cap, ld), 7.0, dtype=t, device="cuda")
    dw = torch.full((rows, k), 7.0, device="cuda")
    code = M.TYPES.index(dtype)
    core.combine_rows_device(0, code, y.data_ptr(), cap, cols, ld, slots.data_ptr(), w.data_ptr(),
                             rows, k, out.data_ptr(), ld, stream=M._stream(torch))
    core.combine_rows_grad_device(0, code, y.data_ptr(), cap, cols, ld, order.data_ptr(),
                                  slots.data_ptr(), w.data_ptr(), rows, k, dout.data_ptr(), ld,
                                  dy.data_ptr(), ld, dw.data_ptr(), stream=M._stream(torch))
    half = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]
    there = (slots >= 0)[:, :, None]
    picked = torch.where(there, y.double()[slots.clamp(min=0).long(), :cols], 0.0)
    terms = picked * torch.where(there, w.double()[:, :, None], 0.0)
    err = (out[:, :cols].double() - terms.sum(1)).abs()
    assert torch.all(err <= (k + 2) * M.U * terms.abs().sum(1) + half * terms.sum(1).abs() + 3e-8)
    prod = picked * dout.double()[:, None, :cols]
    assert torch.all((dw.double() - prod.sum(2)).abs() <= (cols + 2) * M.U * prod.abs().sum(2))
    want = torch.zeros((cap, cols), dtype=t, device="cuda")
    want[slots[slots >= 0].long()] = (w[:, :, None] * dout.float()[:, None, :cols]).to(t)[slots >= 0]
    assert torch.equal(dy[:, :cols], want)
    assert torch.all(out[:, cols:] == 7.0) and torch.all(dy[:, cols:] == 7.0)
