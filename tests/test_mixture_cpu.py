"""Refusals of the mixture entry points: every argument check precedes the device."""

import pytest

P = 1 << 20  # an aligned address that no refused call dereferences


@pytest.fixture
def core(lib_built):
    return lib_built


def _refused(core, match, fn, *args, **kw):
    with pytest.raises(core.MacBoostError, match=match):
        fn(*args, **kw)


@pytest.mark.parametrize("change,match", [
    (dict(rows=-1), "rows must be"), (dict(experts=0), "experts must be"),
    (dict(experts=1025, ld=1025), "experts must be"), (dict(experts=2 ** 40, ld=2 ** 40), "experts"),
    (dict(k=0), "k must be"), (dict(k=9), "k must be"), (dict(k=33, experts=64, ld=64), "k must be"),
    (dict(ld=7), "ld >= experts"), (dict(norm=2), "norm must be"), (dict(logits=0), "null argument"),
    (dict(ids=0), "null argument"), (dict(weights=P + 2), "aligned"),
    (dict(rows=2 ** 31), "below 2\\^31")])
def test_route_refuses(core, change, match):
    a = dict(logits=P, rows=4, experts=8, ld=8, k=2, norm=0, ids=P, weights=P)
    a.update(change)
    _refused(core, match, core.route_device, 0, a["logits"], a["rows"], a["experts"], a["ld"],
             a["k"], a["norm"], a["ids"], a["weights"])
    _refused(core, match, core.route_grad_device, 0, a["logits"], a["rows"], a["experts"], a["ld"],
             a["k"], a["norm"], a["ids"], a["weights"], P, P, max(a["experts"], 8))


def test_route_gradient_refuses(core):
    _refused(core, "null", core.route_grad_device, 0, P, 4, 8, 8, 2, 0, P, P, 0, P, 8)
    _refused(core, "null", core.route_grad_device, 0, P, 4, 8, 8, 2, 0, P, P, P, 0, 8)
    _refused(core, "ld >= experts", core.route_grad_device, 0, P, 4, 8, 8, 2, 0, P, P, P, P, 7)


@pytest.mark.parametrize("change,match", [
    (dict(align=0), "align"), (dict(align=1025), "align"), (dict(offsets=0), "null"),
    (dict(ids=0), "null"), (dict(order=0), "null"), (dict(offsets=P + 4), "8-byte"),
    (dict(space=0), "workspace"), (dict(room=8), "the sort needs"),
    (dict(k=9), "k must be"), (dict(rows=2 ** 31 - 1, k=1, align=1024), "2\\^31")])
def test_sort_refuses(core, change, match):
    a = dict(ids=P, rows=5000, k=1, experts=8, align=4, offsets=P, counts=P, order=P, slots=P,
             space=P, room=1 << 20)
    a.update(change)
    _refused(core, match, core.sort_rows_device, 0, *a.values())


def test_sort_sizes(core):
    assert core.sort_rows_capacity(10, 2, 4, 4) == 32
    assert core.sort_rows_workspace(0, 1, 4) == 0
    assert core.sort_rows_workspace(500, 1, 4) == 0
    assert core.sort_rows_workspace(10_000_000, 1, 4) > 0
    with pytest.raises(core.MacBoostError):
        core.sort_rows_workspace(10, 5, 4)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=3), "dtype"), (dict(cols=0), "cols"), (dict(ld=15), "ld"), (dict(layout=2), "layout"),
    (dict(layout_out=-1), "layout"), (dict(capacity=7), "capacity"), (dict(x=0), "null"),
    (dict(out=0), "null"), (dict(order=0), "null"), (dict(slots=0), "null"), (dict(x=P + 2), "aligned"),
    (dict(layout=0, ld=3), "ld"), (dict(layout_out=0, ld_out=7), "ld"), (dict(k=9), "k must be")])
def test_gather_refuses(core, change, match):
    a = dict(dtype=0, x=P, rows=4, cols=16, ld=16, layout=1, k=2, experts=8, offsets=P, order=P,
             slots=P, capacity=8, out=P, ld_out=16, layout_out=1)
    a.update(change)
    _refused(core, match, core.gather_rows_device, 0, *a.values())


@pytest.mark.parametrize("change,match", [
    (dict(dtype=-1), "dtype"), (dict(cols=0), "cols"), (dict(ld=9), "ld"), (dict(y=0), "null"),
    (dict(slots=0), "null"), (dict(rows=-1), "rows"), (dict(k=0), "k must be"), (dict(k=33), "k must be"),
    (dict(capacity=2 ** 31), "2\\^31"), (dict(weights=P + 1), "aligned")])
def test_combine_refuses(core, change, match):
    a = dict(dtype=0, y=P, capacity=8, cols=10, ld=10, slots=P, weights=P, rows=4, k=2)
    a.update(change)
    _refused(core, match, core.combine_rows_device, 0, *a.values(), P, 10)
    grad = [a["dtype"], a["y"], a["capacity"], a["cols"], a["ld"], P, a["slots"], a["weights"],
            a["rows"], a["k"]]
    _refused(core, match, core.combine_rows_grad_device, 0, *grad, P, 10, P, 10, P)


def test_combine_gradient_refuses(core):
    args = [0, 0, P, 8, 10, 10, P, P, P, 4, 2, P, 10, P, 10, P]
    for i, v, match in [(6, 0, "null"), (11, 0, "null"), (13, 0, "null"), (12, 9, "ld"),
                        (14, 9, "ld"), (15, P + 2, "aligned")]:
        bad = list(args)
        bad[i] = v
        _refused(core, match, core.combine_rows_grad_device, *bad)


def test_no_rows_is_no_work(core):
    """Calls without rows return before they look for a device."""
    core.route_device(0, 0, 0, 8, 8, 2, 0, 0, 0)
    core.route_grad_device(0, 0, 0, 8, 8, 2, 0, 0, 0, 0, 0, 8)
    core.combine_rows_device(0, 0, 0, 0, 4, 4, 0, 0, 0, 2, 0, 4)
    core.gather_rows_device(0, 0, 0, 0, 4, 4, 1, 2, 8, 0, 0, 0, 0, 0, 4, 1)
