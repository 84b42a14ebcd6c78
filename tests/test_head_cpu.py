"""Refusals and workspace sizes of the softmax head: checked before the device."""

import pytest

P = 1 << 20  # an aligned address that no refused call dereferences


@pytest.fixture
def core(lib_built):
    return lib_built


def _args(**change):
    a = dict(device=0, dtype=1, h=P, rows=4, cols=16, ld_h=16, w=P, classes=100, ld_w=16, labels=P)
    a.update(change)
    return list(a.values())


BAD = [(dict(dtype=2), "dtype"), (dict(dtype=7), "dtype"), (dict(rows=-1), "rows"),
       (dict(rows=2 ** 30 + 1), "rows"), (dict(cols=0), "cols"), (dict(cols=2 ** 20 + 1), "cols"),
       (dict(classes=0), "classes"), (dict(classes=2 ** 31), "classes"), (dict(ld_h=15), "ld"),
       (dict(ld_w=15), "ld"), (dict(h=0), "null"), (dict(w=0), "null"), (dict(labels=0), "null"),
       (dict(h=P + 1), "aligned"), (dict(labels=P + 2), "aligned")]


@pytest.mark.parametrize("change,match", BAD)
def test_refuses(core, change, match):
    with pytest.raises(core.MacBoostError, match=match):
        core.head_loss_device(*_args(**change), P, P, P, 1 << 30)
    with pytest.raises(core.MacBoostError, match=match):
        core.head_grad_device(*_args(**change), P, P, P, 16, P, 16, P, 1 << 30)


def test_refuses_outputs_and_workspace(core):
    for tail, match in [((0, P, P, 1 << 30), "null"), ((P, 0, P, 1 << 30), "null"),
                        ((P, P, 0, 1 << 30), "workspace"), ((P, P, P, 100), "the head needs"),
                        ((P, P, P + 128, 1 << 30), "256-byte")]:
        with pytest.raises(core.MacBoostError, match=match):
            core.head_loss_device(*_args(), *tail)
    for tail, match in [((0, P, P, 16, P, 16, P, 1 << 30), "null"),
                        ((P, 0, P, 16, P, 16, P, 1 << 30), "null"),
                        ((P, P, P, 15, P, 16, P, 1 << 30), "ld"),
                        ((P, P, P, 16, P, 15, P, 1 << 30), "ld"),
                        ((P, P, P + 1, 16, P, 16, P, 1 << 30), "aligned"),
                        ((P, P, P, 16, P, 16, P, 1000), "the head needs")]:
        with pytest.raises(core.MacBoostError, match=match):
            core.head_grad_device(*_args(), *tail)
    with pytest.raises(core.MacBoostError, match="null"):
        core.head_check_device(0, 0)


def test_workspace(core):
    w = core.head_workspace
    assert 0 < w(1, 4, 16, 100) <= w(1, 4, 16, 100, grad=True)
    # rows that do not start on 16 bytes are copied
    assert w(1, 400, 16, 100) < w(1, 400, 16, 100, strided=True) == w(1, 400, 16, 100, strided=True)
    assert w(1, 400, 15, 100) == w(1, 400, 15, 100, strided=True)
    # far below the logits of a large head
    assert w(1, 8192, 1024, 131072, grad=True) < 8192 * 131072 * 2 // 4
    for bad in ((2, 4, 16, 100), (1, -1, 16, 100), (1, 4, 0, 100), (1, 4, 16, 0)):
        with pytest.raises(core.MacBoostError):
            w(*bad)


def test_nothing_to_do(core):
    """No rows, or no gradient asked for: no device is looked for."""
    core.head_loss_device(0, 0, 0, 0, 8, 8, 0, 5, 8, 0, 0, 0, 0, 0)
    core.head_grad_device(0, 0, 0, 0, 8, 8, 0, 5, 8, 0, 0, 0, 0, 8, 0, 8, 0, 0)
    core.head_grad_device(0, 1, P, 4, 16, 16, P, 100, 16, P, P, P, 0, 16, 0, 16, P, 1 << 30)
