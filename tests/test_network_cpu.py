"""Refusals and workspace sizes of the embeddings, the gated block and the clipping of
gradients: checked before the device."""

import re

import pytest

from conftest import ROOT

P = 1 << 20  # an aligned address that no refused call dereferences


@pytest.fixture
def core(lib_built):
    return lib_built


# ---- embeddings -----------------------------------------------------------------

def _embed(**change):
    a = dict(device=0, dtype=1, table=P, entries=100, cols=16, ld=16, ids=P, rows=4, k=2, starts=P,
             scale=1.0, out=P, ld_out=16)
    a.update(change)
    return list(a.values())


def _embed_grad(**change):
    a = dict(device=0, dtype=1, dout=P, rows=4, cols=16, ld_out=16, ids=P, k=2, starts=P, scale=1.0,
             table=P, entries=100, ld=16, room=P, bytes=1 << 30)
    names = {"out": "dout"}
    a.update({names.get(k, k): v for k, v in change.items()})
    return list(a.values())


BAD_EMBED = [(dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(entries=0), "entries"),
             (dict(entries=2 ** 30), "entries"), (dict(cols=0), "cols"), (dict(cols=2 ** 20 + 1), "cols"),
             (dict(rows=-1), "rows"), (dict(rows=2 ** 31), "2\\^31"), (dict(k=0), "k must"),
             (dict(k=2 ** 20 + 1), "k must"), (dict(rows=2 ** 20, k=2 ** 11), "2\\^31"),
             (dict(ld=15), "ld"), (dict(ld_out=15), "ld"), (dict(ld=2 ** 62), "2\\^31 bytes"),
             (dict(ld_out=2 ** 63 - 1), "2\\^31 bytes"), (dict(table=0), "null"), (dict(ids=0), "null"),
             (dict(out=0), "null"), (dict(table=P + 1), "aligned"), (dict(ids=P + 2), "aligned"),
             (dict(starts=P + 1), "aligned"), (dict(out=P + 1), "aligned")]


@pytest.mark.parametrize("change,match", BAD_EMBED)
def test_embed_refuses(core, change, match):
    with pytest.raises(core.MacBoostError, match=match):
        core.embed_device(*_embed(**change))
    with pytest.raises(core.MacBoostError, match=match):
        core.embed_grad_device(*_embed_grad(**change))


def test_embed_workspace(core):
    w = core.embed_workspace
    assert w(100, 16, 0, 2) == 0
    assert 0 < w(100, 16, 4, 2) <= w(100, 16, 4000, 2)
    for change, match in [(dict(room=0), "gradient needs"), (dict(bytes=w(100, 16, 4, 2) - 1), "gradient needs"),
                          (dict(room=P + 128), "256-byte")]:
        with pytest.raises(core.MacBoostError, match=match):
            core.embed_grad_device(*_embed_grad(**change))
    for bad in ((0, 16, 4, 2), (100, 0, 4, 2), (100, 16, -1, 2), (100, 16, 4, 0), (100, 16, 2 ** 40, 2 ** 19)):
        with pytest.raises(core.MacBoostError):
            w(*bad)


# ---- the gated block --------------------------------------------------------------

def _ffn(tail=(P, 32, P, 64, P, 24, P, 1 << 40), **change):
    a = dict(device=0, dtype=1, act=0, x=P, rows=400, cols=16, ld_x=16, w_in=P, width=32, ld_in=16,
             w_out=P, outs=24, ld_out=32)
    a.update(change)
    return [*a.values(), *tail]


GRAD_TAIL = dict(hidden=P, ld_hidden=32, pre=P, ld_pre=64, dy=P, ld_dy=24, dx=P, ld_dx=16, dw_in=P,
                 ld_din=16, dw_out=P, ld_dout=32, room=P, bytes=1 << 40)

BAD_FFN = [(dict(dtype=2), "dtype"), (dict(dtype=9), "dtype"), (dict(act=3), "activation"),
           (dict(act=-1), "activation"), (dict(rows=-1), "rows"), (dict(rows=2 ** 30 + 1), "rows"),
           (dict(cols=0), "cols"), (dict(cols=2 ** 20 + 1), "cols"), (dict(width=0), "width"),
           (dict(width=2 ** 20 + 1), "width"), (dict(outs=0), "outs"), (dict(outs=2 ** 31), "outs"),
           (dict(rows=2 ** 30, width=2 ** 20), "too many"), (dict(ld_x=15), "stride"),
           (dict(ld_in=15), "stride"), (dict(ld_out=31), "stride"), (dict(ld_x=2 ** 62), "stride"),
           (dict(x=0), "null"), (dict(w_in=0), "null"), (dict(w_out=0), "null"), (dict(x=P + 1), "aligned"),
           (dict(w_out=P + 1), "aligned")]


@pytest.mark.parametrize("change,match", BAD_FFN)
def test_ffn_refuses(core, change, match):
    with pytest.raises(core.MacBoostError, match=match):
        core.ffn_device(*_ffn(**change))
    with pytest.raises(core.MacBoostError, match=match):
        core.ffn_grad_device(*_ffn(GRAD_TAIL.values(), **change))


def test_ffn_refuses_outputs_and_workspace(core):
    for tail, match in [((0, 32, P, 64, P, 24, P, 1 << 40), "null"), ((P, 31, P, 64, P, 24, P, 1 << 40), "stride"),
                        ((P, 32, P, 63, P, 24, P, 1 << 40), "stride"), ((P, 32, P, 64, 0, 24, P, 1 << 40), "null"),
                        ((P, 32, P, 64, P, 23, P, 1 << 40), "stride"), ((P, 32, P, 64, P, 24, 0, 1 << 40), "needs"),
                        ((P, 32, P, 64, P, 24, P, 100), "needs"), ((P, 32, P, 64, P, 24, P + 64, 1 << 40), "256-byte"),
                        ((P, 32, P + 1, 64, P, 24, P, 1 << 40), "aligned")]:
        with pytest.raises(core.MacBoostError, match=match):
            core.ffn_device(*_ffn(tail))
    for change, match in [(dict(hidden=0), "null"), (dict(pre=0), "null"), (dict(dy=0), "null"),
                          (dict(ld_pre=63), "stride"), (dict(ld_dy=23), "stride"), (dict(ld_dx=15), "stride"),
                          (dict(ld_din=15), "stride"), (dict(ld_dout=31), "stride"), (dict(dx=P + 1), "aligned"),
                          (dict(dw_in=P + 1), "aligned"), (dict(bytes=1000), "needs")]:
        with pytest.raises(core.MacBoostError, match=match):
            core.ffn_grad_device(*_ffn({**GRAD_TAIL, **change}.values()))
    with pytest.raises(core.MacBoostError, match="null"):
        core.ffn_check_device(0, 0)


def test_ffn_workspace(core):
    w = core.ffn_workspace
    assert 0 < w(1, 400, 16, 32, 24) < w(1, 400, 16, 32, 24, strided=True)
    assert w(1, 400, 16, 32, 24) <= w(1, 400, 16, 32, 24, grad=True)
    assert w(1, 400, 15, 31, 23) == w(1, 400, 15, 31, 23, strided=True)
    for bad in ((2, 4, 16, 32, 24), (1, -1, 16, 32, 24), (1, 4, 0, 32, 24), (1, 4, 16, 0, 24), (1, 4, 16, 32, 0)):
        with pytest.raises(core.MacBoostError):
            w(*bad)


def test_nothing_to_do(core):
    """No rows, or no gradient asked for: no device is looked for."""
    core.embed_device(*_embed(rows=0, ids=0, table=0, out=0))
    core.ffn_device(*_ffn((0, 32, 0, 64, 0, 24, 0, 0), rows=0, x=0, w_in=0, w_out=0))
    none = {**GRAD_TAIL, "dx": 0, "dw_in": 0, "dw_out": 0}
    core.ffn_grad_device(*_ffn(none.values()))
    core.ffn_grad_device(*_ffn({**none, "dx": P}.values(), rows=0))


# ---- clipping ---------------------------------------------------------------------

def test_clip_refuses(core):
    good = core.GradientList([0, 1], [P, P], [10, 20], [P, P])
    room = core.clip_workspace(good)
    assert room > 0
    for g, norm, limit, space, bytes_, match in [
            (good, 1.0, P, 0, 1 << 20, "needs"), (good, 1.0, P, P, room - 1, "needs"),
            (good, -1.0, P, P, room, "max_norm"), (good, float("nan"), P, P, room, "max_norm"),
            (good, 1.0, 0, P, room, "null"), (good, 1.0, P + 2, P, room, "aligned"),
            (good, 1.0, P, P + 4, room, "8-byte"),
            (core.GradientList([0, 3], [P, P], [10, 20], [P, P]), 1.0, P, P, room, "dtype"),
            (core.GradientList([0, 1], [P, P], [10, -1], [P, P]), 1.0, P, P, room, "sizes"),
            (core.GradientList([0, 1], [P, P], [10, 2 ** 41], [P, P]), 1.0, P, P, room, "sizes"),
            (core.GradientList([0, 1], [P, P], [2 ** 40, 2 ** 40], [P, P]), 1.0, P, P, room, "too many"),
            (core.GradientList([0, 1], [P, 0], [10, 20], [P, P]), 1.0, P, P, room, "null"),
            (core.GradientList([0, 1], [P, P], [10, 20], [0, P]), 1.0, P, P, room, "null"),
            (core.GradientList([0, 1], [P, P + 1], [10, 20], [P, P]), 1.0, P, P, room, "aligned"),
            (core.GradientList([0, 1], [P, P], [10, 20], [P + 2, P]), 1.0, P, P, room, "aligned")]:
        with pytest.raises(core.MacBoostError, match=match):
            core.clip_device(0, g, norm, limit, space, bytes_)
    with pytest.raises(ValueError):
        core.GradientList([0], [P, P], [10, 20])
    with pytest.raises(core.MacBoostError):
        core.clip_workspace(core.GradientList([5], [P], [1]))


# ---- the C entry points ------------------------------------------------------------

def test_calls_are_guarded():
    """Each entry point's calls into the library stand inside the functions that catch."""
    source = (ROOT / "macboost_b200" / "csrc" / "capi.cpp").read_text()
    for name in ("embed_device", "embed_workspace", "embed_grad_device", "ffn_workspace", "ffn_device",
                 "ffn_grad_device", "ffn_check_device", "clip_workspace", "clip_device"):
        at = source.index(f"macboost_{name}(")
        body = source[at:source.index("\n}\n", at)]
        call = re.search(r"return guarded(_size)?\((err, )?\[&\].*mb::" + name + r"\(", body, re.S)
        assert call and body.count("mb::" + name) == 1, name
