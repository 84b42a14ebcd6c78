"""Workspaces that calls of a network share: their first 256 bytes are left as they are."""


def test_workspaces_begin_behind_the_status(lib_built):
    core = lib_built
    assert core.embed_workspace(100, 16, 0, 2) == 0
    assert core.clip_workspace(core.GradientList([], [], [])) == 0
    assert core.clip_workspace(core.GradientList([0], [1 << 20], [0])) == 0
    # a block's sum of eight bytes behind them
    assert core.clip_workspace(core.GradientList([0], [1 << 20], [5])) == 256 + 8
    # keys, rows and ends of one entry, each on 256 bytes, and what joins chunks
    assert core.embed_workspace(1, 1, 1, 1) >= 256 + 3 * 256
