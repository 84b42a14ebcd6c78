"""Sizes that do not fit in 64 bits once they are bytes: refused like any other that is too
large."""

import pytest

P = 1 << 20  # an aligned address that no refused call dereferences


@pytest.fixture
def core(lib_built):
    return lib_built


@pytest.mark.parametrize("ld", [2 ** 29, 2 ** 61, 2 ** 62, 2 ** 63 - 1])
def test_row_strides(core, ld):
    for call in (lambda: core.gather_rows_device(0, 0, P, 4, 16, ld, 1, 2, 8, P, P, P, 8, P, 16, 1),
                 lambda: core.gather_rows_device(0, 0, P, 4, 16, 16, 1, 2, 8, P, P, P, 8, P, ld, 1),
                 lambda: core.combine_rows_device(0, 0, P, 8, 10, ld, P, P, 4, 2, P, 10),
                 lambda: core.combine_rows_device(0, 0, P, 8, 10, 10, P, P, 4, 2, P, ld)):
        with pytest.raises(core.MacBoostError, match="rows of less than 2\\^31 bytes"):
            call()
