"""Sizes the adapter's C ABI refuses, without a GPU."""

import pytest

from test_adapter_host import P, lib, preference  # noqa: F401  (lib: the fixture)


@pytest.mark.parametrize("r", [0, -1, (1 << 30) + 1, (1 << 31) - 1])
def test_preference_rejected_rows(lib, r):  # noqa: F811
    assert preference(lib, r=r) == 1 and b"rejected rows" in lib.cvs_last_error()
