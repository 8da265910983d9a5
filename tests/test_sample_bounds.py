"""K11's bounds that the wrapper and the library share (no GPU needed)."""

import pytest

from mdlarc_scale_amd import _lib
from mdlarc_scale_amd import kernels as K


@pytest.fixture(scope="module", autouse=True)
def built():
    if not _lib.available():
        pytest.skip("libmdlarc_hip.so not built (python -m mdlarc_scale_amd.build)")


@pytest.mark.parametrize("rows", [1, 7, 64, 5000])
def test_rows_that_need_no_workspace(rows):
    """The wrapper takes a workspace of its own from the row length on that the library asks for one."""
    assert K.sample_workspace_bytes(rows, K.SAMPLE_LIST) == 0
    assert K.sample_workspace_bytes(rows, K.SAMPLE_LIST + 1) > 0
