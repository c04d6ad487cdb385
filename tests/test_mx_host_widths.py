"""CPU: the weight gradient of a packed matrix without columns, which the format does not have."""
import pytest

P = 4096  # an address that is never read: the calls below launch nothing


@pytest.fixture(scope="module")
def lib():
    import os
    from swat_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib.lib()


@pytest.mark.parametrize("dbias", [None, P])
def test_no_columns_are_refused(lib, dbias):
    """(they used to pass, and leave dbias as it was)"""
    assert lib.swat_mx_linear_wgrad(P, 64, P, P, P, dbias, 4, 64, 0, None, 0, None) < 0
    assert "64 x 0" in lib.swat_last_error().decode()
    assert lib.swat_mx_linear_wgrad_workspace_bytes(4, 64, 0) < 0


def test_no_outputs_are_nothing_to_do(lib):
    assert lib.swat_mx_linear_wgrad(P, 64, P, P, P, P, 4, 0, 32, None, 0, None) == 0
    assert lib.swat_mx_linear_wgrad_workspace_bytes(4, 0, 32) == 0


def test_rows_next_to_two_to_the_31(lib):
    """The workspace of the seam's backward at the most rows that an int holds: that of 2048 teams, as at any large number."""
    most, some = (1 << 31) - 1, 1 << 22
    for d, groups, channels in ((1, 0, 0), (768, 0, 0), (1024, 0, 0), (8192, 0, 0), (4, 1, 1), (2000, 1, 1)):
        assert lib.swat_residual_norm_bwd_workspace_bytes(most, d, groups, channels) == lib.swat_residual_norm_bwd_workspace_bytes(some, d, groups, channels), d
    assert lib.swat_residual_norm_bwd_workspace_bytes(most, 16, 1, 0) == lib.swat_residual_norm_bwd_workspace_bytes(some, 16, 0, 0) + 4 * most
