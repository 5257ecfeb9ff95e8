"""Sizes past what the 4-bit entry points take (no GPU is needed)."""
import pytest


@pytest.fixture(scope="module")
def capi():
    import __graft_entry__ as ge
    ge.build()
    from crucible_strix_halo_b200 import capi
    return capi


def test_workspaces_of_more_rows_than_a_call_takes(capi):
    need = capi.lib.cr_mx4_rows_workspace_bytes
    passes = ((1 << 20) - 1 + 19) // 20                          # of twenty fp32 rows, 256 digit rows each
    assert need((1 << 20) - 1, 64) == passes * 256 * 32 + passes * 2 * 512
    for R in (1 << 20, 1 << 28, 2 ** 31 - 1):
        assert need(R, 64) == 0
