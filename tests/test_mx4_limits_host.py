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


@pytest.mark.parametrize("rows,inner", [(2 ** 32 + 32, 64), (32, 2 ** 32 + 64), (-2 ** 32 + 32, 64)])
def test_matrices_whose_sizes_do_not_fit_are_refused(capi, rows, inner):
    """They were cut to 32 bits: 32 x 64 in each case."""
    import torch
    from crucible_strix_halo_b200 import layers
    m = layers.Mx4(torch.zeros(32, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), rows, inner)
    with pytest.raises(ValueError, match="the 4-bit matrix"):
        layers.mx4_dequant(m)
    with pytest.raises(ValueError, match="x"):
        layers.mx4_gemm(m, m, [])
