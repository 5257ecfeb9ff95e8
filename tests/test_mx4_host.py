"""Refusals and sizes of the 4-bit and logits entry points that need no GPU: every check stands before the first CUDA call."""
import ctypes as C
import math

import pytest


@pytest.fixture(scope="module")
def capi():
    import __graft_entry__ as ge
    ge.build()
    from crucible_strix_halo_b200 import capi
    return capi


BASE = 1 << 20          # an address that nothing reads


def test_sizes(capi):
    lib = capi.lib
    assert lib.cr_mx4_code_bytes(3, 192) == 288
    assert [lib.cr_mx4_scale_bytes(r, k) for r, k in ((1, 64), (128, 128), (129, 192), (12352, 2048))] == [512, 512, 2048, 97 * 16 * 512]
    assert lib.cr_mx4_code_bytes(0, 64) == 0 and lib.cr_mx4_scale_bytes(1, 0) == 0
    assert lib.cr_mx4_code_bytes(1 << 20, 1 << 14) == 1 << 33            # past 32 bits
    assert C.sizeof(capi.Mx4) == 24 and C.sizeof(capi.LogitsArgs) == 7 * 8 + 3 * 8 + 6 * 4


def _mx4(capi, rows=32, inner=64, codes=BASE, scales=BASE):
    return C.byref(capi.Mx4(codes, scales, rows, inner))


@pytest.mark.parametrize("bad", [dict(rows=0), dict(inner=32), dict(inner=96), dict(inner=0), dict(codes=None), dict(scales=None), dict(codes=BASE + 8),
                                 dict(scales=BASE + 4), dict(rows=1 << 24), dict(inner=1 << 24)])
def test_matrices_that_are_refused(capi, bad):
    lib, m, ok = capi.lib, _mx4(capi, **bad), _mx4(capi)
    out = (capi.ProjOut * 1)(capi.ProjOut(BASE, 0, 32, 32, 1))
    assert lib.cr_mx4_quant(BASE, capi.ROW_F32, 1 << 24, m, None) == capi.ERR_INVALID
    assert lib.cr_mx4_dequant(m, BASE, capi.ROW_F32, 1 << 24, None) == capi.ERR_INVALID
    assert lib.cr_mx4_gemm(m, ok, out, 1, None) == capi.ERR_INVALID
    assert lib.cr_mx4_gemm(ok, m, out, 1, None) == capi.ERR_INVALID
    assert lib.cr_mx4_rows(BASE, capi.ROW_F32, 1 << 24, 1, m, BASE, 1 << 30, out, 1, None) == capi.ERR_INVALID
    assert lib.cr_mx4_quant(BASE, capi.ROW_F32, 64, None, None) == capi.ERR_INVALID


@pytest.mark.parametrize("x,dtype,ld,R", [(None, 0, 64, 1), (BASE, 3, 64, 1), (BASE, -1, 64, 1), (BASE, 0, 63, 1), (BASE + 2, 0, 64, 1), (BASE + 1, 1, 64, 1),
                                          (BASE, 0, 64, 0), (BASE, 0, 64, -1)])
def test_rows_that_are_refused(capi, x, dtype, ld, R):
    lib, m = capi.lib, _mx4(capi)
    out = (capi.ProjOut * 1)(capi.ProjOut(BASE, 0, 32, 32, 1))
    assert lib.cr_mx4_rows(x, dtype, ld, R, m, BASE, 1 << 30, out, 1, None) == capi.ERR_INVALID
    if R == 1:
        assert lib.cr_mx4_quant(x, dtype, ld, m, None) == capi.ERR_INVALID
        assert lib.cr_mx4_dequant(m, x, dtype, ld, None) == capi.ERR_INVALID


@pytest.mark.parametrize("outs", [[], [(BASE, 0, 16, 16, 1)], [(BASE, 0, 64, 64, 1)], [(BASE, 32, 32, 32, 1)], [(None, 0, 32, 32, 1)], [(BASE + 4, 0, 32, 32, 1)],
                                  [(BASE, 0, 32, 31, 1)], [(BASE, 0, 32, 34, 1)], [(BASE, 0, 32, 36, 0)], [(BASE, 0, 32, 32, 1)] * 7])
def test_outputs_that_are_refused(capi, outs):
    lib, m = capi.lib, _mx4(capi)
    o = (capi.ProjOut * max(1, len(outs)))(*[capi.ProjOut(*x) for x in outs])
    assert lib.cr_mx4_gemm(m, m, o, len(outs), None) == capi.ERR_INVALID
    assert lib.cr_mx4_rows(BASE, 0, 64, 1, m, BASE, 1 << 30, o, len(outs), None) == capi.ERR_INVALID


@pytest.mark.parametrize("workspace,short", [(None, 0), (BASE + 8, 0), (BASE, 1)])
def test_workspaces_that_are_refused(capi, workspace, short):
    lib = capi.lib
    out = (capi.ProjOut * 1)(capi.ProjOut(BASE, 0, 32, 32, 1))
    need = lib.cr_mx4_rows_workspace_bytes(3, 192)
    assert need == 256 * 96 + 4 * 512 and lib.cr_mx4_rows_workspace_bytes(0, 64) == 0
    assert lib.cr_mx4_rows(BASE, 0, 192, 3, _mx4(capi, inner=192), workspace, need - short, out, 1, None) == capi.ERR_INVALID


def test_operands_of_different_inner_size(capi):
    out = (capi.ProjOut * 1)(capi.ProjOut(BASE, 0, 32, 32, 1))
    assert capi.lib.cr_mx4_gemm(_mx4(capi, inner=128), _mx4(capi), out, 1, None) == capi.ERR_INVALID
    assert b"128" in capi.lib.cr_last_error()


@pytest.mark.parametrize("bad", [dict(R=0), dict(V=0), dict(logits=None), dict(dtype=7), dict(ld=99), dict(out=None, choice=None), dict(out_ld=99),
                                 dict(out=BASE, out_ld=128), dict(mask=BASE, mask_ld=3), dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=math.inf),
                                 dict(repetition=math.nan), dict(frequency=math.nan), dict(presence=math.inf), dict(logits=BASE + 2)])
def test_spans_that_are_refused(capi, bad):
    fine = dict(logits=BASE, out=BASE * 2, choice=BASE * 3, ld=100, out_ld=100, R=2, V=100, dtype=capi.ROW_F32, repetition=1.0)
    spans = (capi.LogitsArgs * 2)(capi.LogitsArgs(**fine), capi.LogitsArgs(**dict(fine, **bad)))
    assert capi.lib.cr_logits_choose(spans, 2, None) == capi.ERR_INVALID
    assert capi.lib.cr_logits_choose(spans, 0, None) == capi.ERR_INVALID
    assert capi.lib.cr_logits_choose(None, 1, None) == capi.ERR_INVALID


def test_in_place_needs_fp32_rows(capi):
    spans = (capi.LogitsArgs * 1)(capi.LogitsArgs(logits=BASE, out=BASE, ld=100, out_ld=100, R=1, V=100, dtype=capi.ROW_BF16, repetition=1.0))
    assert capi.lib.cr_logits_choose(spans, 1, None) == capi.ERR_INVALID


def test_counting_that_is_refused(capi):
    lib = capi.lib
    assert lib.cr_token_count(None, 1, 1, BASE, 10, None) == capi.ERR_INVALID
    assert lib.cr_token_count(BASE, -1, 1, BASE, 10, None) == capi.ERR_INVALID
    assert lib.cr_token_count(BASE, 1, 1, None, 10, None) == capi.ERR_INVALID
    assert lib.cr_token_count(BASE, 1, 1, BASE, 0, None) == capi.ERR_INVALID
    assert lib.cr_token_count(None, 0, 1, BASE, 10, None) == capi.OK       # nothing to do
