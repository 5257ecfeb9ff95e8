"""The binding beside a library that has the core's entry points alone: every call of the others is an exception, raised before anything
else is looked at and while the thread still holds the interpreter lock."""
import os
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "crucible_strix_halo_b200")

CORE = ("cr_proj_gemm", "cr_gdn_step", "cr_qsa_step", "cr_gdn_prefill", "cr_qsa_prefill")

CALLS = ("mx4_quant(torch.ones(1, 64), None)", "mx4_dequant(None, torch.float32)", "mx4_gemm(None, None, [])", "mx4_rows(torch.ones(1, 64), None, [])",
         "logits_choose([], None)", "token_count(torch.ones(1).int(), torch.ones(1).int(), 1)")

MAKE_CALLS = r"""
import importlib.machinery, importlib.util, sys, torch
loader = importlib.machinery.ExtensionFileLoader("_binding", sys.argv[1] + "/_binding.so")
binding = importlib.util.module_from_spec(importlib.util.spec_from_loader("_binding", loader))
for call in sys.argv[2:]:
    try:
        eval("binding." + call)
    except RuntimeError as e:
        print(str(e).splitlines()[0])
"""


@pytest.fixture(scope="module", autouse=True)
def built():
    import __graft_entry__ as ge
    ge.build()


@pytest.mark.parametrize("has", [(), ("cr_mx4_rows",)])             # mx4_rows needs two
def test_a_missing_entry_point_is_an_exception(tmp_path, has):
    stub = "".join("int %s() { return 1; }\n" % n for n in CORE + has) + 'const char* cr_last_error() { return ""; }\n'
    (tmp_path / "stub.c").write_text(stub)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(tmp_path / "libcrucible_attn.so"), str(tmp_path / "stub.c")], check=True)
    with open(os.path.join(PKG, "_binding.so"), "rb") as f:
        (tmp_path / "_binding.so").write_bytes(f.read())
    r = subprocess.run([sys.executable, "-c", MAKE_CALLS, str(tmp_path), *CALLS], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, "status %d\n%s" % (r.returncode, r.stderr[-2000:])
    assert r.stdout.splitlines() == ["the library beside this binding lacks the entry point"] * len(CALLS)
