"""The page selection's launches from the native module run without the GIL
(stand-in library as in test_gpu_host_ops_threads.py)."""

import shutil
import subprocess
import sys

import pytest

from my_vllm_amd import _native
from tests.test_gpu_host_ops_threads import ENTRY_POINTS

pytestmark = pytest.mark.gpu

LAUNCHES = ("mva_update_page_bounds", "mva_select_pages", "mva_paged_decode_selected")

CALLS = """
import importlib.machinery, importlib.util, sys
import torch

loader = importlib.machinery.ExtensionFileLoader("mva_host", sys.argv[1])
host = importlib.util.module_from_spec(importlib.util.spec_from_loader("mva_host", loader))
loader.exec_module(host)
bf = dict(dtype=torch.bfloat16, device="cuda")
i32 = dict(dtype=torch.int32, device="cuda")
q, cache, bounds = torch.zeros(4, 8, 128, **bf), torch.zeros(2, 16, 2, 128, **bf), torch.zeros(2, 2, 2, 128, **bf)
table, lens, starts = torch.zeros(4, 2, **i32), torch.zeros(4, **i32), torch.zeros(5, **i32)
lists, ws = torch.zeros(4, 2, 3, **i32), torch.zeros(64, dtype=torch.uint8, device="cuda")
for name, args in (("update_page_bounds", (cache, bounds, table, lens, None, None)),
                   ("update_page_bounds", (cache, bounds, table, lens, starts, 4)),
                   ("select_pages", (q, bounds, table, lens, 3, 1, 1, ws, None)),
                   ("select_pages", (q, bounds, table, lens, 3, 1, 1, ws, cache)),
                   ("paged_decode_selected", (q, cache, cache, lists, lens, 0.1, None, ws)),
                   ("paged_decode_selected", (q, cache, cache, lists, lens, 0.1, q, ws)),
                   ("sparse_decode", (q, bounds, cache, cache, table, lens, 0.1, 3, 1, 1, q, ws, True))):
    assert getattr(host, name)(*args) is not None, name
print("launched without the GIL")
"""


def test_launches_release_the_gil(gpu, tmp_path):
    source = tmp_path / "stand_in.c"
    source.write_text("extern int PyGILState_Check(void);\n"
                      'const char* mva_last_error(void) { return "the launch holds the GIL"; }\n'
                      "long mva_selection_workspace_bytes(void) { return 64; }\n"
                      + "".join(f"int {name}(void) {{ return PyGILState_Check(); }}\n"
                                for name in (*ENTRY_POINTS, *LAUNCHES)))
    subprocess.run(["gcc", "-shared", "-fPIC", str(source), "-o", str(tmp_path / _native.LIB_PATH.name)], check=True)
    module = shutil.copy(_native.HOST_PATH, tmp_path)
    run = subprocess.run([sys.executable, "-c", CALLS, str(module)], capture_output=True, text=True, timeout=100)
    assert "launched without the GIL" in run.stdout, run.stderr
