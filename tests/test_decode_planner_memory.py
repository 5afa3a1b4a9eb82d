"""CPU: the decode planners report that memory ran out; no exception leaves their C entries."""

import subprocess
import sys
from pathlib import Path

import pytest

CALL = """
import resource, sys
import numpy as np
from my_vllm_amd import _native

_native.load_library()
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (256 << 20),) * 2)
# The capacities are not there, but nothing is written before the memory runs out.
rows, out = np.zeros(64, np.int32).ctypes.data, np.zeros(4, np.int64)
many = 1 << 40
long, short = np.full(2, 2**31 - 1, np.int64), np.full(1, 2**27, np.int64)
calls = {
    "mva_decode_plan_listed": (long.ctypes.data, 2, 0, 0, 1, 2**31 - 2, 128, rows, many, rows, many, rows, 8),
    "mva_decode_plan_listed_mxfp4": (long.ctypes.data, 2, 0, 0, 1, 2**31 - 2, rows, many, rows, many, rows, 8),
    "mva_decode_plan_claims": (short.ctypes.data, 1, 0, 0, 1, many, 1.0, 1, 128, rows, many, rows, 8),
}
try:
    _native.call(sys.argv[1], *calls[sys.argv[1]], out.ctypes.data)
except RuntimeError as error:
    print(error)
"""


@pytest.mark.parametrize("planner", ["mva_decode_plan_listed", "mva_decode_plan_listed_mxfp4",
                                     "mva_decode_plan_claims"])
def test_planners_report_that_memory_ran_out(planner):
    # In a process of its own, with little address space left.
    run = subprocess.run([sys.executable, "-c", CALL, planner], capture_output=True, text=True, timeout=100,
                         cwd=Path(__file__).resolve().parents[1])
    assert run.returncode == 0 and "out of memory" in run.stdout, run.stderr
