"""CPU check: this library and torch in one process share one HIP runtime, whichever
is loaded first.  Each order in a process of its own."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ORDERS = {"library first": "from fe2o3_amd import _lib; _lib.lib()\nimport torch",
          "torch first": "import torch\nfrom fe2o3_amd import _lib; _lib.lib()"}
PRINT_LOADED = """
names = {line.split()[-1] for line in open("/proc/self/maps") if ".so" in line}
print([sum(lib in name for name in names) for lib in ("libamdhip64.so", "libhsa-runtime64.so")])
"""


@pytest.mark.parametrize("order", ORDERS)
def test_one_runtime(order):
    pytest.importorskip("torch")
    r = subprocess.run([sys.executable, "-c", ORDERS[order] + PRINT_LOADED], cwd=ROOT,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip() == "[1, 1]", r.stdout
