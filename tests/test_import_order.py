"""The library and torch share one HIP runtime in a process, whichever of the two is imported first (two of them
end the process at the first tensor on the device)."""
import os
import subprocess
import sys

import pytest

from helpers import ROOT

PACKAGE, TORCH = 'importlib.import_module("turbo-winfare-dense_amd")', "import torch"


@pytest.mark.parametrize("order", [(PACKAGE, TORCH), (TORCH, PACKAGE)], ids=["package first", "torch first"])
def test_one_hip_runtime(order):
    code = "\n".join(["import importlib, sys", f"sys.path.insert(0, {ROOT!r})", *order,
                      "print(len({l.split()[-1] for l in open('/proc/self/maps') if 'libamdhip64' in l}))"])
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "HIP_VISIBLE_DEVICES": ""})
    assert out.returncode == 0, out.stderr
    assert out.stdout.split()[-1] == "1"
