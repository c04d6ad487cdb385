"""CPU: on a torch built without GPU support the bindings still import, and refuse at the call in their own words."""
import os
import subprocess
import sys

CODE = """
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
from swat_amd import _lib, mx, ops
x = torch.zeros(4, 32)
for f in (lambda: mx.quantize(x), lambda: ops.residual_norm_fwd(x, x), lambda: _lib.vec_ptr(x, "x", 4, 32), lambda: _lib.ptr(x)):
    try:
        f()
    except _lib.SwatHipError as e:
        assert "GPU" in str(e) or "CPU" in str(e), e
    else:
        raise AssertionError("taken")
print("refused")
"""


def test_import_and_refusal():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CODE], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0 and "refused" in r.stdout, r.stdout[-2000:]
