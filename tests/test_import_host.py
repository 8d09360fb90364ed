"""CPU: the op module's import on a torch without its private shortcuts."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import sys
import torch
sys.path.insert(0, {where!r})
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
import gfx906_fa
assert gfx906_fa._get_device is torch.cuda.current_device
assert gfx906_fa._raw_stream is None
print("imported")
"""


def test_import_without_private_torch_functions():
    r = subprocess.run([sys.executable, "-c", CODE.format(where=os.path.join(ROOT, "gfx906-fa-vllm_amd"))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "imported" in r.stdout, r.stderr[-2000:]
