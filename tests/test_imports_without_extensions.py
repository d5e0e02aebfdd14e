"""The Python modules import on a machine without built libraries (or with a torch that torch_calls.so does not fit); the first call
that needs a library says how to build it. Run in processes of their own, in which the compiled module cannot be found."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCK = """
import importlib.abc, sys
class Block(importlib.abc.MetaPathFinder):
    def find_spec(self, name, path, target=None):
        if name == "dace_onnx_b200.torch_calls":
            raise ImportError("undefined symbol: none_such")
sys.meta_path.insert(0, Block())
"""


def run(code):
    r = subprocess.run([sys.executable, "-c", BLOCK + code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


def test_imports():
    run("from dace_onnx_b200 import ops, lowbit, donnx, graphs, encoder, onnx_model, torch_module, sharding")


def test_first_call_names_the_build():
    out = run("""
import torch
from dace_onnx_b200 import ops
x = torch.zeros(2, 16)
for call in (lambda: ops.rmsnorm(x), lambda: ops.quantize_rows(x), lambda: ops.matmul_scaled(x, x)):
    try:
        call()
    except ImportError as e:
        assert "python -m dace_onnx_b200.build" in str(e) and "none_such" in str(e)
        print("refused")
""")
    assert out.split() == ["refused"] * 3
