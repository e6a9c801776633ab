"""The package imports where torch was built without CUDA (no GPU needed): what such a build lacks is
looked up when a call needs it."""
import subprocess
import sys
from pathlib import Path


def test_modules_import_without_torch_cuda_bindings():
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            "import fitllm_b200.ops, fitllm_b200.lm_head, fitllm_b200.verify, fitllm_b200.layer, fitllm_b200.engine\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0, r.stderr[-800:]
