"""The native torch binding: what works without it, and when it is built."""
import subprocess
import sys
from pathlib import Path

import pytest

pytest.importorskip("torch")

REPO = Path(__file__).resolve().parent.parent


def test_ops_without_the_binding():
    """A tree whose _bind.so does not fit the installed torch: every operator of
    the ctypes binding is there, the four that need it say so when called."""
    code = """
import sys
sys.modules["pixal3d.cpp_b200._bind"] = None
from pixal3d.cpp_b200 import flow, ops
import torch
assert callable(ops.linear) and callable(ops.varlen_attention)
x = torch.zeros((2, 16))
for call in (lambda: ops.quantize_rows(x), lambda: ops.rotary(x, x[0].double(), 1, 16),
             lambda: ops.linear_i8(x, x, x, x), lambda: ops.masked_attention(x, x, x, x, x, 1, 1, 1, 1.0)):
    try:
        call()
    except ImportError as e:
        assert "_bind.so" in str(e)
    else:
        raise SystemExit("not refused")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
